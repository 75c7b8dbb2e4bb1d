"""Linear attention with decays (zeno_b200/operators.py) against a 64-bit plain implementation.

Tolerances (2-norm of the error over that of the result).  32-bit results: operands are exact or cut at 24 bits, sums
are held in 32 bits and may be truncated (2^-23 each).  A chunk's result sums at most 128 / 16 + 32 / 16 steps of six terms,
60 truncations, and the states in front of it come with as many again; errors of single terms do not line up over
a norm, so a quarter of 120 * 2^-23, 3.6e-6, is allowed.  bfloat16 results: half a step of the result's own rounding (2^-8 of the value),
element by element, and 2^-16 of the result's size for second limbs that are rounded, eight times that for the largest of many.  The 32-bit results of a bfloat16 call are held to the 32-bit figure, the gradient of a decay that
all tokens of a head share to that figure of the sum of its terms' magnitudes (errors of one sign)."""
import pytest
import torch

import zeno_b200
import memory_plain as plain
from operators_plain import off

pytestmark = pytest.mark.gpu
TOL = 3.6e-6
DEV = "cuda"
NAMES = ("out", "state", "d_q", "d_k", "d_v", "d_g", "d_initial")


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def inputs(B, T, Hk, H, dk, dv, dtype, seed=0, reset=0.1, initial=True, fixed=False):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device=DEV)
    q, k, v = normal(B, T, Hk, dk).to(dtype), normal(B, T, Hk, dk).to(dtype), normal(B, T, H, dv).to(dtype)
    g = -torch.rand((H,) if fixed else (B, T, H), generator=gen, device=DEV) * 0.3
    r = (torch.rand((B, T), generator=gen, device=DEV) < reset).to(torch.uint8) if reset is not None else None
    return [q, k, v, g, r, normal(B, H, dk, dv) if initial else None]


def gradients(f, x, d_out, d_final=None, **kw):
    """out, final state and the gradients of the floating inputs that are there."""
    leaves = [t.detach().requires_grad_(True) if t is not None and t.is_floating_point() else t for t in x]
    out, final = f(*leaves, **kw)
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    outs, seeds = ([out], [d_out.to(out.dtype)]) if d_final is None else ([out, final], [d_out.to(out.dtype), d_final.to(final.dtype)])
    got = torch.autograd.grad(outs, wanted, seeds, allow_unused=True)
    return [out.detach(), final.detach(), *(torch.zeros_like(t) if y is None else y for y, t in zip(got, wanted))]


def exact(x, *args, **kw):
    return gradients(plain.linear_attention, [t.double() if t is not None and t.is_floating_point() else t for t in x], *args, **kw)


def check(got, want, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    if got.dtype == torch.float32:
        assert off(got, want) <= TOL, (what, off(got, want))
    elif got.numel():
        error = (got.double() - want.double()).abs() - 2.0 ** -8 * want.double().abs()
        size = float(want.double().square().mean()) ** 0.5
        assert float(error.max()) <= 8 * 2.0 ** -16 * size, (what, float(error.max()) / size)


def check_all(x, d_out, d_final=None, **kw):
    got = gradients(zeno_b200.linear_attention, x, d_out, d_final, **kw)
    want = exact(x, d_out, d_final, **kw)
    for name, a, b in zip(NAMES, got, want):
        if name == "d_g" and a.dim() == 1:  # one decay for all tokens: a sum that may leave little of its terms, whose errors count
            terms = exact([*x[:3], x[3].expand(x[2].shape[:3]), *x[4:]], d_out, d_final, **kw)[5]
            assert (a.double() - b.double()).abs().le(TOL * terms.double().abs().sum((0, 1))).all()
            continue
        check(a, b, name)
    with torch.no_grad():
        out, final = zeno_b200.linear_attention(*x, **kw)
    assert torch.equal(out, got[0]) and torch.equal(final, got[1])


HEADS = [(1, 1), (2, 2), (1, 3), (2, 4)]
WIDTHS = [(64, 64), (1, 1), (7, 13), (16, 32), (40, 24), (33, 64), (65, 9), (128, 128), (100, 128), (127, 33)]
LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 128, 193]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", LENGTHS)
def test_lengths(T, dtype):
    for i, (Hk, H) in enumerate(HEADS):
        dk, dv = WIDTHS[(T + i) % len(WIDTHS)]
        x = inputs(3, T, Hk, H, dk, dv, dtype, seed=T, initial=i % 2 == 0, fixed=i >= 2, reset=(None, 0.05, 0.3, 0.1)[i])
        d = torch.randn(3, T, H, dv, device=DEV).to(dtype)
        check_all(x, d, torch.randn(3, H, dk, dv, device=DEV) if i != 1 else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
def test_widths(dk, dv, dtype):
    for T, fixed in ((20, True), (90, False)):
        x = inputs(2, T, 2, 2, dk, dv, dtype, seed=dk, fixed=fixed)
        check_all(x, torch.randn(2, T, 2, dv, device=DEV).to(dtype), torch.randn(2, 2, dk, dv, device=DEV), scale=0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hk,H,dk,dv", [(1, 1000, 1, 1, 64, 64), (2, 700, 1, 2, 128, 100), (1, 1500, 2, 2, 24, 40), (3, 400, 1, 1, 64, 128),
                                            (60, 130, 1, 1, 32, 32)])
def test_few_long_rollouts(B, T, Hk, H, dk, dv, dtype):
    """Rollouts that are cut into segments, with episodes longer and shorter than one."""
    for fixed, reset in ((True, None), (False, 0.004), (True, 0.1)):
        x = inputs(B, T, Hk, H, dk, dv, dtype, seed=T, fixed=fixed, reset=reset)
        x[3] = x[3] * 0.03  # memories of a few hundred tokens
        check_all(x, torch.randn(B, T, H, dv, device=DEV).to(dtype), torch.randn(B, H, dk, dv, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_environments_of_several_chunks(dtype):
    x = inputs(500, 70, 1, 2, 32, 48, dtype)
    check_all(x, torch.randn(500, 70, 2, 48, device=DEV).to(dtype))


@pytest.mark.parametrize("dk,dv", [(64, 64), (1, 1), (7, 13), (16, 32), (32, 32), (40, 24), (33, 64), (64, 9), (128, 64)])
@pytest.mark.parametrize("T", [1, 2, 7, 15, 16, 17, 31, 32])
def test_short_rollouts_of_many_environments(T, dk, dv):
    """A warp a head."""
    for i, (Hk, H, fixed, reset, initial, d_final) in enumerate([(1, 1, True, None, False, False), (2, 2, False, 0.1, True, False),
                                                                (1, 3, True, 0.2, True, False), (1, 2, False, None, False, True)]):
        B = (700, 311, 200, 300)[i]
        x = inputs(B, T, Hk, H, dk, dv, torch.bfloat16, seed=T + i, fixed=fixed, reset=reset, initial=initial)
        check_all(x, torch.randn(B, T, H, dv, device=DEV).bfloat16(), torch.randn(B, H, dk, dv, device=DEV) if d_final else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [5, 350])
def test_strides(B, dtype):
    """Time-major buffers, heads out of a packed projection, rows that are not 16-byte aligned, a last axis that is not
    contiguous: the same results as of contiguous copies, bit for bit."""
    T, H, d = 40 if B == 5 else 20, 2, 48
    base = inputs(B, T, H, H, d, d, dtype)
    d_out = torch.randn(B, T, H, d, device=DEV).to(dtype)
    want = gradients(zeno_b200.linear_attention, base, d_out)
    packed = torch.stack(base[:3], 2)  # [B, T, 3, H, d]
    wide = torch.cat([torch.zeros(B, T, H, 3, device=DEV, dtype=dtype), base[0], torch.zeros(B, T, H, 2, device=DEV, dtype=dtype)], -1)
    time_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in base[:5]] + [base[5]]
    variants = [time_major, [packed[:, :, 0], packed[:, :, 1], packed[:, :, 2], *base[3:]], [wide[..., 3:3 + d], *base[1:]],
                [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in base[:3]] + base[3:],
                [*base[:4], base[4].bool(), base[5].transpose(2, 3).contiguous().transpose(2, 3)]]
    for x in variants:
        for grad in (d_out, d_out.transpose(0, 1).contiguous().transpose(0, 1), d_out.mT.contiguous().mT):
            for a, b in zip(gradients(zeno_b200.linear_attention, x, grad), want):
                assert torch.equal(a, b)
    # a gradient that is broadcast, as sum() hands it back
    check_all(base, torch.ones((), device=DEV, dtype=dtype).expand(B, T, H, d))


def test_broadcast_inputs():
    """Decays and keys that are expanded: the gradients of what they were expanded from are the sums."""
    B, T, H, d = 3, 50, 4, 32
    x = inputs(B, T, H, H, d, d, torch.float32, fixed=True)
    k = torch.randn(B, 1, H, d, device=DEV, requires_grad=True)
    g = x[3].clone().requires_grad_(True)
    d_out = torch.randn(B, T, H, d, device=DEV)
    got = torch.autograd.grad(zeno_b200.linear_attention(x[0], k.expand(B, T, H, d), x[2], g, x[4], x[5])[0], (k, g), d_out)
    per_token = torch.autograd.grad(zeno_b200.linear_attention(x[0], k.expand(B, T, H, d), x[2], g.expand(B, T, H), x[4], x[5])[0], (k, g), d_out)
    want = torch.autograd.grad(plain.linear_attention(x[0], k.expand(B, T, H, d), x[2], g, x[4], x[5])[0], (k, g), d_out.double())
    for a, b, c in zip(got, per_token, want):
        check(a, c), check(b, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ends_of_the_decays(dtype):
    """Decays of nothing, to nothing and growing ones; each token its own episode; resets at both ends."""
    B, T, H, d = 4, 100, 1, 32
    d_out = torch.randn(B, T, H, d, device=DEV).to(dtype)
    for name in ("none", "minus infinity", "far", "growing", "mixed", "all reset", "ends"):
        x = inputs(B, T, H, H, d, d, dtype, reset=None)
        if name == "none":
            x[3] = torch.zeros_like(x[3])
        if name == "minus infinity":
            x[3][:, ::7] = -float("inf")
        if name == "far":
            x[3] = x[3] * 1000
        if name == "growing":
            x[3] = x[3] * -0.1
        if name == "mixed":  # one decay far larger than the others, whose sums would lose them
            x[3] = x[3] * 0.01
            x[3][:, 5::31] = -80.0
        x[4] = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
        if name == "all reset":
            x[4][:] = 1
        if name == "ends":
            x[4][:, 0] = x[4][:, -1] = 1
            x[4][:, 31] = x[4][:, 64] = 255
        check_all(x, d_out, torch.randn(B, H, d, d, device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_and_small_values(dtype):
    """Nothing is scaled: results follow the inputs' powers of two exactly."""
    x = inputs(2, 70, 1, 1, 32, 32, dtype)
    d_out = torch.randn(2, 70, 1, 32, device=DEV).to(dtype)
    base = gradients(zeno_b200.linear_attention, x, d_out)
    for e in (-40, 40):
        s = 2.0 ** e
        y = [x[0] / s, x[1] / s, x[2] * s, x[3], x[4], x[5].clone()]
        got = gradients(zeno_b200.linear_attention, y, d_out)
        for name, a, b, f in zip(NAMES, got, base, (1 / s, 1, 1, 1, 1 / s / s, 1 / s, 1 / s)):
            if name in ("state", "d_initial", "d_q", "out"):  # of these the initial state is a part that does not follow
                continue
            check(a / f, b, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name,value", [("q", "nan"), ("k", "nan"), ("k", "-inf"), ("v", "inf"), ("v", "nan"), ("g", "nan"), ("d_out", "nan"), ("d_out", "inf")])
@pytest.mark.parametrize("B,T,resets,bad_at", [(2, 70, (20, 45), 30), (2, 70, (20, 32), 40), (2, 33, (32,), 32), (2, 900, (300, 500), 310), (2, 20, (7,), 3),
                                               (300, 20, (7,), 3), (300, 32, (5, 20), 20), (300, 32, (5, 20), 10)])
@pytest.mark.parametrize("fixed,d", [(False, 32), (True, 32), (False, 128), (True, 100)])
def test_what_is_not_finite_stays_in_its_episode(B, T, resets, bad_at, fixed, d, name, value, dtype):
    H = 2
    if d > 64 and (B > 2 or dtype == torch.float32):
        return  # (the wide instances of bfloat16)
    x = inputs(B, T, H, H, d, d, dtype, reset=None, fixed=fixed)
    if fixed and name == "g":
        return  # (then it is in every episode)
    x[4] = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
    for r in resets:
        x[4][:, r] = 1
    d_out = torch.randn(B, T, H, d, device=DEV).to(dtype)
    want = exact(x, d_out)
    y = [t.clone() for t in x]
    z = d_out.clone()
    bad = z if name == "d_out" else y["qkvg".index(name)]
    if name == "g":
        bad[0, bad_at, 1] = float(value)
    else:
        bad[0, bad_at, 1, 5] = float(value)
    got = gradients(zeno_b200.linear_attention, y, z)
    first = max([0, *(r for r in resets if r <= bad_at)])
    last = min([T, *(r for r in resets if r > bad_at)])
    outside = [t for t in range(T) if not first <= t < last]
    assert outside
    for what, a, b in zip(NAMES, got, want):
        if fixed and what == "d_g":
            check(a[0], b[0], what)  # (the other head's)
            continue
        if what in ("state", "d_initial"):
            episode = last == T if what == "state" else first == 0
            pick = [(slice(1, B), slice(None)), (slice(0, 1), slice(0, 1))] + ([] if episode else [(slice(0, 1), slice(1, 2))])
            for p in pick:
                check(a[p], b[p], what)
            continue
        check(a[1:], b[1:], what)
        check(a[0, :, 0], b[0, :, 0], what)
        check(a[0, outside, 1], b[0, outside, 1], what)
    if name != "d_out":  # and what comes before it in its episode
        check(got[0][0, first:bad_at, 1], want[0][0, first:bad_at, 1]) if bad_at > first else None
        # (the decay of an episode's first token is not looked at)
        assert torch.isfinite(got[0][0, bad_at, 1]).all() == (name == "g" and bad_at in resets)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,w", [(3, 40, 16), (600, 30, 48), (3, 200, 128)])
def test_a_dropped_state_may_hold_anything(B, T, w, dtype):
    x = inputs(B, T, 1, 1, w, w, dtype, reset=None)
    x[4] = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
    x[4][:, 0] = 1
    d = torch.randn(B, T, 1, w, device=DEV).to(dtype)
    want = exact(x, d)
    x[5][:] = float("nan")
    for a, b in zip(gradients(zeno_b200.linear_attention, x, d), want):
        check(a, b)
    state = x[5].clone()
    out = zeno_b200.linear_attention_step(*(t[:, 0] for t in x[:4]), state, x[4][:, 0])
    check(out, want[0][:, 0])
    assert torch.isfinite(state).all()


def test_gradients_against_differences():
    """The 32-bit gradients along random directions against central differences of the 64-bit result.  The function is of third
    degree along a direction in q, k, v and the state, and smooth in g: steps of 1e-3 leave 1e-6 of it."""
    x = inputs(2, 75, 1, 2, 24, 20, torch.float32, seed=3)
    d_out, d_final = torch.randn(2, 75, 2, 20, device=DEV), torch.randn(2, 2, 24, 20, device=DEV)
    got = gradients(zeno_b200.linear_attention, x, d_out, d_final)[2:]

    def loss(y):
        out, final = plain.linear_attention(*y)
        return (out * d_out.double()).sum() + (final * d_final.double()).sum()
    places = [0, 1, 2, 3, 5]
    for at, grad in zip(places, got):
        torch.manual_seed(at)
        for _ in range(3):
            way = torch.randn_like(x[at]).double()
            y = [t.double() if t is not None and t.is_floating_point() else t for t in x]
            e = 1e-4
            y[at] = x[at].double() + e * way
            up = loss(y)
            y[at] = x[at].double() - e * way
            slope = (up - loss(y)) / (2 * e)
            scale = grad.double().norm() * way.norm() / way.numel() ** 0.5
            assert abs(float((grad.double() * way).sum() - slope)) <= 1e-5 * float(scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,Hk,H,dk,dv", [(1, 4, 4, 64, 64), (3, 1, 2, 16, 16), (5, 2, 4, 33, 30), (700, 1, 1, 128, 64), (1300, 1, 2, 20, 8), (2400, 1, 1, 7, 50),
                                          (2400, 1, 1, 16, 127), (2, 1, 1, 1, 1)])
def test_step(B, Hk, H, dk, dv, dtype):
    for fixed, with_reset in ((True, False), (False, True)):
        x = inputs(B, 3, Hk, H, dk, dv, dtype, fixed=fixed, reset=0.3 if with_reset else None)
        want, last = plain.linear_attention(*x)
        state = x[5].clone()
        version = state._version
        for t in range(3):
            out = zeno_b200.linear_attention_step(*(y[:, t] for y in x[:3]), x[3] if fixed else x[3][:, t], state, x[4][:, t] if with_reset else None)
            check(out, want[:, t], t)
        check(state, last)
        assert state._version > version


def test_step_is_the_rollout():
    """A memory that acted token by token is the memory of the rollout."""
    x = inputs(6, 40, 2, 2, 24, 24, torch.float32)
    out, last = zeno_b200.linear_attention(*x)
    state = x[5].clone()
    acted = torch.stack([zeno_b200.linear_attention_step(*(y[:, t] for y in x[:4]), state, x[4][:, t]) for t in range(40)], 1)
    check(acted, out), check(state, last)


def test_step_state_seen_by_autograd():
    x = inputs(2, 8, 1, 1, 16, 16, torch.float32)
    q = x[0].clone().requires_grad_(True)
    out, _ = zeno_b200.linear_attention(q, *x[1:])
    zeno_b200.linear_attention_step(*(y[:, 0] for y in x[:4]), x[5])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    with torch.inference_mode():
        zeno_b200.linear_attention_step(*(y[:, 0] for y in x[:4]), x[5].clone())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_empty(dtype):
    x = inputs(2, 0, 1, 1, 16, 16, dtype)
    got = gradients(zeno_b200.linear_attention, x, torch.zeros(2, 0, 1, 16, device=DEV, dtype=dtype), torch.ones(2, 1, 16, 16, device=DEV))
    assert got[0].shape == (2, 0, 1, 16) and torch.equal(got[1], x[5]) and torch.equal(got[-1], torch.ones_like(x[5]))
    x = inputs(2, 0, 1, 1, 16, 16, dtype, initial=False, fixed=True)
    got = gradients(zeno_b200.linear_attention, x, torch.zeros(2, 0, 1, 16, device=DEV, dtype=dtype))
    assert not got[1].any() and not got[5].any()
    x = inputs(0, 5, 1, 2, 16, 16, dtype, fixed=True)
    got = gradients(zeno_b200.linear_attention, x, torch.zeros(0, 5, 2, 16, device=DEV, dtype=dtype))
    assert got[0].shape == (0, 5, 2, 16) and got[1].shape == (0, 2, 16, 16) and not got[5].any()
    assert zeno_b200.linear_attention_step(x[0][:, 0], x[1][:, 0], x[2][:, 0], x[3], x[5]).shape == (0, 2, 16)


@pytest.mark.parametrize("d,T,B", [(128, 300, 2), (128, 64, 40), (100, 700, 1)])
@pytest.mark.parametrize("fixed", [False, True])
@pytest.mark.parametrize("Hk,H", [(2, 2), (1, 3)])
def test_wide_heads(Hk, H, fixed, B, T, d):
    """tcgen05: whole and padded widths, segments and none, shared heads, with and without what lies in front and behind."""
    for initial, behind in ((True, True), (False, False), (True, False)):
        x = inputs(B, T, Hk, H, d, d, torch.bfloat16, seed=T, fixed=fixed, reset=0.02, initial=initial)
        check_all(x, torch.randn(B, T, H, d, device=DEV).bfloat16(), torch.randn(B, H, d, d, device=DEV) if behind else None)


def test_products_that_are_not_waited_for_are_not_a_number():
    """A block that gives up on its products writes NaN, in every result, and the next call is as before."""
    from zeno_b200._ffi import _lib
    x = inputs(2, 300, 1, 2, 128, 128, torch.bfloat16, fixed=True)
    d = torch.randn(2, 300, 2, 128, device=DEV).bfloat16()
    want = gradients(zeno_b200.linear_attention, x, d)
    before = _lib.zeno_linear_attention_wait_limit(0)
    try:
        got = gradients(zeno_b200.linear_attention, x, d)
        torch.cuda.synchronize()
    finally:
        assert _lib.zeno_linear_attention_wait_limit(before) == 0
    assert before == 2000000000
    for t in got:
        assert torch.isnan(t).all()
    for a, b in zip(gradients(zeno_b200.linear_attention, x, d), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B,T,w,dtype", [(1, 1500, 128, torch.bfloat16), (1, 1500, 32, torch.float32), (700, 20, 64, torch.bfloat16), (3, 50, 40, torch.float32)])
def test_the_final_state_in_place_of_the_initial_one(B, T, w, dtype):
    """At the C entry, which allows it: rollouts in segments, by warps and by blocks."""
    from zeno_b200._ffi import _lib, ffi
    x = inputs(B, T, 1, 1, w, w, dtype, fixed=True, reset=0.001)
    out, final = zeno_b200.linear_attention(*x)

    def tensor(t):
        s = t.stride()
        return dict(data=ffi.cast("void*", t.data_ptr()), stride=[s[0], s[1], s[2] if len(s) > 2 else 0])
    p = ffi.new("ZenoLinearAttention*")
    p.batch, p.tokens, p.key_heads, p.value_heads, p.key_dim, p.value_dim = B, T, 1, 1, w, w
    p.dtype, p.scale = int(dtype == torch.bfloat16), w ** -0.5
    p.q, p.k, p.v, p.reset = (tensor(x[i]) for i in (0, 1, 2, 4))
    p.g = dict(data=ffi.cast("void*", x[3].data_ptr()), stride=[0, 0, 1])
    got, state = torch.empty_like(out), x[5].clone()
    p.out = tensor(got)
    p.initial_state = p.final_state = ffi.cast("float*", state.data_ptr())
    need = _lib.zeno_linear_attention_workspace_bytes(p, 0)
    work = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    stream = ffi.cast("void*", torch.cuda.current_stream().cuda_stream)
    assert _lib.zeno_linear_attention_forward(p, ffi.cast("void*", work.data_ptr()), need, stream) == 0
    assert torch.equal(got, out) and torch.equal(state, final)


def test_second_derivatives_are_refused():
    x = inputs(2, 5, 1, 1, 16, 16, torch.float32)
    q = x[0].clone().requires_grad_(True)
    out, _ = zeno_b200.linear_attention(q, *x[1:])
    once, = torch.autograd.grad(out.sum(), q, create_graph=True)
    check(once, exact([q.detach(), *x[1:]], torch.ones_like(out))[2])
    with pytest.raises(RuntimeError, match="once"):
        once.sum().backward()


def test_growing_decays_of_any_size():
    """exp(g) past what a float holds: what is infinite or not a number stays in its episode."""
    x = inputs(2, 70, 1, 1, 16, 16, torch.float32, reset=None)
    x[4] = torch.zeros(2, 70, device=DEV, dtype=torch.uint8)
    x[4][:, 40] = 1
    want = exact(x, torch.zeros(2, 70, 1, 16, device=DEV))[0]
    for value in (100.0, 1e4, 1e9, float("inf")):
        y = [t.clone() for t in x]
        y[3][:, 20] = value
        got = zeno_b200.linear_attention(*y)[0]
        check(got[:, :20], want[:, :20]), check(got[:, 40:], want[:, 40:])
        assert not torch.isfinite(got[:, 20:40]).any()


def test_repeats_bit_for_bit():
    for x in (inputs(3, 300, 1, 2, 128, 128, torch.bfloat16, fixed=True), inputs(700, 30, 1, 2, 64, 64, torch.bfloat16), inputs(9, 200, 1, 2, 64, 64, torch.bfloat16, fixed=True), inputs(1, 900, 1, 1, 64, 64, torch.float32)):
        d = torch.randn(x[2].shape, device=DEV).to(x[2].dtype)
        first = gradients(zeno_b200.linear_attention, x, d)
        for _ in range(3):
            for a, b in zip(gradients(zeno_b200.linear_attention, x, d), first):
                assert torch.equal(a, b)


def test_partial_gradients():
    """Leaves that want no gradient, a loss of the final state alone, a constant state."""
    x = inputs(2, 50, 1, 2, 16, 24, torch.float32)
    want = exact(x, torch.zeros(2, 50, 2, 24, device=DEV), torch.ones(2, 2, 16, 24, device=DEV))
    k = x[1].clone().requires_grad_(True)
    _, final = zeno_b200.linear_attention(x[0], k, *x[2:])
    check(torch.autograd.grad(final.sum(), k)[0], want[3])
    g = x[3].clone().requires_grad_(True)
    _, final = zeno_b200.linear_attention(*x[:3], g, *x[4:])
    check(torch.autograd.grad(final.sum(), g)[0], want[5])


def test_in_a_cuda_graph():
    """Two graphs whose calls share a memory pool, replayed in turn on new inputs, forward and backward."""
    make = [lambda s: inputs(5, 300, 1, 2, 64, 64, torch.bfloat16, seed=s, fixed=True), lambda s: inputs(1, 700, 1, 1, 32, 32, torch.float32, seed=s)]
    pool, graphs = None, []
    for f in make:
        x = f(1)
        d = torch.randn(x[2].shape, device=DEV).to(x[2].dtype)
        want = gradients(zeno_b200.linear_attention, x, d)
        still = [t.clone() for t in f(2)]

        def work():
            state = still[5].clone()
            out = zeno_b200.linear_attention_step(*(t[:, 0] for t in still[:3]), still[3] if still[3].dim() == 1 else still[3][:, 0], state, still[4][:, 0])
            return gradients(zeno_b200.linear_attention, still, d) + [out, state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            got = work()
        pool = graph.pool()
        graphs.append((graph, still, x, got, want, d))
    for _ in range(2):
        for graph, still, x, got, want, _ in graphs:
            for a, b in zip(still, x):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_on_another_stream():
    x = inputs(3, 300, 1, 1, 64, 64, torch.bfloat16)
    d = torch.randn(x[2].shape, device=DEV).to(torch.bfloat16)
    want = gradients(zeno_b200.linear_attention, x, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gradients(zeno_b200.linear_attention, x, d)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_offsets_that_pass_32_bits():
    """Buffers and states of more than 2^32 bytes, and strides that reach past 2^31 elements."""
    B, H, d = 70000, 2, 128
    state = torch.zeros((B, H, d, d), device=DEV)  # 2.3e9 elements
    x = inputs(B, 1, H, H, d, d, torch.bfloat16, initial=False, reset=None)
    out = zeno_b200.linear_attention_step(x[0][:, 0], x[1][:, 0], x[2][:, 0], x[3][:, 0], state)
    tail = [y[-3:] for y in x[:4]]
    want, last = plain.linear_attention(*tail)
    check(out[-3:], want[:, 0]), check(state[-3:], last)
    out, final = zeno_b200.linear_attention(*x)
    check(out[-3:], want), check(final[-3:], last)
    del state, final, out
    big = torch.empty(2 ** 31 + 2 ** 20, device=DEV, dtype=torch.bfloat16)
    q = big.as_strided((2, 20, 1, 16), (2 ** 31, 16, 16, 1))
    x = inputs(2, 20, 1, 1, 16, 16, torch.bfloat16)
    q.copy_(x[0])
    d_out = torch.randn(2, 20, 1, 16, device=DEV).to(torch.bfloat16)
    want = gradients(zeno_b200.linear_attention, x, d_out)
    x[0] = q
    with torch.no_grad():
        assert torch.equal(zeno_b200.linear_attention(*x)[0], want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_environments_than_one_axis_of_a_grid(dtype):
    x = inputs(70001, 40, 1, 1, 8, 8, dtype)
    part = [t[-5:] for t in x]
    d = torch.randn(70001, 40, 1, 8, device=DEV).to(dtype)
    got, want = gradients(zeno_b200.linear_attention, x, d), exact(part, d[-5:])
    for name, a, b in zip(NAMES, got, want):
        check(a[-5:], b, name)


def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad
    x = inputs(1, 4, 1, 1, 8, 8, torch.float32)
    with forward_ad.dual_level():
        q = forward_ad.make_dual(x[0], torch.ones_like(x[0]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            zeno_b200.linear_attention(q, *x[1:])


def test_refusals():
    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device=DEV)
    q, v, g = t(2, 3, 2, 8), t(2, 3, 4, 16), t(2, 3, 4)
    f = zeno_b200.linear_attention
    f(q, q, v, g), f(q, q, v, t(4))
    for args, error, match in [
            ((q, t(2, 3, 2, 9), v, g), ValueError, "k must have shape"), ((q, q.bfloat16(), v, g), TypeError, "k must be"),
            ((q.half(), q.half(), v.half(), g), TypeError, "float32 or bfloat16"), ((q, q, v, g.bfloat16()), TypeError, "g must be"),
            ((q, q, v, t(2)), ValueError, "g must have shape"), ((q, q, v, t(2, 3)), ValueError, "g must have shape"),
            ((t(2, 3, 3, 8), t(2, 3, 3, 8), v, g), ValueError, "multiple"), ((t(2, 3, 2, 136), t(2, 3, 2, 136), v, g), ValueError, "widths"),
            ((q, q, v, g, t(2, 4, dtype=torch.uint8)), ValueError, "reset must have shape"), ((q, q, v, g, t(2, 3)), TypeError, "reset must be"),
            ((q, q, v, g, None, t(2, 4, 16, 8)), ValueError, "initial_state must have shape"), ((q[0], q[0], v[0], g[0]), ValueError, "batch, tokens, heads"),
            ((q, q.cpu(), v, g), ValueError, "on cpu"), ((q, q, v, g.cpu()), ValueError, "on cpu")]:
        with pytest.raises(error, match=match):
            f(*args)
    step = zeno_b200.linear_attention_step
    one = (q[:, 0], q[:, 0], v[:, 0], g[:, 0])
    with pytest.raises(ValueError, match="contiguous"):
        step(*one, t(2, 4, 16, 8).mT)
    with pytest.raises(TypeError, match="state must be"):
        step(*one, t(2, 4, 8, 16, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="no gradients"):
        step(*one, t(2, 4, 8, 16).requires_grad_(True))


def test_sizes_beyond_the_entries_are_refused():
    """Before anything is allocated: such sizes would not pass the entries' 32-bit fields."""
    x, g = torch.zeros(1, 1, 1, 1, device=DEV), torch.zeros(1, device=DEV)
    state = torch.zeros(1, 1, 1, 1, device=DEV)
    for shape in ((2 ** 32 + 1, 1, 1, 1), (2 ** 27 + 1, 1, 1, 1), (1, 2 ** 32 + 1, 1, 1), (1, 2 ** 30 + 1, 1, 1), (1, 1, 2 ** 32 + 1, 1), (1, 1, 65536, 1)):
        big = x.expand(shape)
        with pytest.raises(ValueError, match="at most 65535 value heads"):
            zeno_b200.linear_attention(big, big, big, g.expand(shape[2]))
        if shape[1] == 1:
            with pytest.raises(ValueError, match="at most 65535 value heads"):
                zeno_b200.linear_attention_step(big[:, 0], big[:, 0], big[:, 0], g.expand(shape[2]), state.expand(shape[0], shape[2], 1, 1))
