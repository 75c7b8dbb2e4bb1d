"""The policy operators (zeno_b200/operators.py) against 64-bit plain implementations.

Tolerances (2-norm of the error over that of the result).  32-bit results: operands are
split to 22 bits or kept in 32, sums are held in 32 bits over at most 160 terms
(2^-24 * 160 = 1e-5 if every rounding went the same way), so 2e-5 covers two products in
a row at their worst.  bfloat16 results: compared with the 64-bit result rounded to
bfloat16, from which an error of 2e-5 takes a value to its neighbour (2^-8 of it) in one of
a hundred cases: 2e-3 covers a third of all.
Newton-Schulz multiplies an error in a direction of a small singular value by up to 3.4445
in each step (485 in five) while the result's norm is that of the directions already at
one; 32 bits: 2e-5 as above for matrices whose small directions do not dominate; where all
but one direction is empty, 485 times the 2^-22 of a rounding in the first step and less in
the later ones (1 + 1/3.4 + ... = 1.4): 1.6e-4.  (64 bits on inputs moved by 2^-25 already
differ by 2e-5 there, 32-bit torch by 9e-5.)  bfloat16: 16-bit limbs inside (2^-12 a
rounding, three a step, amplified) and the last rounding: 5e-3."""
import pytest
import torch

import zeno_b200
import operators_plain as plain

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 2e-5, torch.bfloat16: 2e-3}
NS_TOL = {torch.float32: 2e-5, torch.bfloat16: 5e-3}
DEV = "cuda"


def inputs(B, T, Hk, H, dk, dv, dtype, seed=0, reset=0.1, initial=True, norm=True):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device=DEV)
    q, k, v = normal(B, T, Hk, dk).to(dtype), normal(B, T, Hk, dk).to(dtype), normal(B, T, H, dv).to(dtype)
    if not norm:
        q, k = q * 0.5, (k * dk ** -0.5 * 0.9).to(dtype)
    g = -torch.rand((B, T, H), generator=gen, device=DEV) * 0.3
    beta = torch.rand((B, T, H), generator=gen, device=DEV)
    r = (torch.rand((B, T), generator=gen, device=DEV) < reset).to(torch.uint8) if reset is not None else None
    return q, k, v, g, beta, r, (normal(B, H, dk, dv) if initial else None)


def check(got, want, dtype, what):
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), what
    want = want.to(got.dtype)
    assert plain.off(got, want) <= TOL[dtype], (what, plain.off(got, want))


def check_forward(x, dtype, **kw):
    out, final = zeno_b200.delta_rule(*x, **kw)
    want, state = plain.delta_rule(*x, **kw)
    assert out.dtype == dtype and final.dtype == torch.float32
    check(out, want, dtype, "out")
    check(final, state, torch.float32, "state")


def gradients(f, x, d_out, d_final, **kw):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None and t.is_floating_point() else t for t in x]
    out, final = f(*leaves, **kw)
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    return torch.autograd.grad((out, final), wanted, (d_out.to(out.dtype), d_final.to(final.dtype)))


def check_gradients(x, dtype, d_final=True, **kw):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(99)
    q, _, v = x[:3]
    d_out = (1e-3 * torch.randn(v.shape, generator=gen, device=DEV)).to(dtype)
    d_fin = 1e-3 * torch.randn((v.shape[0], v.shape[2], q.shape[3], v.shape[3]), generator=gen, device=DEV)
    if not d_final:
        d_fin = torch.zeros_like(d_fin)
    got = gradients(zeno_b200.delta_rule, x, d_out, d_fin, **kw)
    want = gradients(plain.delta_rule, [None if t is None else t.double() if t.is_floating_point() else t for t in x], d_out, d_fin, **kw)
    names = ["q", "k", "v", "g", "beta", "initial"]
    for name, a, b in zip(names, got, want):
        # the gates' gradients are differences of sums: held to the size of what is summed, which the
        # gradients of v and q share; 32 bits throughout
        check(a, b, a.dtype, "d_" + name)
    return got


TOKENS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 257]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", TOKENS)
def test_lengths(T, dtype):
    x = inputs(3, T, 2, 2, 64, 64, dtype, seed=T)
    check_forward(x, dtype)
    check_gradients(x, dtype)


WIDTHS = [(8, 8), (16, 128), (24, 40), (32, 32), (33, 31), (63, 65), (64, 128), (65, 16), (72, 72), (100, 56), (128, 24), (127, 127),
          (128, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
def test_widths(dk, dv, dtype):
    x = inputs(2, 70, 1, 2, dk, dv, dtype, seed=dk)
    check_forward(x, dtype)
    check_gradients(x, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_width_one(dtype):
    # a normalised row of width 1 has no gradient to compare (its norm takes it away)
    x = inputs(3, 40, 1, 1, 1, 1, dtype, norm=False)
    check_forward(x, dtype, normalize=False, scale=1.0)
    check_gradients(x, dtype, normalize=False, scale=1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hk,H", [(1, 1), (1, 5), (2, 6), (3, 3), (4, 8)])
def test_shared_heads(Hk, H, dtype):
    x = inputs(2, 45, Hk, H, 48, 32, dtype, seed=H)
    check_forward(x, dtype)
    check_gradients(x, dtype, d_final=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_not_normalised_and_scale(dtype):
    x = inputs(2, 75, 2, 2, 64, 64, dtype, norm=False)
    check_forward(x, dtype, normalize=False, scale=0.3)
    check_gradients(x, dtype, normalize=False, scale=0.3)


# few long rollouts, which are split over the tokens
LONG = [(1, 1000, 1, 2, 64, 64, 0.01, True), (1, 4099, 1, 1, 128, 128, 0.001, True), (1, 777, 1, 1, 40, 24, 0.0, False),
        (1, 1025, 1, 1, 33, 100, 0.003, True), (2, 600, 1, 2, 128, 32, None, True), (5, 288, 1, 2, 16, 16, 0.005, True)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hk,H,dk,dv,reset,initial", LONG)
def test_long(B, T, Hk, H, dk, dv, reset, initial, dtype):
    x = inputs(B, T, Hk, H, dk, dv, dtype, seed=T, reset=reset, initial=initial)
    check_forward(x, dtype)
    check_gradients(x, dtype)


def test_long_with_an_episode_that_is_not_finite():
    x = list(inputs(1, 1200, 1, 1, 32, 32, torch.float32, reset=0.0))
    for t in (300, 700):
        x[5][:, t] = 1
    d_out, d_fin = torch.ones_like(x[2]), torch.ones((1, 1, 32, 32), device=DEV)
    want, state = plain.delta_rule(*x)
    grads = gradients(plain.delta_rule, [t.double() if t.is_floating_point() else t for t in x], d_out, d_fin)
    x[2][0, 400, 0, 5] = float("nan")
    out, final = zeno_b200.delta_rule(*x)
    got = gradients(zeno_b200.delta_rule, x, d_out, d_fin)
    check(final, state, torch.float32, "state")
    for part in (slice(0, 400), slice(700, 1200)):
        check(out[:, part], want[:, part], torch.float32, "outside the episode")
    for a, b in zip(got[:5], grads[:5]):
        for part in (slice(0, 300), slice(700, 1200)):
            check(a[:, part], b[:, part], torch.float32, "gradients outside the episode")
    check(got[5], grads[5], torch.float32, "d_initial")


@pytest.mark.parametrize("reset", [None, 0.0, 0.3, 1.0])
@pytest.mark.parametrize("initial", [False, True])
def test_episodes(reset, initial):
    x = inputs(4, 67, 2, 2, 32, 32, torch.float32, reset=reset, initial=initial)
    check_forward(x, torch.float32)
    got = check_gradients(x, torch.float32)
    if reset == 1.0 and initial:  # nothing of the initial state is ever read
        assert not got[5].any()


def test_reset_as_bool_and_at_every_position():
    for at in range(0, 34):
        x = list(inputs(1, 34, 1, 1, 16, 16, torch.float32, reset=0.0))
        x[5][0, at] = 1
        check_forward(x, torch.float32)
        y = list(x)
        y[5] = x[5].bool()
        for a, b in zip(zeno_b200.delta_rule(*x), zeno_b200.delta_rule(*y)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min, -1e4, -200.0])
def test_decay_to_nothing_is_a_reset(low):
    x = list(inputs(2, 70, 1, 2, 32, 32, torch.float32, reset=0.0))
    for t in (0, 7, 31, 32, 50, 69):
        x[3][:, t] = low
    check_forward(x, torch.float32)
    got = check_gradients(x, torch.float32)
    assert not got[3][:, [0, 7, 31, 32, 50, 69]].any()


def test_long_strong_decays_keep_the_later_ones():
    x = list(inputs(2, 96, 1, 1, 32, 32, torch.float32, reset=0.0))
    x[3][:, :60] -= 50.0  # sums of -3000 in front of decays of -0.1
    check_forward(x, torch.float32)
    check_gradients(x, torch.float32)


def test_extreme_gates_and_zero_rows():
    x = list(inputs(2, 70, 2, 2, 64, 64, torch.float32, reset=0.0))
    x[4][:, ::3] = 0.0      # nothing written
    x[4][:, 1::3] = 1.0
    x[3][:, ::2] = 0.0      # no decay
    x[0][:, 5] = 0.0
    x[1][:, 9:20] = 0.0     # keys of length zero
    x[2][:, 30] = 0.0
    check_forward(x, torch.float32)
    check_gradients(x, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", [False, True])
def test_tiny_and_empty_rows(norm, dtype):
    x = list(inputs(2, 70, 2, 2, 64, 64, dtype, norm=norm))
    for t, f in [(3, 0.0), (20, 1e-4), (21, 1e-9), (40, 1e-12), (50, 0.0), (66, 1e-6)]:
        x[0][:, t] *= f
        x[1][:, t + 2] *= f
    check_forward(x, dtype, normalize=norm)
    check_gradients(x, dtype, normalize=norm)
    x[0][:] = 0
    check_gradients(x, dtype, normalize=norm)
    x[1][:] = 0
    check_gradients(x, dtype, normalize=norm)


@pytest.mark.parametrize("size", [1e-15, 1e-3, 1e6, 1e15])
def test_magnitudes(size):
    x = list(inputs(2, 50, 1, 2, 64, 64, torch.float32))
    x[2] = x[2] * size
    x[6] = x[6] * size
    check_forward(x, torch.float32)
    check_gradients(x, torch.float32)


def test_rows_of_very_different_magnitude():
    x = list(inputs(2, 50, 1, 2, 64, 64, torch.float32))
    f = torch.logspace(-6, 6, 50, device=DEV)[torch.randperm(50, generator=torch.Generator().manual_seed(1)).to(DEV)]
    x[0], x[1] = x[0] * f[None, :, None, None], x[1] * f.flip(0)[None, :, None, None]
    check_forward(x, torch.float32)
    got = check_gradients([t if i > 1 else t for i, t in enumerate(x)], torch.float32)
    assert all(torch.isfinite(t).all() for t in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    x = inputs(5, 37, 2, 4, 40, 24, dtype)
    want = zeno_b200.delta_rule(*x)
    grads = gradients(zeno_b200.delta_rule, x, want[0], want[1])

    def same(y):
        for a, b in zip(zeno_b200.delta_rule(*y), want):
            assert torch.equal(a, b)
        leaves = [t.detach().requires_grad_(True) if t is not None and t.is_floating_point() else t for t in y]
        out, final = zeno_b200.delta_rule(*leaves)
        got = torch.autograd.grad((out, final), [t for t in leaves if t is not None and t.requires_grad], want)
        for a, b in zip(got, grads):
            assert torch.equal(a, b)

    def time_major(t):
        return t if t is None or t.dim() == 4 and t.shape[1] != 37 else t.transpose(0, 1).contiguous().transpose(0, 1)
    same([time_major(t) if i < 6 else t for i, t in enumerate(x)])

    def odd_offset(t):  # rows that start at odd elements, and gaps between them
        if t is None:
            return t
        big = torch.zeros((*t.shape[:-1], t.shape[-1] + 3), dtype=t.dtype, device=DEV)
        big[..., 1:-2] = t
        return big[..., 1:-2]
    same([odd_offset(t) if i < 6 else t for i, t in enumerate(x)])
    same([t.mT.contiguous().mT if i < 3 else t for i, t in enumerate(x)])  # last axis not contiguous: copied
    heads_first = [t.permute(2, 0, 1, *range(3, t.dim())).contiguous().permute(1, 2, 0, *range(3, t.dim())) if i < 5 else t
                   for i, t in enumerate(x)]
    same(heads_first)


def test_broadcast_inputs_and_their_gradients():
    q, k, v, g, beta, r, s0 = inputs(3, 40, 2, 2, 32, 32, torch.float32)
    one = torch.rand((1, 1, 2), device=DEV, requires_grad=True)
    shared = torch.randn((1, 40, 2, 32), device=DEV, requires_grad=True)
    learned = torch.randn((1, 2, 32, 32), device=DEV, requires_grad=True)
    out, final = zeno_b200.delta_rule(shared.expand(3, -1, -1, -1), k, v, g, one.expand(3, 40, 2), r, learned.expand(3, -1, -1, -1))
    want, state = plain.delta_rule(shared.expand(3, -1, -1, -1), k, v, g, one.expand(3, 40, 2), r, learned.expand(3, -1, -1, -1))
    d = torch.randn_like(out)
    got = torch.autograd.grad(out, (one, shared, learned), d)
    ref = torch.autograd.grad(want, (one, shared, learned), d.double())
    for a, b in zip(got, ref):
        check(a, b, torch.float32, "broadcast")


def test_unused_outputs():
    x = inputs(2, 40, 1, 1, 32, 32, torch.float32)
    leaves = [t.clone().requires_grad_(True) if t is not None and t.is_floating_point() else t for t in x]
    ref = [t.detach().double().requires_grad_(True) if t is not None and t.is_floating_point() else t for t in x]
    _, final = zeno_b200.delta_rule(*leaves)
    _, want = plain.delta_rule(*ref)
    pick = [1, 2, 3, 4, 6]
    for a, b in zip(torch.autograd.grad(final.sum(), [leaves[i] for i in pick]), torch.autograd.grad(want.sum(), [ref[i] for i in pick])):
        check(a, b, torch.float32, "through the state alone")


def test_gradient_against_differences():
    x = list(inputs(2, 45, 1, 2, 32, 24, torch.float32))
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    d_out = torch.randn(x[2].shape, generator=gen, device=DEV)
    d_fin = torch.randn(x[6].shape, generator=gen, device=DEV)
    got = gradients(zeno_b200.delta_rule, x, d_out, d_fin)
    at = [0, 1, 2, 3, 4, 6]
    for i, grad in zip(at, got):
        way = torch.randn(x[i].shape, generator=gen, device=DEV).double()
        h = 1e-5  # 64-bit central differences: error h^2 = 1e-10 and 2^-53 / h = 1e-11 of the sums
        side = []
        for s in (h, -h):
            y = [None if t is None else t.double() if t.is_floating_point() else t for t in x]
            y[i] = y[i] + s * way
            out, final = plain.delta_rule(*y)
            side.append((out * d_out).sum() + (final * d_fin).sum())
        slope = float((side[0] - side[1]) / (2 * h))
        # the kernel's gradient is 2e-5 off in norm at most, and so is its product with a direction
        assert abs(float((grad.double() * way).sum()) - slope) <= 2e-5 * float(grad.double().norm() * way.norm()) + 1e-7 * abs(slope)


def test_value_that_is_not_finite_stays_in_its_episode():
    for bad_at, name in [(3, "v"), (12, "k"), (20, "q"), (33, "v"), (5, "g"), (6, "beta"), (2, "state")]:
        x = list(inputs(2, 70, 1, 1, 32, 32, torch.float32, reset=0.0))
        for t in (10, 25, 40, 64):
            x[5][:, t] = 1
        clean = plain.delta_rule(*x)
        y = [None if t is None else t.clone() for t in x]
        if name == "state":
            y[6][0] = float("nan")
            bad_at = 0
        else:
            y[{"q": 0, "k": 1, "v": 2, "g": 3, "beta": 4}[name]][0, bad_at] = float("nan")
        out, final = zeno_b200.delta_rule(*y)
        ends = [t for t in (10, 25, 40, 64, 70) if t > bad_at]
        # other environments, earlier tokens and later episodes have their values
        assert plain.off(out[1], clean[0][1]) <= 2e-5 and plain.off(out[0, :bad_at], clean[0][0, :bad_at]) <= 2e-5
        assert plain.off(out[0, ends[0]:], clean[0][0, ends[0]:]) <= 2e-5
        assert plain.off(final, clean[1]) <= 2e-5
        touched = out[0, bad_at] if name == "q" else out[0, bad_at:ends[0]]
        assert torch.isnan(touched).all()
        if name == "q":
            assert plain.off(out[0, bad_at + 1:], clean[0][0, bad_at + 1:]) <= 2e-5


def test_gradients_beside_an_episode_that_is_not_finite():
    x = list(inputs(1, 70, 1, 1, 32, 32, torch.float32, reset=0.0))
    for t in (20, 45):
        x[5][:, t] = 1
    d_out, d_fin = torch.ones_like(x[2]), torch.zeros((1, 1, 32, 32), device=DEV)
    clean = gradients(plain.delta_rule, [t.double() if t.is_floating_point() else t for t in x], d_out, d_fin)
    x[2][0, 30] = float("inf")
    got = gradients(zeno_b200.delta_rule, x, d_out, d_fin)
    for a, b in zip(got[:5], clean[:5]):
        for part in (slice(0, 20), slice(45, 70)):
            check(a[:, part], b[:, part], torch.float32, "outside the episode")


def test_empty():
    for B, T in [(0, 5), (3, 0), (0, 0)]:
        x = inputs(B, T, 1, 2, 16, 8, torch.float32)
        out, final = zeno_b200.delta_rule(*x)
        assert out.shape == (B, T, 2, 8) and torch.equal(final, x[6])
        got = gradients(zeno_b200.delta_rule, x, out, torch.ones_like(final))
        assert torch.equal(got[5], torch.ones_like(final))
    assert zeno_b200.orthogonalize(torch.zeros((0, 4, 5), device=DEV)).shape == (0, 4, 5)
    assert zeno_b200.orthogonalize(torch.zeros((3, 0, 5), device=DEV)).shape == (3, 0, 5)


def test_repeats_bit_for_bit_and_on_another_stream():
    x = inputs(7, 90, 2, 4, 64, 64, torch.bfloat16)
    d = torch.randn_like(x[2]), torch.randn((7, 4, 64, 64), device=DEV)
    first = [*zeno_b200.delta_rule(*x), *gradients(zeno_b200.delta_rule, x, *d)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = [*zeno_b200.delta_rule(*x), *gradients(zeno_b200.delta_rule, x, *d)]
        other = zeno_b200.orthogonalize(x[6].reshape(-1, 64, 64))
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    assert torch.equal(other, zeno_b200.orthogonalize(x[6].reshape(-1, 64, 64)))


def test_outside_autograd_is_the_same():
    x = inputs(2, 90, 1, 2, 64, 32, torch.bfloat16)
    y = [t.clone().requires_grad_(True) if t is not None and t.is_floating_point() else t for t in x]
    for a, b in zip(zeno_b200.delta_rule(*x), zeno_b200.delta_rule(*y)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,Hk,H,dk,dv", [(1, 1, 1, 1, 1), (3, 1, 3, 7, 5), (5, 2, 2, 16, 128), (4, 2, 4, 33, 30), (9, 3, 3, 64, 64),
                                          (130, 1, 2, 128, 128), (2, 1, 1, 100, 17), (3, 1, 2, 32, 36)])
def test_step(B, Hk, H, dk, dv, dtype):
    norm = dk > 1
    q, k, v, g, beta, r, s0 = inputs(B, 6, Hk, H, dk, dv, dtype, reset=0.3, norm=norm)
    want, state = plain.delta_rule(q, k, v, g, beta, r, s0, normalize=norm)
    s = s0.clone()
    for t in range(6):
        out = zeno_b200.delta_rule_step(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], s, r[:, t], normalize=norm)
        check(out, want[:, t], dtype, "step %d" % t)
    check(s, state, torch.float32, "state")


def test_step_clears_what_is_not_finite():
    q, k, v, g, beta, _, s = inputs(4, 1, 1, 2, 32, 32, torch.float32)
    s[1], s[2, 1, 3, 4] = float("nan"), float("inf")
    r = torch.tensor([0, 1, 1, 0], dtype=torch.uint8, device=DEV)
    clean = torch.where(torch.isfinite(s), s, torch.zeros_like(s))
    want, state = plain.delta_rule(q, k, v, g, beta, r[:, None], clean)
    out = zeno_b200.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], s, r)
    check(out, want[:, 0], torch.float32, "out")
    check(s, state, torch.float32, "state")


def test_step_on_a_slice_of_a_larger_state():
    q, k, v, g, beta, r, s0 = inputs(3, 1, 1, 1, 20, 12, torch.float32)
    big = torch.zeros(3 * 20 * 12 + 1, device=DEV)  # a state that is not aligned to 16 bytes
    s = big[1:].view(3, 1, 20, 12)
    s.copy_(s0)
    want, state = plain.delta_rule(q, k, v, g, beta, r, s0)
    check(zeno_b200.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], s, r[:, 0]), want[:, 0], torch.float32, "out")
    check(s, state, torch.float32, "state")
    assert big[0] == 0


def matrix(shape, dtype, seed=0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return (0.02 * torch.randn(shape, generator=gen, device=DEV)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (29, 64), (64, 29), (64, 64), (65, 100), (127, 129), (128, 512), (200, 513),
                                   (300, 100), (512, 512), (3, 64, 80), (2, 2, 40, 130), (5, 260, 140), (1100, 700),
                                   (3, 20, 257), (2, 64, 512), (64, 513), (900, 33), (2, 17, 2049), (40, 4096), (50, 4100)])
def test_orthogonalize(shape, dtype):
    m = matrix(shape, dtype)
    got = zeno_b200.orthogonalize(m)
    assert got.dtype == dtype and got.is_contiguous() and got.shape == m.shape and torch.isfinite(got).all()
    assert plain.off(got, plain.orthogonalize(m)) <= NS_TOL[dtype]


@pytest.mark.parametrize("steps", [0, 1, 2, 8])
def test_orthogonalize_steps(steps):
    m = matrix((70, 90), torch.float32)
    assert plain.off(zeno_b200.orthogonalize(m, steps), plain.orthogonalize(m, steps)) <= 2e-5 * max(1.0, 3.4445 ** (steps - 5))


@pytest.mark.parametrize("size", [1e-18, 1e-6, 1e6, 1e18])
def test_orthogonalize_magnitudes(size):
    m = matrix((90, 150), torch.float32) * size
    assert plain.off(zeno_b200.orthogonalize(m), plain.orthogonalize(m)) <= 2e-5


def test_orthogonalize_strides_zero_and_rank_one():
    m = matrix((3, 80, 130), torch.float32)
    want = zeno_b200.orthogonalize(m)
    assert torch.equal(zeno_b200.orthogonalize(m.mT.contiguous().mT), want)
    big = torch.zeros((3, 81, 133), device=DEV)
    big[:, 1:, 2:-1] = m
    assert torch.equal(zeno_b200.orthogonalize(big[:, 1:, 2:-1]), want)
    assert torch.equal(zeno_b200.orthogonalize(m[1]), want[1])
    assert plain.off(zeno_b200.orthogonalize(m.mT), want.mT) <= 2e-5
    assert not zeno_b200.orthogonalize(torch.zeros((50, 60), device=DEV)).any()
    flat = m[0, :1].T @ m[0, :1] * 30
    assert plain.off(zeno_b200.orthogonalize(flat), plain.orthogonalize(flat)) <= 485 * 2 ** -22 * 1.4
    eye = torch.eye(200, device=DEV)
    assert plain.off(zeno_b200.orthogonalize(eye), plain.orthogonalize(eye)) <= 2e-5


def test_orthogonalize_keeps_matrices_apart():
    m = matrix((4, 60, 70), torch.float32)
    want = zeno_b200.orthogonalize(m)
    m[1, 3, 4] = float("nan")
    m[2] *= 1e10
    got = zeno_b200.orthogonalize(m)
    assert torch.isnan(got[1]).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3]) and plain.off(got[2], want[2]) <= 2e-5
