"""Linear attention where its parts meet: chunks within a segment of a long rollout, short rollouts of wide heads, results that are
asked for together, views.

Tolerances and the plain implementation are those of test_linear_attention_gpu.py."""
import pytest
import torch

import zeno_b200
from test_linear_attention_gpu import NAMES, TOL, check, check_all, exact, gradients, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bad", ["nan gate", "growing gates", "nan key", "inf value"])
@pytest.mark.parametrize("dtype,d,segment", [(torch.bfloat16, 64, 256), (torch.float32, 64, 224), (torch.bfloat16, 32, 224), (torch.bfloat16, 128, 512),
                                             (torch.bfloat16, 100, 512), (torch.float32, 128, 224)])
def test_a_reset_in_another_chunk_of_a_segment(dtype, d, segment, bad):
    """32 rollouts of 2000 tokens are cut into segments of several chunks.  In one of them an episode holds a gate that is not a number, gates whose
    product is past a float, or rows that are not finite, and a reset in a chunk in front of it and in one behind it ends that: every other
    episode, the state behind the rollout and the gradient of the one in front are what they are without it."""
    B, T, H = 16, 2000, 2
    begin, at, end = 2 * segment + 4, 2 * segment + 68, 2 * segment + 135  # three chunks of one segment, of 32 tokens or of 64
    assert end < 3 * segment
    x = inputs(B, T, H, H, d, d, dtype, reset=None)
    x[4] = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
    x[4][:, begin] = x[4][:, end] = 1
    d_out, d_final = torch.randn(B, T, H, d, device=DEV).to(dtype), torch.randn(B, H, d, d, device=DEV)
    two = [t[:2] for t in x]
    want = exact(two, d_out[:2], d_final[:2])
    y = [t.clone() for t in x]
    if bad == "nan gate":
        y[3][0, at, 1] = float("nan")
    elif bad == "growing gates":
        y[3][0, at:at + 24, 1] = 4.0  # exp(96)
    elif bad == "nan key":
        y[1][0, at, 1, 5] = float("nan")
    else:
        y[2][0, at, 1, 5] = float("inf")
    got = [t[:2] for t in gradients(zeno_b200.linear_attention, y, d_out, d_final)]
    outside = [t for t in range(T) if not begin <= t < end]
    for name, a, b in zip(NAMES, got, want):
        if name in ("state", "d_initial"):
            check(a, b, name)
            continue
        check(a[1], b[1], name), check(a[0, :, 0], b[0, :, 0], name)
        check(a[0, outside, 1], b[0, outside, 1], name)


def entry(t):
    """A tensor as the C entries take it: [B, T, heads, ...], or [B, T]."""
    from zeno_b200._ffi import ffi
    s = t.stride()
    return dict(data=ffi.cast("void*", t.data_ptr()), stride=[s[0], s[1], s[2] if len(s) > 2 else 0])


@pytest.mark.parametrize("B,T,Hk,H,d,dtype,infinite", [
    (300, 20, 2, 2, 64, torch.bfloat16, False), (300, 32, 1, 2, 40, torch.bfloat16, False), (300, 9, 2, 2, 128, torch.bfloat16, False),
    (300, 20, 2, 2, 32, torch.bfloat16, True), (2, 300, 2, 2, 128, torch.bfloat16, False), (40, 64, 1, 2, 100, torch.bfloat16, False),
    (3, 50, 1, 1, 40, torch.float32, False), (1, 900, 1, 2, 64, torch.bfloat16, False)])
def test_both_gradients_of_the_decays(B, T, Hk, H, d, dtype, infinite):
    """The C entry gives each token's gradient, their sum over batch and tokens, or both: by warps (`infinite`: element by element), on tcgen05, by blocks.
    The sum is one in 64 bits of the 32-bit gradients, rounded once (2^-24)."""
    from zeno_b200._ffi import _lib, ffi
    x = inputs(B, T, Hk, H, d, d, dtype, reset=0.05)
    if infinite:  # in every head, where it is masked from the gradients of the decays: a token that is its own episode
        x[4][:, 4:6] = 1
        x[0][:, 4, :, 3] = float("inf")
    d_out = torch.randn(B, T, H, d, device=DEV).to(dtype)
    p, grads = ffi.new("ZenoLinearAttention*"), ffi.new("ZenoLinearAttentionGrads*")
    p.batch, p.tokens, p.key_heads, p.value_heads, p.key_dim, p.value_dim = B, T, Hk, H, d, d
    p.dtype, p.scale = int(dtype == torch.bfloat16), d ** -0.5
    out, (d_q, d_k, d_v, d_g) = torch.empty_like(x[2]), [torch.empty_like(t) for t in x[:4]]
    d_decay = torch.full((H,), float("nan"), device=DEV)
    p.q, p.k, p.v, p.g, p.reset, p.out = (entry(t) for t in (*x[:5], out))
    p.initial_state = ffi.cast("float*", x[5].data_ptr())
    saved = torch.empty(max(1, _lib.zeno_linear_attention_saved_bytes(p) // 4), device=DEV)
    p.saved = ffi.cast("float*", saved.data_ptr())
    need = max(_lib.zeno_linear_attention_workspace_bytes(p, i) for i in (0, 1))
    work = torch.full((max(need // 4, 1),), float("nan"), device=DEV)
    at, stream = ffi.cast("void*", work.data_ptr()), ffi.cast("void*", torch.cuda.current_stream().cuda_stream)
    assert _lib.zeno_linear_attention_forward(p, at, need, stream) == 0
    grads.d_out, grads.d_q, grads.d_k, grads.d_v, grads.d_g = (entry(t) for t in (d_out, d_q, d_k, d_v, d_g))
    grads.d_decay = ffi.cast("float*", d_decay.data_ptr())
    work.fill_(float("nan"))
    assert _lib.zeno_linear_attention_backward(p, grads, at, need, stream) == 0
    want = gradients(zeno_b200.linear_attention, x, d_out)
    for a, b in zip((d_q, d_k, d_v, d_g), want[2:]):
        assert torch.equal(a, b) or infinite
    if infinite:
        return check_sum(d_decay, d_g, finite=torch.isfinite(d_g).all())
    check_sum(d_decay, d_g)
    grads.d_g.data = ffi.NULL  # the sum alone
    alone = torch.full((H,), float("nan"), device=DEV)
    grads.d_decay = ffi.cast("float*", alone.data_ptr())
    assert _lib.zeno_linear_attention_backward(p, grads, at, need, stream) == 0
    # (there a pair's term is counted once, times the tokens it passes: other roundings, at most 3.6e-6 of the terms)
    assert ((alone - d_decay).abs().double() <= 3.6e-6 * d_g.double().abs().sum((0, 1))).all()


def check_sum(d_decay, d_g, finite=True):
    assert finite
    terms = d_g.double()
    assert ((d_decay.double() - terms.sum((0, 1))).abs() <= 2.0 ** -24 * terms.sum((0, 1)).abs() + 2.0 ** -40 * terms.abs().sum((0, 1))).all()


def negative(t):
    """t's values in a view that is negative by its flag, as the imaginary part of a conjugate is."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_views_that_are_negative_by_a_flag():
    x = inputs(3, 40, 1, 2, 24, 20, torch.float32)
    d_out, d_final = torch.randn(3, 40, 2, 20, device=DEV), torch.randn(3, 2, 24, 20, device=DEV)
    want = gradients(zeno_b200.linear_attention, x, d_out, d_final)
    y = [negative(t) if t.is_floating_point() else t for t in x]
    leaves = [t.requires_grad_(True) if t.is_floating_point() else t for t in y]
    out, final = zeno_b200.linear_attention(*leaves)
    got = [out, final, *torch.autograd.grad([out, final], [t for t in leaves if t.requires_grad], [negative(d_out), negative(d_final)])]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with torch.no_grad():
        one = [t[:, 0] for t in x[:4]]
        state, other = x[5].clone(), x[5].clone()
        assert torch.equal(zeno_b200.linear_attention_step(*one, state), zeno_b200.linear_attention_step(*(negative(t) for t in one), other))
        assert torch.equal(state, other)
        with pytest.raises(ValueError, match="conjugated"):
            zeno_b200.linear_attention_step(*one, negative(x[5]))


@pytest.mark.parametrize("T", [1, 7, 16, 17, 32])
@pytest.mark.parametrize("dk,dv", [(128, 128), (100, 128), (128, 7)])
def test_short_rollouts_of_wide_heads(T, dk, dv):
    """A warp a head of whole and of padded width past 64 channels, with and without what lies in front and behind, shared heads."""
    for i, (B, Hk, H, fixed, reset, initial, behind) in enumerate([(600, 1, 1, True, None, False, False), (311, 2, 2, False, 0.1, True, False),
                                                                   (200, 1, 3, True, 0.2, True, False), (300, 1, 2, False, None, False, True)]):
        x = inputs(B, T, Hk, H, dk, dv, torch.bfloat16, seed=T + i, fixed=fixed, reset=reset, initial=initial)
        check_all(x, torch.randn(B, T, H, dv, device=DEV).bfloat16(), torch.randn(B, H, dk, dv, device=DEV) if behind else None)


BAD = [("q", "nan"), ("k", "-inf"), ("v", "inf"), ("v", "nan"), ("g", "nan"), ("d_out", "nan"), ("d_out", "inf")]


@pytest.mark.parametrize("name,value,fixed", [(*b, f) for b in BAD for f in (False, True) if not (f and b[0] == "g")])
@pytest.mark.parametrize("B,T,resets,at,d,dtype", [
    (300, 20, (7,), 3, 128, torch.bfloat16), (300, 32, (5, 20), 20, 100, torch.bfloat16), (300, 32, (5, 20), 10, 128, torch.bfloat16),
    (2, 70, (20, 45), 30, 128, torch.float32), (2, 900, (300, 500), 310, 100, torch.float32), (300, 20, (7,), 3, 128, torch.float32)])
def test_what_is_not_finite_in_wide_heads(B, T, resets, at, d, dtype, name, value, fixed):
    """By warps past 64 channels, and the wide instances of 32 bits: episodes on either side, the other head and the other environments are
    what they are without it.  (One decay for all tokens has a gradient with every episode in it: the other head's is looked at.)"""
    H = 2
    x = inputs(B, T, H, H, d, d, dtype, reset=None, fixed=fixed)
    x[4] = torch.zeros(B, T, device=DEV, dtype=torch.uint8)
    for r in resets:
        x[4][:, r] = 1
    d_out = torch.randn(B, T, H, d, device=DEV).to(dtype)
    want = exact(x, d_out)
    y, z = [t.clone() for t in x], d_out.clone()
    bad = z if name == "d_out" else y["qkvg".index(name)]
    bad[(0, at, 1) if name == "g" else (0, at, 1, 5)] = float(value)
    got = gradients(zeno_b200.linear_attention, y, z)
    first, last = max([0, *(r for r in resets if r <= at)]), min([T, *(r for r in resets if r > at)])
    outside = [t for t in range(T) if not first <= t < last]
    for what, a, b in zip(NAMES, got, want):
        if fixed and what == "d_g":
            terms = exact([*x[:3], x[3].expand(B, T, H), *x[4:]], d_out)[5]
            assert (a[0].double() - b[0].double()).abs() <= TOL * terms[..., 0].abs().sum()
            continue
        check(a[1:], b[1:], what), check(a[0, ..., 0, :, :] if what in ("state", "d_initial") else a[0, :, 0], b[0, ..., 0, :, :] if what in ("state", "d_initial") else b[0, :, 0], what)
        if what in ("state", "d_initial"):
            if not (last == T if what == "state" else first == 0):
                check(a[0, 1], b[0, 1], what)
            continue
        check(a[0, outside, 1], b[0, outside, 1], what)
    if name != "d_out":
        assert not torch.isfinite(got[0][0, at, 1]).all() or (name == "g" and at in resets)


def check_rounding(got, want, off):
    """A bfloat16 result is the rounding of a value within `off` of the exact one (all of one sign); a 32-bit one is within `off`."""
    if got.dtype == torch.float32:
        worst = float(((got.double() - want).abs() / want.abs()).max())
        assert worst <= off, worst
        return
    low, high = (want * (1 - off)).to(torch.bfloat16), (want * (1 + off)).to(torch.bfloat16)
    missed = (got < low) | (got > high)
    assert not missed.any(), float(missed.double().mean())


SHAPES = [(700, 20, 64, torch.bfloat16), (700, 7, 128, torch.bfloat16), (500, 70, 64, torch.bfloat16), (500, 50, 32, torch.bfloat16), (40, 100, 128, torch.bfloat16),
          (2, 400, 128, torch.bfloat16), (300, 40, 16, torch.float32), (1, 900, 16, torch.float32)]


@pytest.mark.parametrize("B,T,d,dtype", SHAPES)
def test_single_terms_to_their_limbs(B, T, d, dtype):
    """Each token its own episode, every value positive: out = scale (q . k) v is one term, and so are the gradients.  In a bfloat16 call q . k loses at most
    d / 16 truncations of 2^-23 and three roundings of 2^-24; then its limbs: of a value in [2^e, 2^(e+1)) the first, 8 bits, leaves at most 2^(e-8), of which the second,
    8 bits below 2^(e-8), leaves 2^(e-17); their two products are truncated once: (1 + 8 / 64 + 1 / 42 + 1 / 64) 2^-17 for 128 channels, 1.2 * 2^-17.  In a 32-bit call
    of 16 channels: one truncation, the rounding of the small terms' sum into it, of the scale and of the result, and twice the dropped products (2^-8 * 2^-17
    twice): 2.75 * 2^-23."""
    off = 1.2 * 2.0 ** -17 if dtype == torch.bfloat16 else 2.75 * 2.0 ** -23
    x = inputs(B, T, 1, 1, d, d, dtype, initial=False)
    x[:3] = [(t.float().abs() + 0.5).to(dtype) for t in x[:3]]
    x[4][:] = 1
    d_out = (torch.rand(B, T, 1, d, device=DEV) + 0.5).to(dtype)
    for a, b in zip(gradients(zeno_b200.linear_attention, x, d_out), exact(x, d_out)):
        if a.dim() == 4 and a.shape == x[0].shape:
            check_rounding(a, b, off)


@pytest.mark.parametrize("B,T,d,dtype", SHAPES)
def test_states_to_their_limbs(B, T, d, dtype):
    """Nothing but a positive state in front (keys of zero) or its gradient behind (no gradient of the outputs): out = scale c S^T q, dv = e R^T k.  As above, the limbs'
    products in 2 * 8 truncations, and what a state loses on its way through the chunks and by their decays, 2^-22 each."""
    off = 1.4 * 2.0 ** -17 + T / 32 * 2.0 ** -22 if dtype == torch.bfloat16 else (8 + T / 16) * 2.0 ** -23
    x = inputs(B, T, 1, 1, d, d, dtype, reset=None, fixed=True)
    x[3] = x[3] * 0.03
    x[0], x[2], x[5] = ((t.float().abs() + 0.5).to(t.dtype) for t in (x[0], x[2], x[5]))
    x[1] = torch.zeros_like(x[1])
    zero = torch.zeros(B, T, 1, d, device=DEV, dtype=dtype)
    check_rounding(zeno_b200.linear_attention(*x)[0], exact(x, zero)[0], off)
    x[1], x[5] = x[0].clone(), None
    behind = torch.rand(B, 1, d, d, device=DEV) + 0.5
    got, want = gradients(zeno_b200.linear_attention, x, zero, behind), exact(x, zero, behind)
    check_rounding(got[4], want[4], off)


def test_states_next_to_the_largest_float():
    """Their first limb would round to infinity."""
    for B, T, d, dtype in SHAPES:
        x = inputs(B, T, 1, 1, d, d, dtype, reset=None, fixed=True)
        x[1], x[3] = torch.zeros_like(x[1]), torch.zeros_like(x[3])
        x[0], x[5] = ((x[0].float().abs() + 0.5) * 2.0 ** -20).to(dtype), torch.full_like(x[5], 3.4e38)
        got = zeno_b200.linear_attention(*x)
        check_rounding(got[0], exact(x, torch.zeros_like(x[2]))[0], 1.4 * 2.0 ** -17 + T / 32 * 2.0 ** -22 if dtype == torch.bfloat16 else (8 + T / 16) * 2.0 ** -23)
        assert torch.equal(got[1], x[5])


@pytest.mark.parametrize("name", ["q", "k", "v", "d_out"])
@pytest.mark.parametrize("B,T,at,d,dtype", [(300, 20, 4, 64, torch.bfloat16), (300, 32, 31, 128, torch.bfloat16), (3, 60, 31, 32, torch.bfloat16), (3, 70, 9, 64, torch.bfloat16),
                                            (3, 200, 63, 128, torch.bfloat16), (3, 200, 64, 100, torch.bfloat16), (3, 70, 31, 40, torch.float32), (1, 900, 95, 16, torch.float32)])
def test_an_episode_of_one_token_has_no_part_in_the_decays(B, T, at, d, dtype, name):
    """Whatever it holds: one decay for all tokens of a head has the gradient of the other episodes."""
    x = inputs(B, T, 1, 2, d, d, dtype, fixed=True, reset=0.1)
    x[4][:, at] = 1
    if at + 1 < T:
        x[4][:, at + 1] = 1
    d_out = torch.randn(B, T, 2, d, device=DEV).to(dtype)
    want = gradients(zeno_b200.linear_attention, x, d_out)[5]
    y, z = [t.clone() for t in x], d_out.clone()
    bad = z if name == "d_out" else y["qkv".index(name)]
    bad[0, at, -1, 3] = float("inf")
    got = gradients(zeno_b200.linear_attention, y, z)[5]
    terms = exact([*x[:3], x[3].expand(B, T, 2), *x[4:]], d_out)[5]
    assert ((got - want).abs() <= TOL * terms.abs().sum((0, 1))).all()
