"""Inputs at the ends of their ranges, and what torch expects of an operator, for the policy operators.

Tolerances where nothing else is said are those of test_operators_gpu.py."""
import pytest
import torch

import zeno_b200
from zeno_b200._ffi import _lib, ffi
import operators_plain as plain
from test_operators_gpu import DEV, check, check_forward, check_gradients, gradients, inputs, matrix

pytestmark = pytest.mark.gpu


# bfloat16 updates.  32-bit work is 2e-5 off the 64-bit result at most (1.6e-4 where most directions are empty, as
# test_operators_gpu.py derives); an error e of a value takes its rounding to the neighbour in e / ulp of the cases, so
# that the squares of the differences add to e ulp, with an ulp of 2^-7 of the value at most: sqrt(2e-5 * 2^-7) = 4e-4 and
# sqrt(1.6e-4 * 2^-7) = 1.2e-3 against the 64-bit result rounded to bfloat16.
@pytest.mark.parametrize("shape", [(64, 29), (128, 512), (129, 300), (200, 513), (512, 1024), (3, 260, 140), (1100, 700)])
def test_orthogonalize_bfloat16_as_32_bits_rounded_once(shape):
    m = matrix(shape, torch.bfloat16, seed=1)
    assert plain.off(zeno_b200.orthogonalize(m), plain.orthogonalize(m).bfloat16()) <= 4e-4


@pytest.mark.parametrize("shape", [(60, 90), (200, 300), (512, 1024), (700, 150)])
def test_orthogonalize_bfloat16_of_low_rank(shape):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    left, right = (torch.randint(-1, 2, s, generator=gen, device=DEV).float() for s in ((shape[0], 4), (4, shape[1])))
    m = (left @ right).bfloat16()  # whole numbers up to 4: of rank 4 to the last bit
    assert plain.off(zeno_b200.orthogonalize(m), plain.orthogonalize(m).bfloat16()) <= 1.2e-3


def c_step(x, initial, final, out, tokens):
    """zeno_delta_rule_step on [batch, tokens, ...] tensors; None: no data."""
    q, k, v, g, beta, reset = x
    p = ffi.new("ZenoDeltaRule*")
    p.batch, p.tokens, p.key_heads, p.key_dim, p.value_heads, p.value_dim = q.shape[0], tokens, *q.shape[2:], *v.shape[2:]
    p.dtype, p.normalize, p.scale = int(q.dtype == torch.bfloat16), 1, q.shape[3] ** -0.5
    for name, t in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta), ("reset", reset), ("out", out)):
        if t is not None and tokens:
            getattr(p, name).data = ffi.cast("void*", t.data_ptr())
            getattr(p, name).stride = (list(t.stride()) + [0])[:3]
    if reset is not None:
        p.reset.data = ffi.cast("void*", reset.data_ptr())
    p.initial_state, p.final_state = (ffi.cast("float*", 0 if t is None else t.data_ptr()) for t in (initial, final))
    assert _lib.zeno_delta_rule_step(p, ffi.cast("void*", torch.cuda.current_stream().cuda_stream)) == 0


@pytest.mark.parametrize("dk,dv", [(16, 16), (33, 30), (128, 64)])
def test_step_of_no_tokens_keeps_the_state(dk, dv):
    q, k, v, g, beta, _, state = inputs(3, 1, 1, 2, dk, dv, torch.float32)
    marks = torch.ones((3, 1), dtype=torch.uint8, device=DEV)  # of the token that is not there
    keep, final = state.clone(), torch.full_like(state, 7.0)
    c_step((q, k, v, g, beta, marks), state, state, v, 0)
    c_step((q, k, v, g, beta, marks), state, final, v, 0)
    assert torch.equal(state, keep) and torch.equal(final, keep)
    c_step((q, k, v, g, beta, marks), None, final, v, 0)
    assert not final.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hk,H,dk,dv", [(3, 2, 1, 2, 16, 16), (2, 41, 2, 4, 33, 30), (140, 7, 1, 1, 128, 64)])
def test_step_of_several_tokens(B, T, Hk, H, dk, dv, dtype):
    *x, state = inputs(B, T, Hk, H, dk, dv, dtype, reset=0.2)
    want, after = plain.delta_rule(*x, state)
    out, final = torch.empty_like(x[2]), torch.empty_like(state)
    c_step(x, state, final, out, T)
    check(out, want, dtype, "out")
    check(final, after, torch.float32, "state")
    c_step(x, state, state, out, T)
    assert torch.equal(state, final)
    c_step(x, None, final, out, T)
    want, after = plain.delta_rule(*x)
    check(out, want, dtype, "out from nothing")
    check(final, after, torch.float32, "state from nothing")


def test_backward_after_a_step_on_its_initial_state_is_refused():
    q, k, v, g, beta, _, state = inputs(3, 5, 1, 2, 16, 16, torch.float32)
    leaf = v.clone().requires_grad_(True)
    out, _ = zeno_b200.delta_rule(q, k, leaf, g, beta, None, state)
    before = state._version
    zeno_b200.delta_rule_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state)
    assert state._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_step_in_inference_mode():
    with torch.inference_mode():
        q, k, v, g, beta, _, state = inputs(3, 1, 1, 2, 16, 16, torch.float32)
        want, after = plain.delta_rule(q, k, v, g, beta, None, state)
        args = (q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0])
        check(zeno_b200.delta_rule_step(*args, state), want[:, 0], torch.float32, "out")
        check(state, after, torch.float32, "state")
    zeno_b200.delta_rule_step(*args, state)  # a state made there, used outside


HUGE = [(3, 1e17), (9, 1e19), (20, 1e22), (21, 1e30), (40, 3e37)]  # squares that leave 32 bits from 1.8e19 on


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_squares_overflow(dtype):
    x = list(inputs(2, 70, 1, 2, 64, 48, dtype, seed=4, reset=0.03))
    for t, f in HUGE:
        x[0][:, t] *= f
        x[1][:, t + 1] *= f
    out, final = zeno_b200.delta_rule(*x)
    want, state = plain.delta_rule(*x)
    check(out, want, dtype, "out")
    check(final, state, torch.float32, "state")
    s = x[6].clone()
    for t in range(70):
        check(zeno_b200.delta_rule_step(*(y[:, t] for y in x[:5]), s, x[5][:, t]), want[:, t], dtype, "step %d" % t)
    check(s, state, torch.float32, "state of the steps")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_rows_whose_squares_overflow(dtype):
    x = list(inputs(2, 70, 1, 2, 64, 48, dtype, seed=4, reset=0.03))
    x[0], x[1] = x[0] * 1e30, x[1] * 1e25  # all of them, so that their own gradients (of 1e-30) are seen
    d_out, d_fin = torch.randn_like(x[2]), torch.randn((2, 2, 64, 48), device=DEV)
    got = gradients(zeno_b200.delta_rule, x, d_out, d_fin)
    want = gradients(plain.delta_rule, [t.double() if t.is_floating_point() else t for t in x], d_out, d_fin)
    for name, a, b in zip(["q", "k", "v", "g", "beta", "initial"], got, want):
        check(a, b, a.dtype, "d_" + name)


@pytest.mark.parametrize("steps", [1, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(100, 290), (700, 130), (3, 260, 140)])
def test_orthogonalize_that_gives_up_is_not_a_number(shape, dtype, steps):
    m = matrix(shape, dtype)
    want = zeno_b200.orthogonalize(m, steps)
    assert torch.isfinite(want).all()
    before = _lib.zeno_orthogonalize_wait_limit(0)  # no product waits for anything
    try:
        got = zeno_b200.orthogonalize(m, steps)
        torch.cuda.synchronize()
    finally:
        assert _lib.zeno_orthogonalize_wait_limit(before) == 0
    assert before == 2_000_000_000
    assert torch.isnan(got).all()
    assert torch.equal(zeno_b200.orthogonalize(m, steps), want)


def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad
    q, k, v, g, beta, _, state = inputs(2, 3, 1, 1, 8, 8, torch.float32)
    with forward_ad.dual_level():
        for i in range(6):
            x = [q, k, v, g, beta, state]
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                zeno_b200.delta_rule(*x[:5], None, x[5])
            one = [y[:, 0] for y in x[:5]]
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                zeno_b200.delta_rule_step(*one, x[5])
        with pytest.raises(RuntimeError, match="forward-mode"):
            zeno_b200.orthogonalize(forward_ad.make_dual(state[0, 0], state[1, 0]))
        zeno_b200.delta_rule(q, k, v, g, beta, None, state)  # none of these has a tangent
        zeno_b200.orthogonalize(state)


# 2e-5 as at other widths: what a sum of n terms loses may not grow with n
@pytest.mark.parametrize("shape", [(70, 4200), (70, 20000), (130, 262144), (300000, 33), (4300, 4400)])
def test_orthogonalize_long_sums(shape):
    m = matrix(shape, torch.float32, seed=2)
    assert plain.off(zeno_b200.orthogonalize(m), plain.orthogonalize(m)) <= 2e-5


@pytest.mark.parametrize("steps", [1, 2])
def test_orthogonalize_long_sums_of_one_and_two_steps(steps):
    for shape in [(4300, 4400), (8, 9000)]:
        m = matrix(shape, torch.float32, seed=2)
        assert plain.off(zeno_b200.orthogonalize(m, steps), plain.orthogonalize(m, steps)) <= 2e-5


@pytest.mark.parametrize("shape", [(30, 40), (90, 150)])
@pytest.mark.parametrize("size", [1e-21, 1e-23, 1e-26, 1e-30, 1e-36])
def test_orthogonalize_of_next_to_nothing(size, shape):
    m = matrix(shape, torch.float32) * size
    want = plain.orthogonalize(m)
    got = zeno_b200.orthogonalize(m)
    assert got.any() and plain.off(got * 2.0 ** 40, want * 2.0 ** 40) <= 2e-5


@pytest.mark.parametrize("B,T,Hk,H,dk,dv,dtype", [(600, 100, 1, 2, 32, 32, torch.float32), (300, 130, 2, 2, 64, 64, torch.bfloat16),
                                                  (5000, 33, 1, 1, 16, 16, torch.bfloat16)])
def test_many_environments_of_several_chunks(B, T, Hk, H, dk, dv, dtype):
    x = inputs(B, T, Hk, H, dk, dv, dtype, seed=T, reset=0.02)
    check_forward(x, dtype)
    check_gradients(x, dtype)


def test_in_a_cuda_graph():
    x = [inputs(5, 300, 1, 2, 64, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    d = [torch.randn_like(x[0][2]), torch.randn_like(x[0][6])]
    m = [matrix((2, 200, 300), torch.float32, seed=s) for s in (1, 2)]
    small = [matrix((3, 40, 300), torch.float32, seed=s) for s in (1, 2)]

    def work(x, m, small):
        state = x[6].clone()
        out = zeno_b200.delta_rule_step(*(t[:, 0] for t in x[:5]), state, x[5][:, 0])
        return [out, state, *gradients(zeno_b200.delta_rule, x, *d), zeno_b200.orthogonalize(m), zeno_b200.orthogonalize(small)]
    want = work(x[1], m[1], small[1])
    still = [[t.clone() for t in x[0]], m[0].clone(), small[0].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(*still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(*still)
    for a, b in zip([*still[0], still[1], still[2]], [*x[1], m[1], small[1]]):
        a.copy_(b)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_threads_with_streams_of_their_own():
    import threading
    x = [inputs(6, 200, 1, 2, 64, 64, torch.bfloat16, seed=s) for s in range(4)]
    m = [matrix((2, 150, 200), torch.float32, seed=s) for s in range(4)]

    def work(i):
        d = torch.ones_like(x[i][2]), torch.ones_like(x[i][6])
        return [*zeno_b200.delta_rule(*x[i]), *gradients(zeno_b200.delta_rule, x[i], *d), zeno_b200.orthogonalize(m[i])]
    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    got, wrong = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = work(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # seen by the test, not lost in the thread
            wrong.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_muon_is_momentum_orthogonalised():
    from zeno_b200.policy import Muon
    shapes = [(20, 70), (300, 90), (3, 40, 50), (17,)]
    params = [torch.zeros(s, device=DEV, requires_grad=True) for s in shapes]
    optimiser = Muon(params, lr=0.1, momentum=0.9)
    plain_params, moments = [[torch.zeros(s, device=DEV, dtype=torch.float64) for s in shapes] for _ in range(2)]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(7)
    for _ in range(2):
        for p, want, mom in zip(params, plain_params, moments):
            p.grad = torch.randn(p.shape, generator=gen, device=DEV)
            mom.mul_(0.9).add_(p.grad)
            update = p.grad.double() + 0.9 * mom
            if p.dim() > 1:
                update = plain.orthogonalize(update) * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
            want.sub_(0.1 * update)
        optimiser.step()
    for p, want in zip(params, plain_params):
        assert plain.off(p, want) <= 4e-5  # two orthogonalised updates


def test_offsets_that_pass_32_bits():
    """Rows of one buffer of 5 GB, the environments' 1.2e9 elements apart."""
    x = list(inputs(3, 40, 1, 2, 32, 16, torch.bfloat16))
    far = torch.zeros(2_500_000_000, dtype=torch.bfloat16, device=DEV)
    at, y = 0, list(x)
    for i in range(3):
        s = list(x[i].stride())
        s[0] = 1_200_000_000
        y[i] = torch.as_strided(far, x[i].shape, s, at)
        y[i].copy_(x[i])
        at += x[i][0].numel()
    for a, b in zip(zeno_b200.delta_rule(*y), zeno_b200.delta_rule(*x)):
        assert torch.equal(a, b)
    d = torch.ones_like(x[2]), torch.ones_like(x[6])
    want = gradients(zeno_b200.delta_rule, x, *d)
    leaves = [t.detach().requires_grad_(True) if t.is_floating_point() else t for t in y]
    got = torch.autograd.grad(zeno_b200.delta_rule(*leaves), [t for t in leaves if t.requires_grad], d)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    states = x[6].clone(), x[6].clone()
    outs = [zeno_b200.delta_rule_step(*(t[:, 3] for t in z[:5]), s) for z, s in zip((x, y), states)]
    assert torch.equal(*outs) and torch.equal(*states)
    for shape in [(3, 20, 30), (3, 140, 150)]:
        m = matrix(shape, torch.bfloat16)
        wide = torch.as_strided(far, shape, (1_200_000_000, shape[2], 1))
        wide.copy_(m)
        assert torch.equal(zeno_b200.orthogonalize(wide), zeno_b200.orthogonalize(m))
        rows = torch.as_strided(far, shape[1:], (17_000_000, 1))
        rows.copy_(m[0])
        assert torch.equal(zeno_b200.orthogonalize(rows), zeno_b200.orthogonalize(m[0]))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("name,value", [("q", "nan"), ("q", "inf"), ("k", "nan"), ("k", "-inf"), ("v", "inf"), ("g", "nan"), ("beta", "nan")])
@pytest.mark.parametrize("T,resets,bad_at", [(70, (20, 45), 30), (70, (20, 32), 40), (33, (32,), 32), (900, (300, 500), 310)])
def test_gradients_outside_an_episode_that_is_not_finite(T, resets, bad_at, name, value, norm):
    x = list(inputs(2, T, 1, 2, 64, 40, torch.float32, reset=0.0, norm=norm))
    for t in resets:
        x[5][:, t] = 1
    d = torch.ones_like(x[2]), torch.ones_like(x[6])
    want = gradients(plain.delta_rule, [t.double() if t.is_floating_point() else t for t in x], *d, normalize=norm)
    i = "q k v g beta".split().index(name)
    x[i][0, bad_at, 0] = float(value)
    got = gradients(zeno_b200.delta_rule, x, *d, normalize=norm)
    begin = max((0, *(t for t in resets if t <= bad_at)))
    end = min((T, *(t for t in resets if t > bad_at)))
    for a, b in zip(got[:5], want[:5]):
        check(a[1], b[1], torch.float32, "another environment")
        check(a[0, end:], b[0, end:], torch.float32, "behind the episode")
        check(a[0, :begin], b[0, :begin], torch.float32, "in front of the episode")
    check(got[5], want[5], torch.float32, "d_initial")
