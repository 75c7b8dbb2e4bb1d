"""layer_norm (zeno_b200/operators.py) against a 64-bit plain implementation.

Tolerances (2-norm of the error over that of the result).  32-bit results are sums held in 32 bits with about ten roundings
each on the way of a value (mean, difference, square root, division, product, sum) and log2 of the row's length in the sums: 32 of 2^-24, 1.9e-6.  Sums over
rows add up to 128 values in a row in a register before they meet others: twice that.  bfloat16 results: half a step of
the result's own rounding (2^-8 of the value) more, element by element: eight times the 32-bit figure covers the largest of some 10^5 errors.  The gradient of x is a difference, rstd (dh - mean(dh) - xhat mean(dh xhat)), each part of
which is rounded at 2^-24 of rstd dh: where next to nothing is left (two values a row: both are one spread from the mean whatever they
are) the error is that of the parts, so it is counted against the larger of the two norms."""
import pytest
import torch

import zeno_b200
import memory_plain as plain
from operators_plain import off

pytestmark = pytest.mark.gpu
TOL = 1.9e-6
DEV = "cuda"


def inputs(shape, dtype, affine, seed=0, mean=0.5):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    x = torch.randn(shape, generator=gen, device=DEV) + mean
    w, b = (torch.randn(shape[-1:], generator=gen, device=DEV) for _ in range(2))
    return x.to(dtype), None if affine is None else w.to(affine), None if affine is None else b.to(affine), torch.randn(shape, generator=gen, device=DEV).to(dtype)


def gradients(f, x, w, b, dy, **kw):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = f(*leaves, **kw)
    return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(y.dtype))]


def exact(x, w, b, dy, **kw):
    return gradients(plain.layer_norm, *(None if t is None else t.double() for t in (x, w, b)), dy, **kw)


def check(got, want, times=1, parts=0.0):
    """``parts``: the 2-norm of what the result is a difference of."""
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    norm = float(want.double().norm())
    size = max(norm or 1.0, parts)
    if got.dtype == torch.float32:
        assert off(got, want) * (norm or 1.0) <= times * TOL * size, off(got, want)
    else:
        error = (got.double() - want.double()).abs() - 2.0 ** -8 * want.double().abs()
        assert float(error.max()) <= 8 * times * TOL * size / want.numel() ** 0.5, float(error.max())


def parts_of(x, w, dy, eps=1e-5):
    """The 2-norm of rstd dh."""
    rstd = (x.double().var(-1, correction=0, keepdim=True) + eps).rsqrt()
    return float((rstd * dy.double() * (1.0 if w is None else w.double())).norm())


def check_all(x, w, b, dy, **kw):
    got = gradients(zeno_b200.layer_norm, x, w, b, dy, **kw)
    want = exact(x, w, b, dy, **kw)
    for i, (a, c) in enumerate(zip(got, want)):
        assert a.dtype == (x, x, w, b)[i].dtype
        check(a, c, 2 if i > 1 else 1, parts_of(x, w, dy) if i == 1 else 0.0)
    assert torch.equal(zeno_b200.layer_norm(x, w, b, **kw), got[0])


TYPES = [(torch.float32, None), (torch.float32, torch.float32), (torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)]


@pytest.mark.parametrize("dtype,affine", TYPES)
@pytest.mark.parametrize("width", [2, 3, 4, 5, 8, 16, 29, 31, 32, 33, 64, 65, 100, 128, 129, 250, 256, 257, 511, 512, 513, 516, 520, 777, 1000, 1024, 2048, 4099, 8191,
                                   8192, 8193, 8200, 20000])
def test_widths(width, dtype, affine):
    for rows in (1, 3, 37):
        check_all(*inputs((rows, width), dtype, affine, seed=width + rows), eps=1e-5)


@pytest.mark.parametrize("dtype,affine", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 256), (5000, 64), (30000, 29), (7001, 256), (700, 1030), (400, 4096), (160, 9000), (3000, 1), (2000, 500)])
def test_rows(rows, width, dtype, affine):
    x, w, b, dy = inputs((rows, width), dtype, affine, seed=rows)
    if width == 1:  # nothing but the bias is left
        y = gradients(zeno_b200.layer_norm, x, w, b, dy)
        assert torch.equal(y[0], torch.zeros_like(x) if b is None else b.expand(rows, 1).to(dtype)) and not y[1].any()
        return
    check_all(x, w, b, dy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Views, bit for bit as of a contiguous copy: time-major, a slice of channels, heads, rows out of alignment, a last axis that is not contiguous,
    more axes than three, a single row."""
    for width in (48, 50):
        a, b, c = 6, 7, 4
        x, w, bias, dy = inputs((a, b, c, width), dtype, torch.float32)
        want = gradients(zeno_b200.layer_norm, x, w, bias, dy)
        wide = torch.cat([x, x], -1)
        odd = torch.cat([torch.zeros(a, b, c, 3, device=DEV, dtype=dtype), x], -1)
        big = torch.zeros(2 * a, b, 3 * c, width, device=DEV, dtype=dtype)
        big[::2, :, ::3] = x
        views = [x, x.transpose(0, 1).contiguous().transpose(0, 1), x.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3), wide[..., width:], odd[..., 3:],
                 big[::2, :, ::3], x.mT.contiguous().mT]
        grads = [dy, dy.transpose(0, 1).contiguous().transpose(0, 1), dy.mT.contiguous().mT]
        for v in views:
            for d in grads:
                got = gradients(zeno_b200.layer_norm, v, w, bias, d)
                if v is views[4]:  # not aligned to 16 bytes: another instance, whose sums run in another order
                    for i, t in enumerate(exact(x, w, bias, dy)):
                        check(got[i], t, 2 if i > 1 else 1, parts_of(x, w, dy) if i == 1 else 0.0)
                    continue
                for p, q in zip(got, want):
                    assert torch.equal(p, q)
        assert zeno_b200.layer_norm(views[1], w, bias).stride() == views[1].stride()
        got = gradients(zeno_b200.layer_norm, x.view(2, 3, b, 2, 2, width), w, bias, dy.view(2, 3, b, 2, 2, width))
        for p, q in zip(got, want):
            assert torch.equal(p.reshape(q.shape), q)
        assert torch.equal(zeno_b200.layer_norm(x[1, 2, 3], w, bias), want[0][1, 2, 3])
        wide_w = torch.stack([w, bias], 1)
        assert torch.equal(zeno_b200.layer_norm(x, wide_w[:, 0], wide_w[:, 1]), want[0])
        off4 = torch.cat([torch.zeros(1, device=DEV), w])[1:]  # a weight that is not 16-byte aligned
        check(zeno_b200.layer_norm(x, off4, bias), plain.layer_norm(x, w, bias))


def test_broadcast_rows():
    """An input that is expanded, and a gradient that is."""
    x, w, b, dy = inputs((5, 1, 64), torch.float32, torch.float32)
    leaf = x.clone().requires_grad_(True)
    y = zeno_b200.layer_norm(leaf.expand(5, 9, 64), w, b)
    got = torch.autograd.grad(y, leaf, dy.expand(5, 9, 64))[0]
    leaf64 = x.double().requires_grad_(True)
    want = torch.autograd.grad(plain.layer_norm(leaf64.expand(5, 9, 64), w, b), leaf64, dy.double().expand(5, 9, 64))[0]
    check(got, want, 2)
    x, w, b, _ = inputs((50, 96), torch.float32, torch.float32)
    check_all(x, w, b, torch.ones((), device=DEV).expand(50, 96) * torch.arange(96, device=DEV))


@pytest.mark.parametrize("mean", [0.0, 1e2, 1e4])
@pytest.mark.parametrize("width", [64, 300, 3000])
def test_means_far_from_zero(mean, width):
    """The mean's own rounding does not enter the variance: what is left is the inputs' (of which the 64-bit result knows) and that of one
    difference, 2^-24 of the mean against a spread of one, gradients by way of the mean that is kept (again 2^-24 of it)."""
    x, w, b, dy = inputs((40, width), torch.float32, torch.float32, mean=mean)
    got = gradients(zeno_b200.layer_norm, x, w, b, dy)
    for a, c in zip(got, exact(x, w, b, dy)):
        assert off(a, c) <= 2 * TOL + 2 * mean * 2.0 ** -24


def test_constant_and_extreme_rows():
    x, w, b, dy = inputs((6, 128), torch.float32, torch.float32)
    x[0] = 7.0  # no spread: the bias is left
    x[1] = 0.0
    x[2] *= 1e15
    x[3] *= 1e-15
    got = gradients(zeno_b200.layer_norm, x, w, b, dy)
    want = exact(x, w, b, dy)
    assert torch.equal(got[0][0], b) and torch.equal(got[0][1], b)
    for r in range(6):
        for a, c in zip(got[:2], want[:2]):
            assert off(a[r], c[r]) <= 4 * TOL
    # one row that is not finite leaves the others as they are
    for value in ("nan", "inf"):
        y = x.clone()
        y[4, 9] = float(value)
        bad = gradients(zeno_b200.layer_norm, y, w, b, dy)
        keep = [0, 1, 2, 3, 5]
        assert torch.equal(bad[0][keep], got[0][keep]) and torch.equal(bad[1][keep], got[1][keep])
        assert torch.isnan(bad[0][4]).any() and torch.isnan(bad[2]).any()


def test_gradients_against_differences():
    x, w, b, dy = inputs((20, 70), torch.float32, torch.float32)
    got = gradients(zeno_b200.layer_norm, x, w, b, dy)[1:]
    for at, grad in enumerate(got):
        torch.manual_seed(at)
        way = torch.randn_like(grad).double()
        args = [t.double() for t in (x, w, b)]

        def loss(e):
            args[at] = (x, w, b)[at].double() + e * way
            return (plain.layer_norm(*args) * dy.double()).sum()
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(float((grad.double() * way).sum() - slope)) <= 1e-5 * float(grad.double().norm() * way.norm() / way.numel() ** 0.5)


@pytest.mark.parametrize("dtype,affine", TYPES[:4])
def test_empty(dtype, affine):
    for shape in ((0, 16), (3, 0, 16)):
        x, w, b, dy = inputs(shape, dtype, affine)
        got = gradients(zeno_b200.layer_norm, x, w, b, dy)
        assert got[0].shape == shape and got[1].shape == shape
        assert all(not t.any() for t in got[2:])


def test_partial_gradients():
    x, w, b, dy = inputs((300, 96), torch.bfloat16, torch.float32)
    want = gradients(zeno_b200.layer_norm, x, w, b, dy)
    for mask in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(zeno_b200.layer_norm(*leaves), [t for t in leaves if t.requires_grad], dy)
        for a, c in zip(got, [want[1 + i] for i in range(3) if mask >> i & 1]):
            assert torch.equal(a, c)
    for weight, bias in ((w, None), (None, b)):
        got, ref = gradients(zeno_b200.layer_norm, x, weight, bias, dy), exact(x, weight, bias, dy)
        for a, c in zip(got, ref):
            check(a, c, 2)


def test_in_a_cuda_graph_and_on_streams():
    x, w, b, dy = inputs((4000, 96), torch.bfloat16, torch.float32, seed=1)
    want = gradients(zeno_b200.layer_norm, x, w, b, dy)
    still = [t.clone() for t in inputs((4000, 96), torch.bfloat16, torch.float32, seed=2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = gradients(zeno_b200.layer_norm, x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(again, want):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gradients(zeno_b200.layer_norm, *still)
    for a, c in zip(still, (x, w, b, dy)):
        a.copy_(c)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert torch.equal(a, c)


def test_offsets_that_pass_32_bits():
    x = torch.empty(2 ** 31 // 64 + 5, 64, device=DEV, dtype=torch.bfloat16)  # 4 GB
    x[-7:] = torch.randn(7, 64, device=DEV)
    x[:-7] = 1.0
    y = zeno_b200.layer_norm(x)
    check(y[-7:], plain.layer_norm(x[-7:]))
    assert not y[:-7].any()


def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad
    x = torch.randn(3, 8, device=DEV)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            zeno_b200.layer_norm(forward_ad.make_dual(x, torch.ones_like(x)))


def test_second_derivatives_are_refused():
    x, w, b, dy = inputs((4, 32), torch.float32, torch.float32)
    w.requires_grad_(True)
    once, = torch.autograd.grad(zeno_b200.layer_norm(x, w, b), w, dy, create_graph=True)
    check(once, exact(x, w.detach(), b, dy)[2], 2)
    with pytest.raises(RuntimeError, match="once"):
        once.sum().backward()


def test_refusals():
    x, w = torch.zeros(3, 8, device=DEV), torch.zeros(8, device=DEV)
    f = zeno_b200.layer_norm
    for args, kw, error, match in [
            ((x.half(),), {}, TypeError, "float32 or bfloat16"), ((x, w[:7]), {}, ValueError, "weight must have shape"), ((x, w, w[None]), {}, ValueError, "bias must have shape"),
            ((x, w.bfloat16()), {}, TypeError, "weight must be"), ((x.bfloat16(), w, w.bfloat16()), {}, TypeError, "one type"), ((x, w.cpu()), {}, ValueError, "on cpu"),
            ((x,), {"eps": -1.0}, ValueError, "eps"), ((x,), {"eps": float("nan")}, ValueError, "eps"), ((x[:, :0],), {}, ValueError, "last axis"), ((x[0, 0],), {}, ValueError, "last axis")]:
        with pytest.raises(error, match=match):
            f(*args, **kw)


def test_sizes_beyond_the_entries_are_refused():
    """Before anything is allocated: such a width would not pass the entry's 32-bit field."""
    x = torch.zeros(1, 1, device=DEV)
    for shape in ((1, 2 ** 32 + 8), (1, 2 ** 30 + 1), (2 ** 31 + 1, 1), (2 ** 16, 2 ** 16, 1)):
        with pytest.raises(ValueError, match="at most 2\\^31 rows"):
            zeno_b200.layer_norm(x.expand(shape))
