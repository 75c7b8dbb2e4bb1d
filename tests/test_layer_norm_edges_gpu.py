"""layer_norm over the whole range of a float: spreads whose squares overflow or vanish.

Tolerances and the plain implementation are those of test_layer_norm_gpu.py."""
import pytest
import torch

import zeno_b200
from operators_plain import off
from test_layer_norm_gpu import TOL, TYPES, exact, gradients, inputs

pytestmark = pytest.mark.gpu

# every instance: lanes of a row, a warp, a block, more than a block holds; whole vectors and single values
WIDTHS = [3, 8, 29, 64, 100, 256, 500, 777, 1024, 4096, 4099, 9000]


def check_rows(got, want, dtype, wide):
    """Row by row, since rows are of any size: 32-bit results to four times the figure (as rows of one spread each), bfloat16 ones by
    the rounding besides; a result below the least normal value is rounded at 2^-149, in bfloat16 at 2^-133."""
    least = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -134
    for r, (a, b) in enumerate(zip(got, want)):
        assert torch.isfinite(a).all(), r
        error, b = (a.double() - b).abs(), b.abs()
        allowed = 4 * TOL * float(b.square().mean()) ** 0.5 + least * 8
        if dtype == torch.float32:
            assert float(error.square().mean()) ** 0.5 <= allowed, (r, off(a, b))
        else:
            assert float((error - 2.0 ** -8 * b).max()) <= 8 * allowed, (r, float((error - 2.0 ** -8 * b).max()))


@pytest.mark.parametrize("dtype,affine", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_spreads_of_any_size(width, dtype, affine):
    """Rows of spreads from 1e-5 to the largest float, rows whose plain sum overflows, rows of both signs at the end of the range, next to ordinary
    rows: each is the definition's value, in a column's sums too."""
    x, w, b, dy = inputs((40, width), torch.float32, affine, seed=width)
    sizes = [1e-5, 1.0, 1e15, 1.7e19, 2e19, 1e25, 1e30, 1e37, 2e37]
    scale = torch.tensor([sizes[r % len(sizes)] for r in range(40)], device="cuda")
    x = x.clamp(-4, 4) * scale[:, None]
    x[9] = 3.3e38 * (1 - 0.1 * torch.rand(width, device="cuda"))  # (whose sum is past the largest float)
    x[20] = 3.3e38 * torch.where(torch.arange(width, device="cuda") % 3 == 0, 1.0, -1.0)
    x[21] = -x[20]
    x[30] = 0.0
    x[30, width // 2] = 3e38
    x, dy = x.to(dtype), dy.to(dtype)
    keep = [r for r in range(40) if scale[r] == 1.0 and r not in (9, 20, 21, 30)]
    got, want = gradients(zeno_b200.layer_norm, x, w, b, dy), exact(x, w, b, dy)
    for a, c in zip(got[:2], want[:2]):
        check_rows(a, c, dtype, width > 8192)
    for a, c in zip(got[2:], want[2:]):
        assert torch.isfinite(a).all()
        if a.dtype == torch.float32:
            assert off(a, c) <= 4 * TOL
        else:
            error = (a.double() - c).abs() - 2.0 ** -8 * c.abs()
            assert float(error.max()) <= 8 * 4 * TOL * float(c.square().mean()) ** 0.5
    assert torch.equal(zeno_b200.layer_norm(x, w, b), got[0])
    # an ordinary row is what it is among ordinary rows
    assert torch.equal(zeno_b200.layer_norm(x[keep], w, b), got[0][keep])


@pytest.mark.parametrize("dtype,affine", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_spreads_of_next_to_nothing_without_eps(width, dtype, affine):
    """eps = 0: squares of spreads below 1e-19 are not a float's any more, the result is.  (No spread at all is 0 / 0: what is left there is the mean's
    rounding over itself, NaN where there is none.  500 values of 7.0 times 1 / 500, which is no float, are a mean of 7 (1 + 2^-24).)"""
    x, w, b, dy = inputs((24, width), torch.float32, affine, seed=width, mean=0.0)
    sizes = [1.0, 1e-15, 1e-18, 1e-20, 1e-22, 1e-25, 1e-30, 1e-33]
    x = x * torch.tensor([sizes[r % len(sizes)] for r in range(24)], device="cuda")[:, None]
    dy = dy * 1e-6  # (the gradients of x are of the size of dy over the spread)
    x[5] = 7.0
    x, dy = x.to(dtype), dy.to(dtype)
    rows = [r for r in range(24) if r != 5]
    got, want = gradients(zeno_b200.layer_norm, x, w, b, dy, eps=0.0), exact(x, w, b, dy, eps=0.0)
    check_rows(got[0][rows], want[0][rows], dtype, width > 8192)
    if width > 3:  # (of few values next to nothing of the gradient is left: a difference of its parts)
        check_rows(got[1][rows], want[1][rows], dtype, width > 8192)
    got, want = gradients(zeno_b200.layer_norm, x[rows], w, b, dy[rows], eps=0.0), exact(x[rows], w, b, dy[rows], eps=0.0)
    for a, c in zip(got[2:], want[2:]):
        assert torch.isfinite(a).all() and off(a, c) <= (4 * TOL if a.dtype == torch.float32 else 2.0 ** -8)


def test_eps_of_any_size():
    x, w, b, dy = inputs((9, 64), torch.float32, torch.float32)
    x[3] *= 1e25
    for eps in (1e-45, 1e-35, 1e30, 1e38):
        got, want = gradients(zeno_b200.layer_norm, x, w, b, dy, eps=eps), exact(x, w, b, dy, eps=float(torch.tensor(eps)))
        for a, c in zip(got[:2], want[:2]):
            check_rows(a, c, torch.float32, False)
    for t in (zeno_b200.layer_norm(x, w, b, eps=1e300), zeno_b200.layer_norm(x, w, b, eps=float("inf"))):
        assert torch.equal(t, b.expand(9, 64))  # (as a float, eps is infinite)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_what_is_not_finite_stays_in_its_row(width, value):
    for dtype, affine in TYPES:
        x, w, b, dy = inputs((40, width), dtype, affine, seed=width)
        want = gradients(zeno_b200.layer_norm, x, w, b, dy)
        x[17, width - 1] = float(value)
        got = gradients(zeno_b200.layer_norm, x, w, b, dy)
        rows = [r for r in range(40) if r != 17]
        for a, c in zip(got[:2], want[:2]):
            assert torch.equal(a[rows], c[rows]) and torch.isnan(a[17]).all()


def test_views_that_are_negative_by_a_flag():
    """As the imaginary part of a conjugate is, which holds the opposite of its values."""
    x, w, b, dy = inputs((9, 40), torch.float32, torch.float32)
    want = gradients(zeno_b200.layer_norm, x, w, b, dy)
    views = [torch._neg_view(-t) for t in (x, w, b, dy)]
    assert all(t.is_neg() for t in views)
    leaves = [t.requires_grad_(True) for t in views[:3]]
    y = zeno_b200.layer_norm(*leaves)
    for a, c in zip([y, *torch.autograd.grad(y, leaves, views[3])], want):
        assert torch.equal(a, c)
