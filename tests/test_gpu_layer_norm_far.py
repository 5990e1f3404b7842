"""The layer norm's gradients on rows whose mean is far from zero, bounded by the normalised row."""
import pytest
import torch

from dsalt.kernels import add_layer_norm, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gradient(z, w, dy, eps, mean):
    """dz of the formula in float64 with this mean of the rows."""
    r = torch.rsqrt((z - z.mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + eps)
    n, a = (z - mean) * r, dy * w
    return r * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True)), n, r


@pytest.mark.parametrize("d", [512, 1000, 1024, 4096, 8191])
@pytest.mark.parametrize("add", [False, True])
def test_gradients_of_far_rows(d, add):
    """x around 10^6 with a deviation of 2. x - mean is exact in fp32 (both lie within a factor of two), and what the
    mean's own rounding, up to 2^-5 here, left of it is taken off: n is then off by roundings of values of its own size, and
    so are the sums over n, each within 2^-18 of its terms (64 terms a lane, then trees). dz has three such factors (r, n and the
    mean of a n): 2^-16 of r max|dy| max|w| (1 + max n^2). The bound has to tell the mean's rounding: the formula with
    the mean rounded to fp32 is refused by it, and so is a gradient of zeros."""
    g = torch.Generator(device=DEV).manual_seed(d)
    x = (torch.randn(33, d, device=DEV, generator=g) * 2 + 1e6).requires_grad_()
    w = (torch.randn(d, device=DEV, generator=g) * 0.25 + 1).requires_grad_()
    b = torch.zeros(d, device=DEV).requires_grad_()
    h = torch.zeros(33, d, device=DEV)
    y = add_layer_norm(x, h, w, b)[1] if add else layer_norm(x, w, b)
    z, W = x.detach().double(), w.detach().double()
    mean = z.mean(-1, keepdim=True)
    dy = ((z - mean) / 2).float()  # along n: the mean of a n is near 1
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want, n, r = gradient(z, W, dy.double(), 1e-5, mean)
    scale = float(r.max() * dy.abs().max() * W.abs().max() * (1 + n.abs().max() ** 2))
    tol = 2.0 ** -24 * want.abs() + 2.0 ** -16 * scale
    assert bool(((dx.double() - want).abs() <= tol).all()), float(((dx.double() - want).abs() / tol).max())
    assert not bool((want.abs() <= tol).all())
    rounded, _, _ = gradient(z, W, dy.double(), 1e-5, mean.float().double())
    assert not bool(((rounded - want).abs() <= tol).all()), float(((rounded - want).abs() / tol).max())
    sums = 2.0 ** -18 * (dy.double().abs() * (1 + n.abs())).sum(0)
    assert bool(((dw.double() - (dy.double() * n).sum(0)).abs() <= sums).all())
    assert bool(((db.double() - dy.double().sum(0)).abs() <= sums).all())
    assert bool(((y.double() - n * W).abs() <= 2.0 ** -16 * (1 + n.abs()) * W.abs()).all())
