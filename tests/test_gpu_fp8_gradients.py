"""8-bit products and quantisation refuse whatever requires a gradient while gradients are recorded."""
import pytest
import torch

from dsalt import DsaltError
from dsalt.kernels import FP8Linear, fp8_linear, fp8_matmul, fp8_quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows", [4, 70])
def test_operands_that_require_a_gradient(rows):
    x, w = torch.randn(rows, 256, device=DEV), torch.randn(64, 256, device=DEV)
    (a, sa), (b, sb), bias = fp8_quantize(x, scale_dtype=torch.float32), fp8_quantize(w, True, torch.float32), torch.zeros(64, device=DEV)
    want, lin = fp8_matmul(a, sa, b, sb, bias), fp8_linear(x, b, sb, bias)

    def leaf(t):
        return t.detach().clone().requires_grad_()

    calls = [lambda: fp8_matmul(a, leaf(sa), b, sb, bias), lambda: fp8_matmul(a, sa, b, leaf(sb), bias),
             lambda: fp8_matmul(a, sa, b, sb, leaf(bias)), lambda: fp8_linear(x, b, leaf(sb), bias),
             lambda: fp8_linear(leaf(x), b, sb, bias), lambda: fp8_linear(x, b, sb, leaf(bias)),
             lambda: fp8_quantize(leaf(x)), lambda: fp8_quantize(leaf(w), tile=True)]
    for call in calls:
        with pytest.raises(DsaltError, match="inference"):
            call()
    with torch.no_grad():
        results = [call() for call in calls]
    assert all(torch.equal(y, want) for y in results[:3]) and all(torch.equal(y, lin) for y in results[3:6])
    assert torch.equal(results[6][0].float(), a.float()) and torch.equal(results[7][0].float(), b.float())
    layer = FP8Linear.from_linear(torch.nn.Linear(256, 64, device=DEV))  # takes the weight as it is
    assert layer(x).shape == (rows, 64)


def test_transforms_refuse_alike():
    """Under functorch the gradient would reach the scales of torch's form: the same refusal."""
    x, w = torch.randn(4, 256, device=DEV), torch.randn(64, 256, device=DEV)
    b, sb = fp8_quantize(w, True, torch.float32)
    for fn, at in ((lambda s: fp8_linear(x, b, s).sum(), sb), (lambda t: fp8_quantize(t)[1].float().sum(), x)):
        with pytest.raises(DsaltError, match="inference"):
            torch.func.grad(fn)(at)
