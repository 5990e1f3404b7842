"""The distillation loss on the CPU: its torch form at the edges, and the LM's use of it."""
import pytest
import torch

from dsalt import DsaltError
from dsalt.kernels.distill import torch_distill_loss


def operands(rows=5, V=11, K=3, seed=1):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn(rows, V, generator=g).requires_grad_()
    z, ids = torch.randn(rows, K, generator=g), torch.randint(0, V, (rows, K), generator=g)
    return s, z, ids, torch.randint(0, V, (rows,), generator=g)


@pytest.mark.parametrize("tau", [0.25, 1.0, 2.0])
def test_teacher_of_lowest_values(tau):
    """All slots alike have 1 / K each, also where the logits over the temperature are past fp32's range."""
    s, z, ids, _ = operands()
    z[1], z[2, 1:] = torch.finfo(torch.float32).min, torch.finfo(torch.float32).min
    got = torch_distill_loss(s, z, ids, None, (tau, 0.0, -100, "none"))
    want = torch_distill_loss(s.double(), z.double(), ids, None, (tau, 0.0, -100, "none"))
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)
