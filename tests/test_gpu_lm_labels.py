"""The LM's distillation loss with labels that are no token, against distill_loss of its logits."""
import pytest
import torch

from dsalt.kernels import distill_loss
from test_gpu_lm_teacher import DEV, lm, packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
@pytest.mark.parametrize("chunk", [2048, 50])
def test_mean_over_the_rows_that_count(ints, chunk):
    ids, cu = packed(4)
    T = ids.numel()
    g = torch.Generator(device=DEV).manual_seed(9)
    zt = torch.randn(T, 12, device=DEV, generator=g) * 2
    ti = torch.rand(T, 500, device=DEV, generator=g).topk(12).indices.to(ints)
    y = torch.roll(ids, -1).to(ints)
    y[::7], y[1::7], y[2::7] = -100, 500, -1
    model = lm(lm_head_chunk_size=chunk).eval()
    with torch.no_grad():
        got = model(ids, cu_seqlens=cu, labels=y, teacher_logits=zt, teacher_ids=ti, temperature=2.0, label_weight=0.4)["loss"]
        want = distill_loss(model(ids, cu_seqlens=cu)["logits"], zt, ti, y, temperature=2.0, label_weight=0.4)
    assert abs(float(got - want)) < 1e-5 * max(1.0, float(want))
