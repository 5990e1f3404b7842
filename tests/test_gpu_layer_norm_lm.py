"""The LM with layer norms where a feed-forward was replaced by one that returns a wider type than the stream's."""
import pytest
import torch
import torch.nn as nn

from test_gpu_lm_teacher import BF, DEV, lm, packed

pytestmark = pytest.mark.gpu


class Wide(nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x).float()


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("at", [0, 1])
def test_answers_with_a_wide_feed_forward(norm, at):
    """Under autocast the 16-bit stream goes on in fp32 behind it: answers without autograd are those of the blocks
    one by one (with it), but for 16-bit roundings at some ten places."""
    ids, cu = packed(2)
    model = lm(norm=norm).eval()
    model.layers[at].ffn = Wide(model.layers[at].ffn)
    with torch.autocast("cuda", dtype=BF):
        with torch.no_grad():
            got = model(ids, cu_seqlens=cu)["logits"].float()
        want = model(ids, cu_seqlens=cu)["logits"].detach().float()
    assert float((got - want).norm() / want.norm()) < 10 * 2.0 ** -9
