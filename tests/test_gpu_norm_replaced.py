"""The LM without autograd, whose residual adds and norms are one pass each: a replaced or hooked norm is called as it is."""
import pytest
import torch
import torch.nn as nn

from dsalt.kernels import RMSENorm
from test_gpu_lm_teacher import BF, DEV, lm, packed

pytestmark = pytest.mark.gpu


class Scaled(RMSENorm):
    def forward(self, x):
        return super().forward(x) * 2


def torch_norm():
    m = nn.LayerNorm(128).to(DEV, BF)
    nn.init.normal_(m.bias)
    return m


@pytest.mark.parametrize("place", ["attn", "ffn", "final"])
@pytest.mark.parametrize("what", ["torch", "subclass", "hook"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_replaced_norms(place, what, norm):
    """The answers are those of the same blocks with autograd, but for 16-bit roundings at some ten places."""
    if what == "subclass" and norm == "layer":
        norm = "rms"
    ids, cu = packed(2)
    model = lm(norm=norm).to(BF).eval()
    owner, name = {"attn": (model.layers[1], "attn_norm"), "ffn": (model.layers[0], "ffn_norm"), "final": (model, "final_norm")}[place]
    calls = []
    if what == "hook":
        getattr(owner, name).register_forward_hook(lambda m, i, o: (calls.append(1), o * 2)[1])
    else:
        setattr(owner, name, torch_norm() if what == "torch" else Scaled(128).to(DEV, BF))
    with torch.no_grad():
        got = model(ids, cu_seqlens=cu)["logits"].float()
    assert len(calls) == (what == "hook")
    want = model(ids, cu_seqlens=cu)["logits"].detach().float()
    assert float((got - want).norm() / want.norm()) < 10 * 2.0 ** -9
