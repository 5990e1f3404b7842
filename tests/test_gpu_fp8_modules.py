"""quantize_fp8 of feed-forwards and models: all of it, or nothing."""
import pytest
import torch
import torch.nn as nn

from dsalt.kernels import FP8Linear
from dsalt.model import DSALTLMHeadModel
from dsalt.modules import SwiGLUFFN

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def kinds(module):
    return [type(m) for m in module.modules() if isinstance(m, (nn.Linear, FP8Linear))]


def test_refused_quantisation_changes_nothing():
    """A width that 8-bit layers do not take, met behind others that they do."""
    ffn = SwiGLUFFN(32, 40).to(DEV)
    before, x = kinds(ffn), torch.randn(3, 32, device=DEV)
    want = ffn(x)
    with pytest.raises(ValueError, match="multiple of 16"):
        ffn.quantize_fp8()
    assert kinds(ffn) == before and torch.equal(ffn(x), want)
    kw = dict(vocab_size=64, n_layers=2, n_heads=2, n_min=4, n_max=16, k_lmk=4, max_seq_len=64)
    for d_ff, d_model in ((48, 128), (192, 128)):
        model = DSALTLMHeadModel(d_model=d_model, d_ff=d_ff, **kw).to(DEV)
        model.layers[1].ffn.down_proj = nn.Linear(d_ff - 8, d_model, bias=False, device=DEV)
        before = kinds(model)
        with pytest.raises(ValueError, match="multiple of 16"):
            model.quantize_fp8()
        assert kinds(model) == before
    model = DSALTLMHeadModel(d_model=128, d_ff=192, **kw).to(DEV)
    model.lm_head = nn.Linear(128, 64, bias=False, device=DEV, dtype=torch.float64)
    before = kinds(model)
    with pytest.raises(Exception):
        model.quantize_fp8()
    assert kinds(model) == before
