"""Host-side refusals of the layer norm's entry points (no GPU), and the modules' forms on the CPU."""
import ctypes

import pytest
import torch

import dsalt._hip as hip
from dsalt.kernels import LayerNorm, add_layer_norm, layer_norm


def test_layer_norm_refuses_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: layer_norm(x), lambda: add_layer_norm(x, x)):
        with pytest.raises(hip.DsaltError, match="ROCm GPU"):
            call()


def layer_args(**kw):
    a = hip.LayerNormArgs(rows=32, d=64, x_dtype=2, h_dtype=0, y_dtype=0, w_dtype=2, b_dtype=2, eps=1e-5, workspace_bytes=1 << 30)
    for i, n in enumerate(("x", "h", "weight", "bias", "x_out", "y", "stats", "dx_out", "dy", "dx", "dh", "d_weight", "d_bias",
                           "workspace")):
        setattr(a, n, 0x10000000 + i * 0x100000)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,backward,code", [
    ({}, 0, 0), ({}, 1, 0), ({"rows": -1}, 0, 1), ({"rows": (1 << 31) + 1}, 0, 1), ({"d": 0}, 0, 2), ({"d": 8193}, 0, 2), ({"d": 8191}, 0, 0),
    ({"d": 1}, 1, 0), ({"x_dtype": 3}, 0, 1), ({"x_dtype": 0}, 0, 0), ({"x_dtype": 0, "h_dtype": 1}, 0, 2), ({"x_dtype": 0, "y_dtype": 2}, 0, 2),
    ({"x_dtype": 0, "h_dtype": 1, "h": None}, 0, 0), ({"x_dtype": 0, "h_dtype": 1, "h": None}, 1, 2), ({"w_dtype": 1}, 0, 2),
    ({"w_dtype": 1, "weight": None}, 0, 0), ({"b_dtype": 0}, 0, 2), ({"x": None}, 0, 1), ({"y": None}, 0, 1), ({"x_out": None}, 0, 1),
    ({"x_out": None, "h": None}, 0, 0), ({"stats": None}, 0, 0), ({"stats": None}, 1, 1), ({"dy": None}, 1, 1), ({"x": 0x10000002}, 0, 1),
    ({"h": 0x10000002}, 0, 0), ({"y": 0x10000001}, 0, 1), ({"eps": -1.0}, 0, 1), ({"eps": float("nan")}, 0, 1), ({"workspace": None}, 1, 1),
    ({"workspace_bytes": 64}, 1, 1), ({"workspace": None, "d_weight": None, "d_bias": None}, 1, 0),
    ({"rows": 0, "x": None, "y": None}, 0, 0)])
def test_layer_norm_check(kw, backward, code):
    assert hip.lib().dsalt_layer_norm_check(ctypes.byref(layer_args(**kw)), backward) == code, hip.lib().dsalt_last_error()


def test_layer_norm_null_and_workspace():
    lib = hip.lib()
    assert lib.dsalt_layer_norm(None, None) == 1 and lib.dsalt_layer_norm_bwd(None, None) == 1
    assert lib.dsalt_layer_norm_workspace_size(-1, 64) == 0 and lib.dsalt_layer_norm_workspace_size(9, 0) == 0
    assert lib.dsalt_layer_norm_workspace_size(9, 100) >= 2 * 100 * 4


@pytest.mark.parametrize("bias", [True, False])
def test_layer_norm_module_on_the_cpu(bias):
    m = LayerNorm(24, eps=1e-3, bias=bias)
    x, h = torch.randn(5, 24), torch.randn(5, 24)
    with torch.no_grad():
        m.weight.normal_()
    want = torch.nn.functional.layer_norm(x + h, (24,), m.weight, m.bias, 1e-3)
    s, y = m(x, h)
    torch.testing.assert_close(y, want)
    assert torch.equal(s, x + h) and m(x.bfloat16()).dtype == torch.bfloat16
    assert set(dict(m.named_parameters())) == ({"weight", "bias"} if bias else {"weight"})
