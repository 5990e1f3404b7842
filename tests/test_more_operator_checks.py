"""Host-side refusals of the layer norm's, the distillation loss's and the 8-bit products' entry points
(no GPU), and their plain forms on the CPU."""
import ctypes

import pytest
import torch

import dsalt._hip as hip
from dsalt.kernels import FP8Linear, LayerNorm, add_layer_norm, distill_loss, fp8_linear, fp8_matmul, fp8_quantize, layer_norm
from dsalt.kernels.distill import torch_distill_loss
from dsalt.kernels.fp8 import torch_fp8_matmul, torch_fp8_quantize


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


def test_distill_refuses_cpu_tensors_and_bad_values():
    s, z, ids = torch.zeros(2, 9), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(hip.DsaltError, match="ROCm GPU"):
        distill_loss(s, z, ids)
    for kw in (dict(temperature=0.0), dict(label_weight=2.0), dict(label_weight=0.5), dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            distill_loss(s, z, ids, **kw)


def distill_args(**kw):
    a = hip.DistillArgs(rows=4, logits_stride=100, teacher_stride=8, ids_stride=8, ignore_index=-100, vocab=100, k=8, logits_dtype=0,
                        teacher_dtype=2, ids_int64=1, labels_int64=1, reduction=1, temperature=2.0, label_weight=0.5,
                        workspace_bytes=1 << 30)
    for i, n in enumerate(("logits", "teacher", "ids", "labels", "loss", "stats", "d_loss", "d_logits", "workspace")):
        setattr(a, n, 0x10000000 + i * 0x100000)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,backward,code", [
    ({}, 0, 0), ({}, 1, 0), ({"rows": -1}, 0, 1), ({"rows": 1 << 24}, 0, 1), ({"vocab": 0}, 0, 2), ({"vocab": (1 << 30) + 1}, 0, 2),
    ({"k": 0}, 0, 2), ({"k": 1025, "teacher_stride": 1025, "ids_stride": 1025}, 0, 2), ({"logits_dtype": 3}, 0, 1), ({"teacher_dtype": -1}, 0, 1),
    ({"reduction": 3}, 0, 1), ({"temperature": 0.0}, 0, 1), ({"temperature": float("inf")}, 0, 1), ({"temperature": float("nan")}, 0, 1),
    ({"label_weight": 1.01}, 0, 1), ({"label_weight": float("nan")}, 0, 1), ({"labels": None}, 0, 1), ({"labels": None, "label_weight": 0.0}, 0, 0),
    ({"logits_stride": 99}, 0, 1), ({"ids_stride": 7}, 0, 1), ({"teacher_stride": -8}, 0, 1), ({"logits": 0x10000001}, 0, 1),
    ({"logits": 0x10000002}, 0, 0), ({"ids": 0x10000004}, 0, 1), ({"ids": 0x10000004, "ids_int64": 0}, 0, 0), ({"teacher": None}, 0, 1),
    ({"loss": None}, 0, 1), ({"stats": None}, 0, 0), ({"stats": None}, 1, 1), ({"d_loss": None}, 1, 1), ({"d_logits": None}, 1, 1),
    ({"workspace": None}, 0, 1), ({"workspace_bytes": 15}, 0, 1), ({"workspace": None}, 1, 0),
    ({"rows": 0, "logits": None, "teacher": None, "ids": None, "labels": None, "workspace": None}, 0, 0)])
def test_distill_check(kw, backward, code):
    assert hip.lib().dsalt_distill_check(ctypes.byref(distill_args(**kw)), backward) == code, hip.lib().dsalt_last_error()


def test_distill_workspace():
    lib = hip.lib()
    assert lib.dsalt_distill(None, None) == 1 and lib.dsalt_distill_workspace_size(-1, 9) == 0
    need = lib.dsalt_distill_workspace_size(3, 50000)  # few long rows are cut into slices
    assert need > 12 and lib.dsalt_distill_workspace_size(3, 500) == 12
    args = distill_args(rows=3, vocab=50000, logits_stride=50000, workspace_bytes=need - 1)
    assert lib.dsalt_distill_check(ctypes.byref(args), 0) == 1


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distill_in_torch_ops(reduction):
    """The plain form against the definition, rows without slots or label among them."""
    g = torch.Generator().manual_seed(1)
    s, z = torch.randn(5, 11, generator=g, dtype=torch.float64), torch.randn(5, 3, generator=g)
    ids = torch.tensor([[1, 4, 9], [0, 0, -1], [-1, 11, -5], [2, 3, 4], [7, 8, 9]])
    z[4, 0] = float("-inf")
    y = torch.tensor([4, 2, 3, -100, 10])
    want = []
    for r in range(5):
        if y[r] < 0:
            want.append(torch.zeros((), dtype=torch.float64))
            continue
        on = (ids[r] >= 0) & (ids[r] < 11) & (z[r] > float("-inf"))
        p = torch.softmax(z[r][on].double() / 2, 0)
        kl = (p * (p.log() - torch.log_softmax(s[r] / 2, 0)[ids[r][on]])).sum()
        want.append(0.7 * 4 * kl - 0.3 * torch.log_softmax(s[r], 0)[y[r]])
    want = torch.stack(want)
    got = torch_distill_loss(s, z, ids, y, (2.0, 0.3, -100, reduction))
    torch.testing.assert_close(got, {"mean": want.sum() / 4, "sum": want.sum(), "none": want}[reduction])


E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_fp8_refuses_cpu_tensors():
    x, q, s = torch.zeros(4, 64), torch.zeros(4, 64).to(E4), torch.ones(4, 1)
    for call in (lambda: fp8_quantize(x), lambda: fp8_matmul(q, s, q, s[:1]), lambda: fp8_linear(x, q, s[:1])):
        with pytest.raises(hip.DsaltError, match="ROCm GPU"):
            call()
    with pytest.raises(ValueError, match="multiple of 16"):
        FP8Linear(40, 8)


def fp8_args(**kw):
    a = hip.Fp8MatmulArgs(m=100, n=96, k=256, a_dtype=3, a_scale_e8m0=1, b_scale_e8m0=1, bias_dtype=2, out_dtype=0, a_stride=256,
                          a_scale_stride_m=2, a_scale_stride_k=1, b_stride=256, b_scale_stride_n=2, b_scale_stride_k=1,
                          workspace_bytes=1 << 40)
    for i, n in enumerate(("a", "a_scale", "b", "b_scale", "bias", "out", "workspace")):
        setattr(a, n, 0x10000000 + i * 0x100000)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,code", [
    ({}, 0), ({"m": -1}, 1), ({"m": (1 << 24) + 1}, 1), ({"n": 0}, 2), ({"n": (1 << 20) + 1}, 2), ({"k": 0}, 2), ({"k": 120, "a_stride": 128}, 2),
    ({"k": (1 << 20) + 16, "a_stride": 1 << 21, "b_stride": 1 << 21}, 2), ({"m": 1 << 24, "n": 1 << 15}, 2), ({"a_dtype": 4}, 1), ({"a_dtype": 0}, 2),
    ({"a_dtype": 0, "m": 32}, 0), ({"a_dtype": 0, "m": 32, "a_scale": None}, 0), ({"a_scale": None}, 1), ({"out_dtype": 3}, 1),
    ({"bias_dtype": 5}, 1), ({"bias_dtype": 5, "bias": None}, 0), ({"a_stride": 240}, 2), ({"b_stride": 264}, 2), ({"a_stride": (1 << 22) + 16}, 2),
    ({"a_dtype": 2, "m": 3, "a_stride": 1 << 21}, 2), ({"a_scale_stride_m": 0}, 2), ({"b_scale_stride_k": (1 << 21) + 1}, 2), ({"a": 0x10000008}, 1),
    ({"out": 0x10000004}, 1), ({"a_scale": 0x10000003}, 0), ({"a_scale": 0x10000003, "a_scale_e8m0": 0, "b_scale_e8m0": 0}, 1), ({"a_scale_e8m0": 0}, 2),
    ({"a_scale_e8m0": 0, "a_dtype": 0, "m": 8}, 0), ({"bias": 0x10000002}, 1),
    ({"bias": 0x10000002, "bias_dtype": 0}, 0), ({"b": None}, 1), ({"out": None}, 1),
    ({"m": 0, "a": None, "a_scale": None, "out": None}, 0)])
def test_fp8_matmul_check(kw, code):
    assert hip.lib().dsalt_fp8_matmul_check(ctypes.byref(fp8_args(**kw))) == code, hip.lib().dsalt_last_error()


def test_fp8_workspace():
    """A product of few tiles and many blocks of k is split along k and needs room for its parts."""
    lib = hip.lib()
    need = lib.dsalt_fp8_matmul_workspace_size(40, 64, 1 << 14)
    assert need >= 2 * 40 * 64 * 4 and lib.dsalt_fp8_matmul_workspace_size(32, 64, 1 << 14) == 0
    size = dict(m=40, n=64, k=1 << 14, a_stride=1 << 14, b_stride=1 << 14)
    for more, code in (({"workspace_bytes": need}, 0), ({"workspace_bytes": need - 1}, 1), ({"workspace": None}, 1), ({"workspace": 0x10000004}, 1)):
        assert lib.dsalt_fp8_matmul_check(ctypes.byref(fp8_args(**size, **more))) == code
    assert lib.dsalt_fp8_matmul_check(None) == 1 and lib.dsalt_fp8_matmul(None, None) == 1


@pytest.mark.parametrize("kw,code", [
    ({"rows": -1}, 1), ({"k": 0}, 2), ({"k": (1 << 20) + 1}, 2), ({"x_dtype": 3}, 1), ({"x_stride": 299}, 1), ({"scale_stride": 2}, 1),
    ({"x": 0x10000001}, 1), ({"q": 0x10000004}, 1), ({"scale": 0x10000002, "scale_f32": 1}, 1), ({"x": None}, 1), ({"q": None}, 1),
    ({"scale": None}, 1), ({"rows": 1 << 30, "tile": 1}, 2), ({"rows": 0, "x": None}, 0)])
def test_fp8_quantize_check(kw, code):
    a = hip.Fp8QuantizeArgs(rows=4, x_stride=300, scale_stride=3, k=300, x_dtype=0, x=0x10000000, q=0x10100000, scale=0x10200000)
    for n, v in kw.items():
        setattr(a, n, v)
    assert hip.lib().dsalt_fp8_quantize(ctypes.byref(a), None) == code, hip.lib().dsalt_last_error()


def test_fp8_in_torch_ops():
    """The plain forms on values whose scales and roundings can be named."""
    x = torch.zeros(2, 200)
    x[0, 0], x[0, 1], x[0, 150] = 448.0, 17.0, -449.0  # scales 1 and 2; 17 lies between 16 and 18, to even: 16
    x[1, 3] = 3.0
    q, s = torch_fp8_quantize(x, False, E8)
    assert s.float().tolist() == [[1.0, 2.0], [2.0 ** -7, 1.0]]
    assert q.float()[0, :2].tolist() == [448.0, 16.0] and q.float()[0, 150] == -224.0 and q.float()[1, 3] == 384.0
    tq, ts = torch_fp8_quantize(x, True, torch.float32)
    assert ts.tolist() == [[1.0, 2.0]] and tq.shape == x.shape
    w, ws = torch_fp8_quantize(torch.eye(200), True, E8)
    torch.testing.assert_close(torch_fp8_matmul(q, s, w, ws, torch.ones(200), torch.float32),
                               q.float() * s.float().repeat_interleave(128, 1)[:, :200] + 1)


def test_fp8_module_keeps_its_bytes():
    m = FP8Linear(32, 130, bias=True)
    assert m.weight_q.dtype is E4 and m.weight_scale.dtype is E8 and m.weight_scale.shape == (2, 1)
    m.weight_bits.random_(0, 120)
    kept = m.weight_bits.clone()
    m.to(torch.bfloat16)
    assert torch.equal(m.weight_bits, kept) and m.bias.dtype is torch.bfloat16
    other = FP8Linear(32, 130, bias=True)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.weight_bits, kept)
