"""Host-side refusals of the gated feed-forward, dropout and branch-norm entry points (no GPU),
and the plain form of their random bits against published values."""
import ctypes

import numpy as np
import pytest
import torch

import dsalt._hip as hip
from dsalt.kernels import branch_norm, counter_dropout, gated_ffn
from dsalt.kernels.dropout import check_seed, torch_counter_dropout
from philox_reference import keep_mask, philox4x32


def test_philox_known_values():
    """The generator's published known-answer values (10 rounds) pin rounds and key schedule."""
    zero = [np.zeros(1, np.uint64)] * 4
    assert [int(w[0]) for w in philox4x32(zero, (0, 0), 10)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = [np.full(1, 0xFFFFFFFF, np.uint64)] * 4
    assert [int(w[0]) for w in philox4x32(ones, (0xFFFFFFFF, 0xFFFFFFFF), 10)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert keep_mask(1000, 0.0, 1, 0).all() and not keep_mask(1000, 1.0, 1, 0).any()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    for call in (lambda: gated_ffn(x, w, w, w), lambda: counter_dropout(x, 0.1, 1), lambda: branch_norm(x, x, w[0])):
        with pytest.raises(hip.DsaltError, match="ROCm GPU"):
            call()


def ffn_args(**kw):
    a = hip.GatedFfnArgs(rows=32, d=64, f=128, e=64, x_stride=64, w_gate_stride=64, w_up_stride=64, w_down_stride=128,
                         dy_stride=64, workspace_bytes=1 << 40)
    for i, n in enumerate(("x", "w_gate", "w_up", "w_down", "gate_up", "act", "y", "dy", "d_gate_up", "dx", "dw_gate", "dw_up",
                           "dw_down", "workspace")):
        setattr(a, n, 0x10000000 + i * 0x100000)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,code", [
    ({}, 0), ({"rows": -1}, 1), ({"rows": 1 << 40}, 1), ({"d": 60}, 2), ({"f": 0}, 2), ({"e": (1 << 20) + 8}, 2), ({"dtype": 2}, 2),
    ({"dtype": 7}, 2), ({"activation": 4}, 1), ({"activation": -1}, 1), ({"x_stride": 56}, 2), ({"w_gate_stride": 68}, 2),
    ({"w_up_stride": -64}, 2), ({"w_down_stride": (1 << 21) + 8}, 2), ({"x": 0x10000008}, 1), ({"act": None}, 1),
    ({"x": None}, 1), ({"rows": 0, "x": None, "act": None, "y": None}, 0), ({"rows": 1 << 31, "f": 1 << 20, "w_down_stride": 1 << 20}, 2)])
def test_gated_ffn_forward_check(kw, code):
    assert hip.lib().dsalt_gated_ffn_check(ctypes.byref(ffn_args(**kw)), 0) == code, hip.lib().dsalt_last_error()


@pytest.mark.parametrize("kw,code", [
    ({}, 0), ({"dy": None}, 1), ({"dy_stride": 60}, 2), ({"d_gate_up": None}, 1), ({"gate_up": None}, 1), ({"act": None}, 1),
    ({"act": None, "dw_down": None}, 0), ({"x": None}, 1), ({"x": None, "dw_gate": None, "dw_up": None}, 0),
    ({"d_gate_up": None, "dx": None, "dw_gate": None, "dw_up": None, "x": None, "gate_up": None, "w_gate": None}, 0),
    ({"w_up": None}, 1), ({"w_up": None, "w_gate": None, "dx": None}, 0), ({"w_down": None}, 1)])
def test_gated_ffn_backward_check(kw, code):
    assert hip.lib().dsalt_gated_ffn_check(ctypes.byref(ffn_args(**kw)), 1) == code, hip.lib().dsalt_last_error()


@pytest.mark.parametrize("kw,backward,code", [
    ({"rows": 1 << 30, "f": 8, "w_down_stride": 8}, 0, 0), ({"rows": (1 << 30) + 1, "f": 8, "w_down_stride": 8}, 0, 2),
    ({"rows": (1 << 30) + 1, "f": 8, "w_down_stride": 8}, 1, 2), ({"rows": 1 << 23, "f": 1 << 14, "w_down_stride": 1 << 14}, 0, 0),
    ({"rows": (1 << 23) + 1, "f": 1 << 14, "w_down_stride": 1 << 14}, 0, 2), ({"rows": 8, "f": 1 << 20, "w_down_stride": 1 << 20}, 1, 0),
    ({"rows": 8, "f": 1 << 20, "d": 1 << 17, "x_stride": 1 << 17, "w_gate_stride": 1 << 17, "w_up_stride": 1 << 17,
      "w_down_stride": 1 << 20}, 1, 2)])
def test_gated_ffn_grids_that_a_launch_cannot_hold(kw, backward, code):
    """A launch holds fewer than 2^32 threads: what would need more is refused."""
    assert hip.lib().dsalt_gated_ffn_check(ctypes.byref(ffn_args(**kw)), backward) == code, hip.lib().dsalt_last_error()


def test_gated_ffn_workspace_check():
    need = hip.lib().dsalt_gated_ffn_workspace_size(32, 64, 128, 64, 1)
    assert need >= 0 and hip.lib().dsalt_gated_ffn_workspace_size(-1, 64, 128, 64, 1) == 0
    if need:
        assert hip.lib().dsalt_gated_ffn_check(ctypes.byref(ffn_args(workspace_bytes=need - 1)), 1) == 1
    assert hip.lib().dsalt_gated_ffn_check(None, 0) == 1


@pytest.mark.parametrize("kw", [{"n": -1}, {"n": 1 << 41}, {"dtype": 3}, {"threshold": -1}, {"threshold": 65537}, {"x": None},
                                {"out": 0x10000004}, {"seed_ptr": 0x10000004}])
def test_dropout_refusals(kw):
    a = hip.DropoutArgs(n=64, dtype=0, threshold=60000, x=0x10000000, out=0x10100000)
    for n, v in kw.items():
        setattr(a, n, v)
    assert hip.lib().dsalt_dropout(ctypes.byref(a), None) == 1
    assert hip.lib().dsalt_dropout(None, None) == 1


def branch_args(**kw):
    a = hip.BranchNormArgs(rows=32, d=64, x_dtype=2, h_dtype=0, y_dtype=0, w_dtype=2, post_dtype=2, gate_dtype=2, gate_kind=1,
                           threshold=60000, eps=1e-6, post_eps=1e-6, residual_scale=1.0, workspace_bytes=1 << 30)
    for i, n in enumerate(("x", "h", "weight", "post_weight", "gate", "x_out", "y", "rstd", "rstd_post", "dx_out", "dy", "dx", "dh",
                           "d_weight", "d_post_weight", "d_gate", "workspace")):
        setattr(a, n, 0x10000000 + i * 0x100000)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,backward,code", [
    ({}, 0, 0), ({}, 1, 0), ({"rows": -1}, 0, 1), ({"d": 12}, 0, 2), ({"d": 8200}, 0, 2), ({"x_dtype": 0}, 0, 0),
    ({"x_dtype": 0, "h_dtype": 1}, 0, 2), ({"x_dtype": 0, "y_dtype": 2}, 0, 2), ({"x_dtype": 5}, 0, 1), ({"w_dtype": 1}, 0, 2),
    ({"gate_kind": 3}, 0, 1), ({"threshold": 70000}, 0, 1), ({"h": None}, 0, 1), ({"gate": None}, 0, 1),
    ({"gate": None, "gate_kind": 0}, 0, 0), ({"x_out": None}, 0, 1), ({"y": None}, 0, 1), ({"y": None, "weight": None}, 0, 0),
    ({"x": 0x10000008}, 0, 1), ({"gate": 0x10000004}, 0, 1), ({"gate": 0x10000004, "gate_kind": 2}, 0, 0),
    ({"seed_ptr": 0x10000004}, 0, 1), ({"dx_out": None}, 1, 0), ({"dx_out": None, "dy": None}, 1, 1), ({"rstd": None}, 1, 1),
    ({"rstd_post": None}, 1, 1), ({"workspace": None}, 1, 1), ({"workspace_bytes": 16}, 1, 1), ({"post_weight": None}, 1, 1),
    ({"workspace": None, "d_weight": None, "d_post_weight": None, "gate_kind": 2}, 1, 0)])
def test_branch_norm_check(kw, backward, code):
    assert hip.lib().dsalt_branch_norm_check(ctypes.byref(branch_args(**kw)), backward) == code, hip.lib().dsalt_last_error()


def test_argument_values():
    for p in (-0.5, 1.01, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            hip.keep_threshold(p)
    assert [hip.keep_threshold(p) for p in (0.0, 0.5, 1.0, 0.1)] == [65536, 32768, 0, 58982]
    dev = torch.device("cuda", 0)
    assert hip.seed_fields(-1, dev) == (-1, 0) and hip.seed_fields(2 ** 64 - 1, dev) == (-1, 0)
    for bad in (2 ** 64, -2 ** 63 - 1):
        with pytest.raises(ValueError, match="64 bits"):
            hip.seed_fields(bad, dev)
    with pytest.raises(hip.DsaltError):
        hip.seed_fields(torch.tensor([1]), dev)


@pytest.mark.parametrize("lead", [(), (1,), (64,), (3, 5), (64, 1)])
def test_branch_norm_gate_kinds(lead):
    """A channel's gate is [d] and a token's [..., 1] beside x [..., d], x [d] and its gate [1] among
    them: the kind in the argument struct says how many elements the kernels read and write."""
    d = 64
    x = torch.zeros(*lead, d)
    opts = (1.0, 0.0, 0, 1e-6, 1e-6, x.dtype)
    for gate, kind in ((None, 0), (torch.zeros(d), 1), (torch.zeros(*lead, 1), 2)):
        a = hip.BranchNormArgs.from_buffer_copy(hip._branch_pack(x, x, None, None, gate, opts, None))
        assert a.gate_kind == kind and a.d == d and a.rows * d == x.numel()
        assert gate is None or gate.numel() == (a.d if kind == 1 else a.rows)


@pytest.mark.parametrize("kw", [{"weight": None, "dy": None}, {"gate": None, "gate_kind": 0}])
def test_branch_norm_gradients_without_their_tensor(kw):
    """The gradient of a weight or a gate that the call does not have would be left as it was."""
    assert hip.lib().dsalt_branch_norm_check(ctypes.byref(branch_args(**kw)), 1) == 1
    grads = {"d_weight": None} if "weight" in kw else {"d_gate": None}
    assert hip.lib().dsalt_branch_norm_check(ctypes.byref(branch_args(**kw, **grads)), 1) == 0, hip.lib().dsalt_last_error()


@pytest.mark.parametrize("rows,d,f,e,backward", [(1500, 1024, 2816, 1024, 0), (575, 264, 712, 264, 1), (700, 264, 712, 264, 1)])
def test_gated_ffn_workspace_of_split_products(rows, d, f, e, backward):
    """Sizes whose products are split along k keep partial sums: less workspace, or none, is refused."""
    need = hip.lib().dsalt_gated_ffn_workspace_size(rows, d, f, e, backward)
    assert need > 0
    size = dict(rows=rows, d=d, f=f, e=e, x_stride=d, w_gate_stride=d, w_up_stride=d, w_down_stride=f, dy_stride=e)
    for more, code in (({"workspace_bytes": need}, 0), ({"workspace_bytes": need - 1}, 1), ({"workspace_bytes": 0}, 1),
                       ({"workspace": None}, 1), ({"workspace": 0x10000008}, 1)):
        assert hip.lib().dsalt_gated_ffn_check(ctypes.byref(ffn_args(**size, **more)), backward) == code, more


@pytest.mark.parametrize("integer", [np.int64, np.int32, np.uint64, np.uint8, int])
def test_seeds_and_offsets_of_any_integer_type(integer):
    """A seed or offset that a program drew with numpy is its value; one that is no integer is refused by
    type, before anything is packed."""
    dev = torch.device("cuda", 0)
    info = None if integer is int else np.iinfo(integer)
    for v in (0, 5, int(info.max) if info else 2 ** 64 - 1, int(info.min) if info else -2 ** 63):
        assert hip.seed_fields(integer(v), dev) == hip.seed_fields(v, dev)
        check_seed(0.1, integer(v), integer(abs(v) % 100), dev)
    for bad in (1.0, "1", np.float64(2)):
        for seed, offset in ((bad, 0), (1, bad)):
            with pytest.raises(TypeError):
                check_seed(0.1, seed, offset, dev)


@pytest.mark.parametrize("n", [0, 1, 7, 8, 1003])
@pytest.mark.parametrize("p,seed,offset", [(0.25, 11, 3), (0.5, -2 ** 63, 2 ** 63 - 1), (0.97, 2 ** 64 - 1, 2 ** 32), (1.0, 0, 0), (0.0, 5, 1)])
def test_dropout_in_torch_ops_has_the_same_mask(n, p, seed, offset):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n))
    keep = torch.from_numpy(keep_mask(n, p, seed, offset))
    scale = np.float32(65536 / max(hip.keep_threshold(p), 1)).item()
    want = torch.where(keep, x * scale, 0.0)
    assert torch.equal(torch_counter_dropout(x, p, seed, offset), want)
    tensor = torch.tensor([(seed + 2 ** 63) % 2 ** 64 - 2 ** 63])
    assert torch.equal(torch_counter_dropout(x.bfloat16(), p, tensor, offset), torch.where(keep, x.bfloat16().float() * scale, 0.0).bfloat16())
