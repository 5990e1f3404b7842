"""The gated feed-forward block as one differentiable function on hand-written HIP kernels:
``act(x w_gate^T) * (x w_up^T)`` times ``w_down^T`` (SwiGLUFFN, dsalt_transformer.py:10-21, and
its GELU and ReLU relatives).

Both projections, the activation and the product are one kernel, and so are the gradient of
the product and the activation's gradient. Products accumulate in fp32; the hidden activation
and the gradients of gate and up are rounded once, from fp32, and gate and up are kept for the
backward in four or five bits more than the element type has.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .. import _hip
from ._block_train import autocast_dtype, eager, graph_grads, without_autocast
from .dsalt_triton_attn import _dynamo_opaque

_TORCH_ACT = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}


def torch_gated_ffn(x, w_gate, w_up, w_down, activation: str):
    """``gated_ffn`` in torch's ops."""
    return F.linear(_TORCH_ACT[activation](F.linear(x, w_gate)) * F.linear(x, w_up), w_down)


def _versions(*ws):
    """What tells whether a tensor was changed in place (inference tensors count no versions)."""
    return tuple(None if w.is_inference() else w._version for w in ws)


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        # what a gradient needs is saved, as three linears would: a weight changed in place before
        # the backward is refused where a gradient reads it
        need = ctx.needs_input_grad[:4]
        inner = any(need[:3])
        y, kept = _run(x, w_gate, w_up, w_down, activation, inner)
        ctx.save_for_backward(x if inner else None, *((w_gate, w_up) if need[0] else (None, None)),
                              w_down if inner else None, kept)
        ctx.dsalt = x.shape, (w_gate, w_up, w_down), _versions(w_gate, w_up, w_down), activation
        return y

    @staticmethod
    @without_autocast
    def backward(ctx, dy):
        x, _, _, _, kept = ctx.saved_tensors
        shape, ws, versions, activation = ctx.dsalt
        need = ctx.needs_input_grad[:4]
        if torch.is_grad_enabled():  # a graph of the backward is wanted: torch's own ops
            if _versions(*ws) != versions:
                raise RuntimeError("a weight of gated_ffn was changed in place before a backward that records a graph")
            if x is None:  # only w_down has a gradient
                act = kept.view(dy.dtype).view(*shape[:-1], ws[2].shape[1])
                dw, = graph_grads(lambda w: (F.linear(act, w),), ws[2:], (dy,))
                return None, None, None, dw, None
            return *graph_grads(lambda *t: (torch_gated_ffn(*t, activation),), (x, *ws), (dy,)), None
        row = _hip.row_operand
        dy = row(dy.reshape(-1, dy.shape[-1]))
        dx, dwg, dwu, dwd = _hip.gated_ffn_bwd(None if x is None else row(x.reshape(-1, shape[-1])), row(ws[0]), row(ws[1]),
                                               row(ws[2]), activation, kept, dy, need)
        return None if dx is None else dx.view(shape), dwg, dwu, dwd, None


def _run(x, w_gate, w_up, w_down, activation, keep):
    row = _hip.row_operand
    return _hip.gated_ffn(row(x if x.dim() == 2 else x.reshape(-1, x.shape[-1])), row(w_gate), row(w_up), row(w_down),
                          activation, x.shape[:-1], keep)


def gated_ffn_supported(x, w_gate, w_up, w_down) -> bool:
    """Whether `gated_ffn` takes these tensors: bf16 or fp16 on one GPU (fp32 ones under a 16-bit
    autocast are cast), x [..., d], w_gate and w_up [f, d], w_down [e, f] with d, e and f
    multiples of 8."""
    dev = x.device
    if dev.type != "cuda" or w_gate.device != dev or w_up.device != dev or w_down.device != dev:
        return False
    dt = autocast_dtype(x)
    if dt is not torch.bfloat16 and dt is not torch.float16:
        return False
    if not (x.dtype is w_gate.dtype is w_up.dtype is w_down.dtype is dt):
        ok = (dt, torch.float32) if torch.is_autocast_enabled("cuda") else (dt,)
        if x.dtype not in ok or w_gate.dtype not in ok or w_up.dtype not in ok or w_down.dtype not in ok:
            return False
    if x.dim() < 1 or w_gate.dim() != 2 or w_down.dim() != 2 or w_up.shape != w_gate.shape:
        return False
    f, d = w_gate.shape
    e = w_down.shape[0]
    return (x.shape[-1] == d and w_down.shape[1] == f and d % 8 == f % 8 == e % 8 == 0 and 8 <= d <= 1 << 20
            and 8 <= f <= 1 << 20 and 8 <= e <= 1 << 20)


@_dynamo_opaque
def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T``: x [..., d], w_gate and w_up [f, d], w_down [e, f],
    the result [..., e]; ``activation`` "silu", "gelu" (erf), "gelu_tanh" or "relu".

    bf16 or fp16, all of one dtype; under a 16-bit autocast fp32 tensors are cast to its dtype
    first, on every call (autocast's cache of weights is that of torch's own linears). d, e and f
    multiples of 8. Row strides and any number of rows, none included, are taken.
    Differentiable in every tensor; functorch's transforms, forward-mode differentiation,
    tracing and tensor subclasses take torch's ops instead. Other operands raise ``DsaltError``."""
    if activation not in _hip.ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_hip.ACTIVATIONS)}, got {activation!r}")
    if not gated_ffn_supported(x, w_gate, w_up, w_down):
        _hip.require_gpu(x, w_gate, w_up, w_down)
        raise _hip.DsaltError(
            f"gated_ffn needs bf16 or fp16 x [..., d], w_gate and w_up [f, d], w_down [e, f] of one dtype with d, e and f "
            f"multiples of 8 (got {[(tuple(t.shape), t.dtype) for t in (x, w_gate, w_up, w_down)]})")
    if torch.is_autocast_enabled("cuda"):
        dt = autocast_dtype(x)
        x, w_gate, w_up, w_down = x.to(dt), w_gate.to(dt), w_up.to(dt), w_down.to(dt)
    if not eager(x, w_gate, w_up, w_down):
        return torch_gated_ffn(x, w_gate, w_up, w_down, activation)
    if not torch.is_grad_enabled():
        return _run(x, w_gate, w_up, w_down, activation, False)[0]
    return _GatedFFN.apply(x, w_gate, w_up, w_down, activation)
