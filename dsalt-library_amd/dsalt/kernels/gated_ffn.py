"""The gated feed-forward block as one differentiable function on hand-written HIP kernels:
``act(x w_gate^T) * (x w_up^T)`` times ``w_down^T`` (SwiGLUFFN, dsalt_transformer.py:10-21, and
its GELU and ReLU relatives).

Both projections, the activation and the product are one kernel, and so are the gradient of
the product and the activation's gradient. Products accumulate in fp32; the hidden activation
and its gradients are rounded once, from fp32.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .. import _hip
from ._block_train import autocast_dtype, graph_grads, without_autocast
from ._sparse import no_graph
from .dsalt_triton_attn import _dynamo_opaque

_TORCH_ACT = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}


def torch_gated_ffn(x, w_gate, w_up, w_down, activation: str):
    """``gated_ffn`` in torch's ops."""
    return F.linear(_TORCH_ACT[activation](F.linear(x, w_gate)) * F.linear(x, w_up), w_down)


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        # what a gradient needs is saved, as three linears would: a weight changed in place before
        # the backward is refused where a gradient reads it
        need = ctx.needs_input_grad[:4]
        inner = any(need[:3])
        y, gate_up, act = _hip.gated_ffn(_hip.row_operand(x.detach().reshape(-1, x.shape[-1])),
                                         *(_hip.row_operand(w.detach()) for w in (w_gate, w_up, w_down)), activation,
                                         x.shape[:-1], inner)
        ctx.save_for_backward(x if inner else None, *((w_gate, w_up) if need[0] else (None, None)),
                              w_down if inner else None, gate_up, act)
        ws = w_gate, w_up, w_down
        ctx.dsalt = x.shape, ws, tuple(w._version for w in ws), activation
        return y

    @staticmethod
    @without_autocast
    def backward(ctx, dy):
        x, _, _, _, gate_up, act = ctx.saved_tensors
        shape, ws, versions, activation = ctx.dsalt
        need = ctx.needs_input_grad[:4]
        if torch.is_grad_enabled():  # a graph of the backward is wanted: torch's own ops
            if tuple(w._version for w in ws) != versions:
                raise RuntimeError("a weight of gated_ffn was changed in place before a backward that records a graph")
            if x is None:  # only w_down has a gradient
                dw, = graph_grads(lambda w: (F.linear(act.view(*shape[:-1], -1), w),), ws[2:], (dy,))
                return None, None, None, dw, None
            return *graph_grads(lambda *t: (torch_gated_ffn(*t, activation),), (x, *ws), (dy,)), None
        dy = _hip.row_operand(dy.reshape(-1, dy.shape[-1]))
        xr = None if x is None else _hip.row_operand(x.detach().reshape(-1, shape[-1]))
        dx, *dw = _hip.gated_ffn_bwd(xr, *(_hip.row_operand(w.detach()) for w in ws), activation, gate_up, act, dy, need)
        return None if dx is None else dx.view(shape), *dw, None


def gated_ffn_supported(x, w_gate, w_up, w_down) -> bool:
    """Whether `gated_ffn` takes these tensors: bf16 or fp16 on one GPU (fp32 ones under a 16-bit
    autocast are cast), x [..., d], w_gate and w_up [f, d], w_down [e, f] with d, e and f
    multiples of 8."""
    ts = (x, w_gate, w_up, w_down)
    if any(t.device.type != "cuda" or t.device != x.device for t in ts) or x.dim() < 1 or any(w.dim() != 2 for w in ts[1:]):
        return False
    dt = autocast_dtype(x)
    if dt not in (torch.bfloat16, torch.float16):
        return False
    if any(t.dtype != dt and not (t.dtype == torch.float32 and torch.is_autocast_enabled("cuda")) for t in ts):
        return False
    f, d = w_gate.shape
    return (w_up.shape == (f, d) and w_down.shape[1] == f and x.shape[-1] == d
            and all(n >= 8 and n % 8 == 0 and n <= 1 << 20 for n in (d, f, w_down.shape[0])))


@_dynamo_opaque
def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T``: x [..., d], w_gate and w_up [f, d], w_down [e, f],
    the result [..., e]; ``activation`` "silu", "gelu" (erf), "gelu_tanh" or "relu".

    bf16 or fp16, all of one dtype; under a 16-bit autocast fp32 tensors are cast to its dtype
    first. d, e and f multiples of 8. Row strides and any number of rows, none included, are
    taken. Differentiable in every tensor. Other operands raise ``DsaltError``."""
    if activation not in _hip.ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(_hip.ACTIVATIONS)}, got {activation!r}")
    _hip.require_gpu(x, w_gate, w_up, w_down)
    if not gated_ffn_supported(x, w_gate, w_up, w_down):
        raise _hip.DsaltError(
            f"gated_ffn needs bf16 or fp16 x [..., d], w_gate and w_up [f, d], w_down [e, f] of one dtype with d, e and f "
            f"multiples of 8 (got {[(tuple(t.shape), t.dtype) for t in (x, w_gate, w_up, w_down)]})")
    dt = autocast_dtype(x)
    x, w_gate, w_up, w_down = (t if t.dtype == dt else t.to(dt) for t in (x, w_gate, w_up, w_down))
    if no_graph(x, w_gate, w_up, w_down):
        return _hip.gated_ffn(_hip.row_operand(x.reshape(-1, x.shape[-1])),
                              *(_hip.row_operand(w) for w in (w_gate, w_up, w_down)), activation, x.shape[:-1], False)[0]
    return _GatedFFN.apply(x, w_gate, w_up, w_down, activation)
