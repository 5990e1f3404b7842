"""Layer norm of rows, and of a residual stream with a branch added, as one pass forward and one
backward each, and the module that holds its weights: the norm of blocks that centre their rows, beside
the RMSENorm of dsalt/kernels/RMSENorm.py:6-22.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _hip
from ._block_train import eager, graph_grads, keep, kept, without_autocast
from .dsalt_triton_attn import _dynamo_opaque


def torch_layer_norm(x, h, weight, bias, eps: float, out_dtype: torch.dtype):
    """``(x_out, y)`` of ``add_layer_norm`` (without h: ``(y,)``) in torch's ops, in fp32 or more."""
    def wide(t):
        return t.float() if t is not None and t.dtype in (torch.bfloat16, torch.float16) else t

    z = wide(x) if h is None else wide(x) + wide(h)
    y = F.layer_norm(z, z.shape[-1:], None, None, eps)
    y = y if weight is None else y * wide(weight)
    y = (y if bias is None else y + wide(bias)).to(out_dtype)
    return (y,) if h is None else (z.to(x.dtype), y)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, weight, bias, eps, out_dtype):
        ctx.set_materialize_grads(False)
        x_out, y, stats = _hip.layer_norm(*_operands(x, h, weight, bias), eps, out_dtype, True)
        # an fp32 sum is what the backward normalises; a 16-bit one has lost bits of it
        whole = h is not None and x.dtype is torch.float32
        keep(ctx, x_out if whole else x, None if whole else h, weight, bias, stats)
        ctx.dsalt = h is not None, whole, None if h is None else h.dtype, eps, out_dtype
        return y if h is None else (x_out, y)

    @staticmethod
    @without_autocast
    def backward(ctx, *grads):
        x, h, weight, bias, stats = kept(ctx)
        add, whole, h_dtype, eps, out_dtype = ctx.dsalt
        dx_out, dy = grads if add else (None, *grads)
        need_x, need_h, need_w, need_b = ctx.needs_input_grad[:4]
        if dy is None:
            dh = dx_out.to(h_dtype) if need_h and dx_out is not None else None
            return dx_out if need_x else None, dh, None, None, None, None
        if torch.is_grad_enabled():  # a graph of the backward is wanted: torch's own ops
            dx, dh, dw, db = graph_grads(lambda *t: torch_layer_norm(*t, eps, out_dtype), (x, h, weight, bias),
                                         (dx_out, dy) if h is not None else (dy,))
            if whole:  # of the sum, which x and h enter alike
                dx = dx_out if dx is None else dx if dx_out is None else dx + dx_out
                dh = dx.to(h_dtype) if need_h and dx is not None else None
            return dx if need_x else None, dh, dw, db, None, None
        same = need_h and h_dtype is x.dtype  # the branch's gradient is then the residual's
        rows = _hip.contiguous_rows
        x, h, weight, bias = _operands(x, h, weight, bias)
        dx, dh, dw, db = _hip.layer_norm_bwd(x, h, weight, None if bias is None else bias.dtype, stats,
                                             None if dx_out is None else rows(dx_out), rows(dy), h_dtype if need_h else None,
                                             (need_x or same, need_h and not same, need_w, need_b))
        return dx if need_x else None, dx if same else dh, dw, db, None, None


def _operands(*ts):
    return tuple(None if t is None else _hip.contiguous_rows(t) for t in ts)


def _supported(x, h, weight, bias, out_dtype) -> bool:
    dev, dtype = x.device, x.dtype
    wide = dtype is torch.float32
    d = x.shape[-1] if x.dim() else 0

    def vector(w):
        return w is None or (w.shape == (d,) and (w.dtype is dtype or w.dtype is torch.float32) and w.device == dev)

    def branch(dt):
        return dt is dtype or (wide and dt in _hip._SCORE_DTYPES)

    return (dev.type == "cuda" and dtype in _hip._SCORE_DTYPES and 1 <= d <= _hip.LAYER_NORM_MAX_DIM
            and x.numel() // d < 1 << 31 and branch(out_dtype) and vector(weight) and vector(bias)
            and (h is None or (h.device == dev and h.shape == x.shape and branch(h.dtype))))


def _call(what, x, h, weight, bias, eps, out_dtype):
    eps = float(eps)
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0 (got {eps})")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if not _supported(x, h, weight, bias, out_dtype):
        _hip.require_gpu(x, h, weight, bias)
        raise _hip.DsaltError(
            f"{what} needs x [..., d] in bf16, fp16 or fp32 with d up to {_hip.LAYER_NORM_MAX_DIM}, a branch of its shape, the "
            f"branch and the output in x's dtype or x fp32, weight and bias [d] in x's dtype or fp32 (got "
            f"{[None if t is None else (tuple(t.shape), t.dtype) for t in (x, h, weight, bias)]}, {out_dtype})")
    if not eager(*(t for t in (x, h, weight, bias) if t is not None)):
        out = torch_layer_norm(x, h, weight, bias, eps, out_dtype)
        return out[0] if h is None else out
    if not torch.is_grad_enabled():
        x_out, y, _ = _hip.layer_norm(*_operands(x, h, weight, bias), eps, out_dtype, False)
        return y if h is None else (x_out, y)
    return _LayerNorm.apply(x, h, weight, bias, eps, out_dtype)


@_dynamo_opaque
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension of x [..., d], in
    ``out_dtype`` (by default x's).

    x bf16, fp16 or fp32; ``out_dtype`` x's dtype, or any of the three of an fp32 x; weight and bias
    [d] in x's dtype or fp32, or None. Any d up to 8192, any strides (rows that are not contiguous are
    copied). Statistics and sums are fp32; each result is rounded once. Differentiable in x, weight and
    bias; functorch's transforms, forward-mode differentiation, tracing and tensor subclasses take
    torch's ops instead. Other operands raise ``DsaltError``."""
    return _call("layer_norm", x, None, weight, bias, eps, out_dtype)


@_dynamo_opaque
def add_layer_norm(x: torch.Tensor, h: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   eps: float = 1e-5, out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(x_out, y)``: the residual stream x [..., d] with a branch's output h of its shape added, and the
    layer norm of that sum, formed before its rounding to x's dtype. h in x's dtype, or any
    of bf16, fp16 and fp32 beside an fp32 x; otherwise as ``layer_norm``. Differentiable in h too."""
    return _call("add_layer_norm", x, h, weight, bias, eps, out_dtype)


class LayerNorm(nn.Module):
    """Layer norm over the last dimension with a learned scale and shift, in x's dtype (or ``out_dtype``):
    ``layer_norm`` on the GPU, torch's ops on the CPU. Called with a branch it returns ``(x + branch, norm)``
    (``add_layer_norm``)."""

    def __init__(self, d_model: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.eps = eps
        self.normalized_shape = (d_model,)
        self.weight = nn.Parameter(torch.ones(d_model))
        self.bias = nn.Parameter(torch.zeros(d_model)) if bias else None

    def forward(self, x: torch.Tensor, branch: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
        w, b = ((t if t is None or t.dtype is x.dtype else t.float()) for t in (self.weight, self.bias))
        if not x.is_cuda:
            out = torch_layer_norm(x, branch, w, b, self.eps, x.dtype if out_dtype is None else out_dtype)
            return out[0] if branch is None else out
        if branch is None:
            return layer_norm(x, w, b, self.eps, out_dtype)
        return add_layer_norm(x, branch, w, b, self.eps, out_dtype)

    def extra_repr(self) -> str:
        return f"{self.normalized_shape[0]}, eps={self.eps}, bias={self.bias is not None}"
