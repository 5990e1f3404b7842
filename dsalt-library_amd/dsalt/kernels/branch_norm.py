"""A block's branch joined to its residual stream in one pass forward and one backward: dropout
and RMSNorm of the branch's output, its gate, the scaled residual sum, and the RMSNorm that
the next branch reads (the pre-norm block of dsalt_transformer.py:81-84 with a norm after its
branch, a layer scale or token gate and a residual scale).
"""
from __future__ import annotations

import torch

from .. import _hip
from ._block_train import eager, graph_grads, without_autocast
from .dropout import check_seed, counter_dropout
from .dsalt_triton_attn import _dynamo_opaque


def torch_branch_norm(x, h, weight, post_weight, gate, opts, seed):
    """``branch_norm`` in torch's ops and ``counter_dropout``, in fp32 or more."""
    residual_scale, p, offset, eps, post_eps, out_dtype = opts

    def wide(t):
        return t.float() if t.dtype in (torch.bfloat16, torch.float16) else t

    def norm(t, w, e):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + e) * wide(w)

    n = wide(h)
    if _hip.keep_threshold(p) < 65536:
        n = counter_dropout(n, p, seed, offset)
    if post_weight is not None:
        n = norm(n, post_weight, post_eps)
    z = residual_scale * wide(x) + (n if gate is None else wide(gate) * n)
    return z.to(x.dtype), None if weight is None else norm(z, weight, eps).to(out_dtype)


class _BranchNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, weight, post_weight, gate, seed, opts):
        ctx.set_materialize_grads(False)
        x_out, y, stats = _hip.branch_norm(*_operands(x, h, weight, post_weight, gate), opts, seed, True)
        is_tensor = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(x, h, weight, post_weight, gate, stats, seed if is_tensor else None)
        ctx.dsalt = opts, None if is_tensor else seed
        return x_out, y

    @staticmethod
    @without_autocast
    def backward(ctx, dx_out, dy):
        x, h, weight, post_weight, gate, stats, seed = ctx.saved_tensors
        opts, seed_value = ctx.dsalt
        seed = seed_value if seed is None else seed
        need = ctx.needs_input_grad[:5]
        if dx_out is None and dy is None:
            return (None,) * 7
        if torch.is_grad_enabled():  # a graph of the backward is wanted: torch's own ops
            grads = graph_grads(lambda *t: tuple(o for o in torch_branch_norm(*t, opts, seed) if o is not None),
                                (x, h, weight, post_weight, gate), (dx_out, dy) if weight is not None else (dx_out,))
            return *grads, None, None
        if dy is None and need[2]:  # without a gradient of y, none of its norm's weight
            need = (*need[:2], False, *need[3:])
        grads = _hip.branch_norm_bwd(*_operands(x, h, weight, post_weight, gate), opts, seed, stats,
                                     None if dx_out is None else _hip.aligned_rows(dx_out),
                                     None if dy is None else _hip.aligned_rows(dy), need)
        return *grads, None, None


def _operands(x, h, weight, post_weight, gate):
    rows = _hip.aligned_rows
    return (rows(x), rows(h), None if weight is None else rows(weight), None if post_weight is None else rows(post_weight),
            None if gate is None else rows(gate))


def _weight_ok(w, d: int, dtype: torch.dtype, dev: torch.device) -> bool:
    return w is None or (w.shape == (d,) and (w.dtype is dtype or w.dtype is torch.float32) and w.device == dev)


@_dynamo_opaque
def branch_norm(x: torch.Tensor, h: torch.Tensor, weight: torch.Tensor | None = None, *,
                post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                p: float = 0.0, seed=None, offset: int = 0, eps: float = 1e-6, post_eps: float | None = None,
                out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(x_out, y)`` of the residual stream x [..., d] and a branch's output h of its shape::

        n     = rms_norm(dropout(h, p)) * post_weight      (without post_weight: dropout(h, p))
        x_out = residual_scale * x + gate * n
        y     = rms_norm(x_out) * weight                   (None without weight)

    The dropout is ``counter_dropout(h, p, seed, offset)``. ``gate``: per channel [d], per token
    [..., 1], or none. x bf16, fp16 or fp32; h and ``out_dtype`` (y's type, by default x's) x's
    dtype, or any of the three beside an fp32 x; weights and gate in x's dtype or fp32. x_out has
    x's dtype; y is formed from the sum before that rounding. d a multiple of 8 up to 8192.
    Differentiable in x, h, weight, post_weight and gate; functorch's transforms, forward-mode
    differentiation, tracing and tensor subclasses take torch's ops instead. Other operands raise
    ``DsaltError``."""
    dev, dtype = x.device, x.dtype
    out_dtype = dtype if out_dtype is None else out_dtype
    check_seed(p, seed, offset, dev)
    d = x.shape[-1] if x.dim() else 0
    wide = dtype is torch.float32
    ok = (dev.type == "cuda" and h.device == dev and dtype in _hip._SCORE_DTYPES and h.shape == x.shape
          and 8 <= d <= _hip.BRANCH_NORM_MAX_DIM and d % 8 == 0
          and (h.dtype is dtype or (wide and h.dtype in _hip._SCORE_DTYPES))
          and (out_dtype is dtype or (wide and out_dtype in _hip._SCORE_DTYPES))
          and _weight_ok(weight, d, dtype, dev) and _weight_ok(post_weight, d, dtype, dev)
          and (gate is None or ((gate.shape == (d,) or gate.shape == (*x.shape[:-1], 1)) and gate.device == dev
                                and (gate.dtype is dtype or gate.dtype is torch.float32))))
    if not ok:
        _hip.require_gpu(x, h, weight, post_weight, gate)
        raise _hip.DsaltError(
            f"branch_norm needs x and h [..., d] of one shape, d a multiple of 8 up to {_hip.BRANCH_NORM_MAX_DIM}, h and the "
            f"output in x's dtype or x fp32, weights [d] and a gate [d] or [..., 1] in x's dtype or fp32 (got "
            f"{[None if t is None else (tuple(t.shape), t.dtype) for t in (x, h, weight, post_weight, gate)]}, {out_dtype})")
    opts = (float(residual_scale), p, offset, float(eps), float(eps if post_eps is None else post_eps), out_dtype)
    tensors = (x, h, weight, post_weight, gate, seed if isinstance(seed, torch.Tensor) else None)
    if not eager(*(t for t in tensors if t is not None)):
        return torch_branch_norm(x, h, weight, post_weight, gate, opts, seed)
    if not torch.is_grad_enabled():
        return _hip.branch_norm(*_operands(x, h, weight, post_weight, gate), opts, seed, False)[:2]
    return _BranchNorm.apply(x, h, weight, post_weight, gate, seed, opts)
