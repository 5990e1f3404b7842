"""Matrix products in 8-bit floats (e4m3) with a scale for each block of 128, for inference: the
quantisation of weights and activations, the product, and a linear layer on them, for the projections
of dsalt/modules/dsalt_transformer.py and dsalt/model/dsalt_lm.py.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _hip
from .._hip import E4M3, E8M0, FP8_BLOCK
from ._block_train import autocast_dtype, eager
from .dsalt_triton_attn import _dynamo_opaque


def _spread(scale: torch.Tensor, q: torch.Tensor, tile: bool) -> torch.Tensor:
    s = scale.float().repeat_interleave(FP8_BLOCK, -1)[..., :q.shape[-1]]
    return s.repeat_interleave(FP8_BLOCK, -2)[..., :q.shape[-2], :] if tile else s


def torch_fp8_quantize(x: torch.Tensor, tile: bool, scale_dtype: torch.dtype):
    """``fp8_quantize`` in torch's ops, the same bits."""
    k = x.shape[-1]
    pad = F.pad(x.float(), (0, -k % FP8_BLOCK, 0, -x.shape[-2] % FP8_BLOCK if tile else 0) if tile else (0, -k % FP8_BLOCK))
    v = pad.unflatten(-1, (-1, FP8_BLOCK))
    v = v.unflatten(-3, (-1, FP8_BLOCK)) if tile else v
    dims = (-3, -1) if tile else (-1,)
    amax = v.abs().amax(dims, keepdim=True)
    m, e = torch.frexp(amax)
    power = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-127)
    scale = torch.where(amax > 0, torch.exp2(power.to(amax.dtype)), 1.0)
    scale = torch.where(amax < float("inf"), scale, float("nan"))
    q = (v / scale).reshape(pad.shape)[..., :x.shape[-2] if x.dim() > 1 else None, :k] if tile else (v / scale).flatten(-2)[..., :k]
    scale = scale.squeeze(-1) if not tile else scale.squeeze(-1).squeeze(-2)
    return q.to(E4M3), scale.to(scale_dtype)


def torch_fp8_matmul(a, a_scale, b, b_scale, bias, out_dtype):
    """``fp8_matmul`` in torch's ops, in fp32."""
    y = (a.float() * _spread(a_scale, a, False)) @ (b.float() * _spread(b_scale, b, True)).t()
    return (y if bias is None else y + bias.float()).to(out_dtype)


def _blocks(n: int) -> int:
    return -(-n // FP8_BLOCK)


def _weight_ok(b, b_scale, bias, dev) -> bool:
    return (b.dim() == 2 and b.dtype is E4M3 and b.device == dev and 1 <= b.shape[0] <= 1 << 20 and 16 <= b.shape[1] <= 1 << 20
            and b.shape[1] % 16 == 0 and b_scale.shape == (_blocks(b.shape[0]), _blocks(b.shape[1]))
            and b_scale.dtype in (torch.float32, E8M0) and b_scale.device == dev
            and (bias is None or (bias.shape == (b.shape[0],) and bias.dtype in _hip._SCORE_DTYPES and bias.device == dev)))


def _scale(s: torch.Tensor) -> torch.Tensor:
    return s if all(1 <= t <= 1 << 21 for t in s.stride()) else s.clone(memory_format=torch.contiguous_format)


def _no_grad(*ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise _hip.DsaltError("8-bit products and quantisation are for inference: call them under torch.no_grad(), or on tensors "
                              "that require no gradient")


@_dynamo_opaque
def fp8_quantize(x: torch.Tensor, tile: bool = False, scale_dtype: torch.dtype = E8M0) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` of x [..., k]: 8-bit floats (``torch.float8_e4m3fn``) of x's shape, contiguous, and the
    scales that they are multiplied by, one for each 128 elements of a row ([..., ceil(k / 128)]: an
    activation) or, with ``tile``, of x [n, k] for each tile of 128 x 128 ([ceil(n / 128), ceil(k / 128)]: a
    weight).

    A scale is the smallest power of two that brings its block's largest magnitude to at most 448 (1 for a
    block of zeros), as ``torch.float8_e8m0fnu`` or ``torch.float32``; x over it is rounded to nearest even. A
    block that holds an infinity or NaN becomes NaN. x bf16, fp16 or fp32, k up to 2^20, any strides. For
    inference: x that requires a gradient is refused where gradients are recorded. Other operands raise ``DsaltError``."""
    k = x.shape[-1] if x.dim() else 0
    ok = (x.device.type == "cuda" and x.dtype in _hip._SCORE_DTYPES and 1 <= k <= 1 << 20 and scale_dtype in (torch.float32, E8M0)
          and (not tile or x.dim() == 2) and x.numel() // k <= 1 << 30
          and (_blocks(x.shape[0]) if tile else -(-(x.numel() // k) // 64)) * _blocks(k) <= 1 << 23)
    if not ok:
        _hip.require_gpu(x)
        raise _hip.DsaltError(f"fp8_quantize needs bf16, fp16 or fp32 x [..., k], [n, k] for tiles, and fp32 or e8m0 scales "
                              f"(got {tuple(x.shape)} {x.dtype}, {scale_dtype})")
    _no_grad(x)
    if not eager(x):
        return torch_fp8_quantize(x, tile, scale_dtype)
    if x.dim() == 2:
        return _hip.fp8_quantize(_hip.unit_rows(x), tile, scale_dtype is torch.float32)
    q, s = _hip.fp8_quantize(_hip.unit_rows(x.reshape(-1, k)), tile, scale_dtype is torch.float32)
    return q.view(x.shape), s.view(*x.shape[:-1], s.shape[-1])


@_dynamo_opaque
def fp8_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T + bias`` [..., n] of 8-bit floats (``torch.float8_e4m3fn``) a [..., k] and b [n, k] with the
    scales that ``fp8_quantize`` gives: a_scale [..., ceil(k / 128)] and b_scale [ceil(n / 128),
    ceil(k / 128)], ``torch.float8_e8m0fnu`` or any values in fp32 whose products fp32 holds, each its own. One rounding to
    ``out_dtype`` (bf16, fp16 or fp32); bias [n] in any of those. Sums are fp32, but for those of each eight consecutive k, which
    the matrix instruction adds to 13 bits below their largest product: an error of at most 7 * 2^-13 of it, 1.5e-5 of a
    result of normal values (2-norm), more than fp32's where ``out_dtype`` is that.

    k a multiple of 16; k and n up to 2^20; any strides (rows that are not 16-byte aligned are copied). For
    inference: operands that require a gradient are refused where gradients are recorded. Other operands raise
    ``DsaltError``."""
    dev, k = a.device, a.shape[-1] if a.dim() else 0
    ok = (dev.type == "cuda" and a.dtype is E4M3 and _weight_ok(b, b_scale, bias, dev) and k == b.shape[1]
          and a_scale.shape == (*a.shape[:-1], _blocks(k)) and a_scale.dtype in (torch.float32, E8M0) and a_scale.device == dev
          and out_dtype in _hip._SCORE_DTYPES and a.numel() // k <= 1 << 24 and a.numel() // k * b.shape[0] <= 1 << 38)
    if not ok:
        _hip.require_gpu(a, a_scale, b, b_scale, bias)
        raise _hip.DsaltError(
            f"fp8_matmul needs e4m3 a [..., k] and b [n, k], k a multiple of 16, fp32 or e8m0 scales [..., ceil(k / 128)] and "
            f"[ceil(n / 128), ceil(k / 128)], a bias [n] (got "
            f"{[None if t is None else (tuple(t.shape), t.dtype) for t in (a, a_scale, b, b_scale, bias)]}, {out_dtype})")
    _no_grad(a, a_scale, b, b_scale, bias)
    if not eager(*(t for t in (a, a_scale, b, b_scale, bias) if t is not None)):
        return torch_fp8_matmul(a, a_scale, b, b_scale, bias, out_dtype)
    if a_scale.dtype is not b_scale.dtype:  # the kernel takes both alike
        a_scale, b_scale = a_scale.float(), b_scale.float()
    flat, s = (a, a_scale) if a.dim() == 2 else (a.reshape(-1, k), a_scale.reshape(-1, a_scale.shape[-1]))
    return _hip.fp8_matmul(_hip.fp8_operand(flat), _scale(s), _hip.fp8_operand(b), _scale(b_scale),
                           None if bias is None else _hip.contiguous_rows(bias), a.shape[:-1], out_dtype)


@_dynamo_opaque
def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``fp8_matmul(*fp8_quantize(x), weight, weight_scale, bias)`` of x [..., k] in bf16, fp16 or fp32, in
    ``out_dtype`` (by default x's), with its precision; up to 32 rows are quantised by the product's kernel as it reads
    them, to the same 8-bit values. weight [n, k] and its scales as ``fp8_matmul`` takes b. For inference: operands
    that require a gradient are refused where gradients are recorded."""
    dev, k = x.device, x.shape[-1] if x.dim() else 0
    out_dtype = x.dtype if out_dtype is None else out_dtype
    ok = (dev.type == "cuda" and x.dtype in _hip._SCORE_DTYPES and out_dtype in _hip._SCORE_DTYPES
          and _weight_ok(weight, weight_scale, bias, dev) and k == weight.shape[1]
          and x.numel() // k <= 1 << 24 and x.numel() // k * weight.shape[0] <= 1 << 38)
    if not ok:
        _hip.require_gpu(x, weight, weight_scale, bias)
        raise _hip.DsaltError(
            f"fp8_linear needs bf16, fp16 or fp32 x [..., k], e4m3 weight [n, k], k a multiple of 16, fp32 or e8m0 scales "
            f"[ceil(n / 128), ceil(k / 128)], a bias [n] (got "
            f"{[None if t is None else (tuple(t.shape), t.dtype) for t in (x, weight, weight_scale, bias)]}, {out_dtype})")
    _no_grad(x, weight, weight_scale, bias)
    if not eager(*(t for t in (x, weight, weight_scale, bias) if t is not None)):
        return torch_fp8_matmul(*torch_fp8_quantize(x, False, torch.float32), weight, weight_scale, bias, out_dtype)
    flat = x if x.dim() == 2 else x.reshape(-1, k)
    weight, ws = _hip.fp8_operand(weight), _scale(weight_scale)
    bias = None if bias is None else _hip.contiguous_rows(bias)
    if flat.shape[0] <= _hip.FP8_FEW_ROWS:
        return _hip.fp8_matmul(_hip.fp8_operand(flat), None, weight, ws, bias, x.shape[:-1], out_dtype)
    q, s = _hip.fp8_quantize(_hip.unit_rows(flat), False, ws.dtype is torch.float32)
    return _hip.fp8_matmul(q, s, weight, ws, bias, x.shape[:-1], out_dtype)


class FP8Linear(nn.Module):
    """A frozen linear layer in 8 bits (``fp8_linear``): ``FP8Linear.from_linear`` quantises an nn.Linear's
    weight by tiles of 128 x 128. The weight and its scales are kept as bytes, which ``.to(dtype)`` leaves as they are.
    The result has x's dtype, or autocast's. GPU tensors only, for inference."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, device=None, dtype=None):
        super().__init__()
        if in_features < 16 or in_features % 16:
            raise ValueError(f"in_features must be a multiple of 16 (got {in_features})")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("weight_bits", torch.zeros(out_features, in_features, device=device, dtype=torch.uint8))
        self.register_buffer("scale_bits", torch.full((_blocks(out_features), _blocks(in_features)), 127, device=device,
                                                      dtype=torch.uint8))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype), requires_grad=False) if bias else None

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "FP8Linear":
        """The layer of a linear layer on the GPU, whose weight it does not keep."""
        w = linear.weight.detach()
        out = cls(linear.in_features, linear.out_features, linear.bias is not None, w.device, w.dtype)
        q, s = fp8_quantize(w, tile=True)
        out.weight_bits.copy_(q.view(torch.uint8))
        out.scale_bits.copy_(s.view(torch.uint8))
        if linear.bias is not None:
            out.bias.copy_(linear.bias.detach())
        return out.train(linear.training)

    @property
    def weight_q(self) -> torch.Tensor:
        return self.weight_bits.view(E4M3)

    @property
    def weight_scale(self) -> torch.Tensor:
        return self.scale_bits.view(E8M0)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp8_linear(x, self.weight_q, self.weight_scale, self.bias, autocast_dtype(x))

    def extra_repr(self) -> str:
        return f"{self.in_features}, {self.out_features}, bias={self.bias is not None}"
