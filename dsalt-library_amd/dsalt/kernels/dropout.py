"""Dropout whose mask is a function of a seed and the element's index, so that it is never stored:
the backward forms it again. ``nn.Dropout`` draws from torch's generator and keeps the mask.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from .. import _hip
from ._block_train import eager
from .dsalt_triton_attn import _dynamo_opaque


def draw_seed(device: torch.device) -> torch.Tensor:
    """A seed [1] (int64) on the GPU from torch's generator of that device: it follows
    ``torch.manual_seed`` and the generator state that checkpointing restores, costs no
    synchronisation, and a captured graph draws a new one on every replay."""
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), device=device, dtype=torch.int64)


def check_seed(p: float, seed, offset: int, device: torch.device) -> None:
    threshold = _hip.keep_threshold(p)
    if seed is None:
        if threshold < 65536:
            raise ValueError("a dropout probability above 0 needs a seed")
    else:
        _hip.check_seed(seed, device)
    if not 0 <= operator.index(offset) < 2 ** 63:
        raise ValueError(f"offset must be in [0, 2^63) (got {offset})")


def torch_counter_dropout(x: torch.Tensor, p: float, seed, offset: int = 0) -> torch.Tensor:
    """``counter_dropout`` in torch's ops, the same bits: Philox4x32 with 7 rounds at counter (i / 8, offset)
    under key seed in int64 arithmetic, 16 bits for each of eight consecutive elements."""
    threshold, low, n = _hip.keep_threshold(p), 0xFFFFFFFF, x.numel()
    seed, offset = seed if isinstance(seed, torch.Tensor) else operator.index(seed), operator.index(offset)
    ctr = torch.arange(-(-n // 8), device=x.device)
    c0, c1, c2, c3 = ctr & low, ctr >> 32, torch.full_like(ctr, offset & low), torch.full_like(ctr, offset >> 32)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits of the products
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), -1)
    keep = (torch.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)[:n] < threshold).view(x.shape)
    scale = ctypes.c_float(65536 / threshold if threshold else 0.0).value  # in fp32, as the kernels hold it
    return torch.where(keep, x.float() * scale, 0.0).to(x.dtype)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        is_tensor = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(seed if is_tensor else None)
        ctx.dsalt = p, None if is_tensor else seed, offset
        return _hip.dropout(_hip.aligned_rows(x), p, seed, offset)

    @staticmethod
    def backward(ctx, dy):
        p, seed, offset = ctx.dsalt
        saved, = ctx.saved_tensors
        seed = seed if saved is None else saved
        if not torch.is_grad_enabled():
            return _hip.dropout(_hip.aligned_rows(dy), p, seed, offset), None, None, None
        # a graph of the backward is wanted: linear, its gradient is the same function again
        return _Dropout.apply(dy, p, seed, offset), None, None, None


@_dynamo_opaque
def counter_dropout(x: torch.Tensor, p: float, seed, offset: int = 0) -> torch.Tensor:
    """Dropout of x with probability p: a kept element is scaled by the inverse of the probability
    of keeping, a dropped one is 0 whatever it holds. p is taken to the nearest multiple of
    2^-16, and the scale is of that p.

    The mask depends on ``seed`` (an int of 64 bits, or one int64 element on x's GPU, read when
    the kernel runs: a replayed graph sees its new value), ``offset`` (0 to 2^63 - 1: tells
    apart the places that use one seed) and the element's index in x's logical order, and
    on nothing else. bf16, fp16 or fp32 of any shape. Differentiable in x; a seed tensor
    changed in place before the backward is refused. Under functorch's transforms, forward-mode
    differentiation and tracing, and for tensor subclasses, torch's ops run instead, with the
    same bits (under vmap an example's element has its index in the example)."""
    dev = _hip.require_gpu(x)
    if x.dtype not in _hip._SCORE_DTYPES:
        raise _hip.DsaltError(f"counter_dropout needs a bf16, fp16 or fp32 tensor (got {x.dtype})")
    check_seed(p, seed, offset, dev)
    seed = 0 if seed is None else seed
    if not eager(x, *((seed,) if isinstance(seed, torch.Tensor) else ())):
        return torch_counter_dropout(x, p, seed, offset)
    if not torch.is_grad_enabled():
        return _hip.dropout(_hip.aligned_rows(x), p, seed, offset)
    return _Dropout.apply(x, p, seed, offset)
