"""The loss of a student's logits against a teacher's top logits and against labels, with its gradient:
beside the labels' cross-entropy of dsalt/model/dsalt_lm.py, for a model that is trained on what a
larger one would answer.
"""
from __future__ import annotations

import torch

from .. import _hip
from ._block_train import eager, graph_grads, keep, kept, without_autocast
from .dsalt_triton_attn import _dynamo_opaque


def torch_distill_loss(logits, teacher, ids, labels, opts):
    """``distill_loss`` in torch's ops, in fp32 or more."""
    temperature, label_weight, ignore_index, reduction = opts
    s = logits.float() if logits.dtype in (torch.bfloat16, torch.float16) else logits
    vocab = s.shape[-1]
    z = teacher.to(s.dtype)
    counted = None
    if labels is not None:
        counted = (labels != ignore_index) & (labels >= 0) & (labels < vocab)
        s, z = (torch.where(counted.unsqueeze(-1), t, 0.0) for t in (s, z))  # no gradient through what such rows hold
    on = (ids >= 0) & (ids < vocab) & (z != float("-inf"))
    at = torch.where(on, ids, 0).long()
    low = torch.finfo(s.dtype).min
    z = z - torch.where(on, z, low).amax(-1, keepdim=True)  # first: the lowest value has no finite quotient by less than 1
    log_p = torch.log_softmax(torch.where(on, z / temperature, low), -1)
    p = torch.where(on, log_p.exp(), 0.0)  # of a row without slots, too
    log_q = torch.log_softmax((s - s.detach().amax(-1, keepdim=True)) / temperature, -1).gather(-1, at)
    rows = torch.where(p > 0, p * (log_p - log_q), torch.where(on, p, 0.0)).sum(-1) * ((1 - label_weight) * temperature ** 2)
    if label_weight == 1:  # the teacher's term, which may be infinite, is not there
        rows = torch.zeros_like(rows)
    if labels is not None:
        if label_weight:
            at = torch.where(counted, labels, 0).long().unsqueeze(-1)
            rows = rows - label_weight * torch.log_softmax(s, -1).gather(-1, at).squeeze(-1)
        rows = torch.where(counted, rows, 0.0)
    if reduction == "none":
        return rows
    n = 1 if reduction == "sum" else max(rows.numel(), 1) if labels is None else counted.sum().clamp(min=1)
    return rows.sum() / n


def _options(labels, temperature, label_weight, ignore_index, reduction):
    """The options as the kernels take them; values outside their ranges are refused."""
    if reduction not in _hip.REDUCTIONS:
        raise ValueError(f"reduction must be one of {list(_hip.REDUCTIONS)}, got {reduction!r}")
    temperature, label_weight = float(temperature), float(label_weight)
    if not 2.0 ** -63 <= temperature < 2.0 ** 63:  # its inverse and its square in fp32
        raise ValueError(f"temperature must be in [2^-63, 2^63) (got {temperature})")
    if not 0 <= label_weight <= 1:
        raise ValueError(f"label_weight must be in [0, 1] (got {label_weight})")
    if label_weight > 0 and labels is None:
        raise ValueError("label_weight needs labels")
    return temperature, label_weight, int(ignore_index), reduction


def _fit(logits, teacher_logits, teacher_ids, labels, dtypes) -> bool:
    """Whether the operands' shapes, types (of `dtypes`) and devices go together."""
    dev, lead, ints = logits.device, logits.shape[:-1], (torch.int32, torch.int64)
    return (logits.dtype in dtypes and teacher_logits.dtype in dtypes
            and teacher_ids.dtype in ints and logits.dim() >= 1 and 1 <= logits.shape[-1] <= 1 << 30
            and teacher_logits.shape == teacher_ids.shape and teacher_ids.shape[:-1] == lead and teacher_ids.dim() == logits.dim()
            and 1 <= teacher_ids.shape[-1] <= _hip.DISTILL_MAX_K and teacher_logits.device == dev and teacher_ids.device == dev
            and (labels is None or (labels.shape == lead and labels.dtype in ints and labels.device == dev))
            and lead.numel() < 1 << 24)


def _refuse(*operands):
    raise _hip.DsaltError(
        f"distill_loss needs bf16, fp16 or fp32 logits [..., V] and teacher_logits [..., K], int32 or int64 teacher_ids "
        f"[..., K] and labels [...], K up to {_hip.DISTILL_MAX_K} (got "
        f"{[None if t is None else (tuple(t.shape), t.dtype) for t in operands]})")


def cpu_distill_loss(logits, teacher_logits, teacher_ids, labels=None, *, temperature=1.0, label_weight=0.0, ignore_index=-100,
                     reduction="mean"):
    """``distill_loss`` of CPU tensors (of float64 too) in torch's ops, with its checks: for the models."""
    opts = _options(labels, temperature, label_weight, ignore_index, reduction)
    if not _fit(logits, teacher_logits, teacher_ids, labels, (*_hip._SCORE_DTYPES, torch.float64)):
        _refuse(logits, teacher_logits, teacher_ids, labels)
    return torch_distill_loss(logits, teacher_logits.detach(), teacher_ids, labels, opts)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, ids, labels, opts):
        loss, stats = _hip.distill(logits, teacher, ids, labels, opts, True)
        keep(ctx, logits, teacher, ids, labels, stats)
        ctx.dsalt = opts
        return loss

    @staticmethod
    @without_autocast
    def backward(ctx, d_loss):
        logits, teacher, ids, labels, stats = kept(ctx)
        if torch.is_grad_enabled():  # a graph of the backward is wanted: torch's own ops
            d, = graph_grads(lambda s: (torch_distill_loss(s, teacher, ids, labels, ctx.dsalt),), (logits,), (d_loss,))
            return d, None, None, None, None
        return _hip.distill_bwd(logits, teacher, ids, labels, ctx.dsalt, stats, _hip.contiguous_rows(d_loss)), None, None, None, None


@_dynamo_opaque
def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                 labels: torch.Tensor | None = None, *, temperature: float = 1.0, label_weight: float = 0.0,
                 ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The distillation loss of a student's logits [..., V] on a teacher's top logits [..., K] at the tokens
    teacher_ids [..., K], fp32::

        p    = softmax(teacher_logits / temperature)          over the K slots
        loss = (1 - label_weight) * temperature**2 * sum(p * (log p - log softmax(logits / temperature)[teacher_ids]))
             + label_weight * cross_entropy(logits, labels)

    ``reduction``: "mean" (over the rows that count), "sum" or "none" ([...]). ``labels`` [...]: rows whose
    label is ``ignore_index`` (or no token) count for nothing, in both terms; without labels every row
    counts, and label_weight must be 0. A slot whose id is no token (such as -1) or whose logit is -inf is
    left out, so that rows may have fewer than K; a row without any has no first term. An id that
    repeats takes the sum of its slots.

    logits and teacher_logits bf16, fp16 or fp32; teacher_ids and labels int32 or int64; V up to 2^30, K up
    to 1024; rows of any stride; temperature in [2^-63, 2^63). Masks of any finite value are what the formula makes of
    them. Sums are fp32, the gradient is rounded once, and its sums have a fixed order. Differentiable in logits
    alone: no gradient goes to the teacher. Functorch's transforms, forward-mode differentiation, tracing and tensor
    subclasses take torch's ops instead. Other operands raise ``DsaltError``."""
    opts = _options(labels, temperature, label_weight, ignore_index, reduction)
    lead = logits.shape[:-1]
    if not (logits.device.type == "cuda" and _fit(logits, teacher_logits, teacher_ids, labels, _hip._SCORE_DTYPES)):
        _hip.require_gpu(logits, teacher_logits, teacher_ids, labels)
        _refuse(logits, teacher_logits, teacher_ids, labels)
    if not eager(*(t for t in (logits, teacher_logits, teacher_ids, labels) if t is not None)):
        return torch_distill_loss(logits, teacher_logits.detach(), teacher_ids, labels, opts)
    rows = _hip.unit_rows
    s = rows(logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1]))
    t, i = (rows(v if v.dim() == 2 else v.reshape(-1, v.shape[-1])) for v in (teacher_logits.detach(), teacher_ids))
    y = None if labels is None else _hip.contiguous_rows(labels.reshape(-1))
    loss = _Distill.apply(s, t, i, y, opts) if torch.is_grad_enabled() else _hip.distill(s, t, i, y, opts, False)[0]
    return loss.view(lead) if reduction == "none" and logits.dim() != 2 else loss
