"""DSALTLMHeadModel (dsalt/model/dsalt_lm.py:64-284): the causal-LM consumer of the
attention path.

Token embedding -> ``n_layers`` pre-norm DSALT blocks -> final RMSNorm -> LM head (tied
to the embedding by default). Constructor arguments, parameter names, module creation
order and the initialisation rule (every Linear weight N(0, 0.02), out_proj/down_proj
N(0, 0.02 / sqrt(2 n_layers)), biases 0, embedding N(0, 0.02); dsalt_lm.py:164-172)
follow the reference, so seeded models and state dicts agree.

Input: packed ``input_ids [T]`` with ``cu_seqlens`` (sparse HIP attention), or
``[1, T]`` without (the dense batched variant; the reference's batched attention fails
for B > 1 and so does this one, with a clear error). The packed RoPE positions are
derived in the HIP RoPE kernel from cu_seqlens, so no per-token cos/sin gather is built;
the host copy of cu_seqlens is taken once per forward and shared by every layer.
``labels`` gives the mean token cross-entropy (ignore index -100), computed over
``lm_head_chunk_size``-token chunks so that at most [chunk, vocab] logits exist at once.
The Triton-only "liger" loss is not available (as in the reference without Triton).

Inference without autograd in bf16/fp16 runs every residual add in the pass of the
RMSNorm after it (dsalt_add_rms_norm: each block hands its FFN output to the next
block's norm, the last one to the final norm); the FFN's gated product and the window
gate run as HIP passes too (SwiGLUFFN, DSALTAttention).

The options of DSALTTransformerBlock beyond the reference (post_norm, layer_scale,
residual_scale, fused_ffn, activation, counter_dropout, norm) apply to every layer; with
counter_dropout the embedding's dropout is a CounterDropout too, and one seed drawn a forward
serves all places, told apart by their offsets; norm="layer" makes the final norm a LayerNorm too.

Distillation: with ``teacher_logits`` and ``teacher_ids`` [..., K] the loss is ``distill_loss`` against a
teacher's top logits, over the same chunks. ``quantize_fp8`` makes the feed-forwards and the head frozen
8-bit layers, for a model that answers or teaches.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _hip
from ..kernels import _block_train
from ..kernels.LayerNorm import LayerNorm
from ..kernels.RMSENorm import RMSENorm
from ..kernels.distill import cpu_distill_loss, distill_loss
from ..kernels.dropout import draw_seed
from ..kernels.fp8 import FP8Linear
from ..modules.dsalt_transformer import CounterDropout, DSALTTransformerBlock, SwiGLUFFN, norm_class

_LOSS_FNS = ("auto", "liger", "chunked")


def _chunked_cross_entropy(x: torch.Tensor, head, labels: torch.Tensor, chunk_size: int = 512) -> torch.Tensor:
    """Sum of token cross-entropies over chunks of rows of ``head(x)``, divided by
    the number of labels other than -100 (at least 1)."""
    total = torch.zeros((), device=x.device, dtype=torch.float32)
    for a in range(0, x.shape[0], chunk_size):
        logits = head(x[a:a + chunk_size])
        total = total + F.cross_entropy(logits, labels[a:a + chunk_size], ignore_index=-100, reduction="sum")
    n = (labels != -100).sum().clamp(min=1).to(torch.float32)
    return total / n


def _chunked_distillation(x: torch.Tensor, head, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                          labels: torch.Tensor | None, temperature: float, label_weight: float,
                          chunk_size: int = 512) -> torch.Tensor:
    """``distill_loss`` of ``head(x)`` over chunks of rows: its mean over the rows that count (all of them,
    without labels)."""
    total = torch.zeros((), device=x.device, dtype=torch.float32)
    for a in range(0, x.shape[0], chunk_size):
        part = slice(a, a + chunk_size)
        y = None if labels is None else labels[part]
        loss = distill_loss if x.is_cuda else cpu_distill_loss
        logits = head(x[part])
        total = total + loss(logits, teacher_logits[part], teacher_ids[part], y, temperature=temperature,
                             label_weight=label_weight, reduction="sum")
        vocab = logits.shape[-1]
        del logits  # not held while the next chunk's are formed
    if labels is None or not x.shape[0]:
        return total / max(x.shape[0], 1)
    counted = (labels != -100) & (labels >= 0) & (labels < vocab)
    return total / counted.sum().clamp(min=1).to(torch.float32)


class DSALTLMHeadModel(nn.Module):
    def __init__(self, vocab_size: int, d_model: int, n_layers: int, n_heads: int, n_min: int, n_max: int,
                 k_lmk: int, max_seq_len: int, d_ff: int | None = None, dropout: float = 0.0,
                 yarn_scale: float = 1.0, tie_weights: bool = True, padding_idx: int | None = None,
                 lm_head_chunk_size: int = 2048, loss_fn: str = "chunked", aux_loss_weight: float = 0.0,
                 n_kv_heads: int | None = None, qkv_bias: bool = False, rope_base: float = 10000.0,
                 post_norm: bool = False, layer_scale: float | None = None, residual_scale: float = 1.0,
                 fused_ffn: bool = False, activation: str = "silu", counter_dropout: bool = False, norm: str = "rms"):
        super().__init__()
        if loss_fn not in _LOSS_FNS:
            raise ValueError(f"loss_fn must be one of {list(_LOSS_FNS)}, got {loss_fn!r}")
        if loss_fn == "liger":
            raise RuntimeError("loss_fn='liger' needs the Triton fused cross-entropy, which this build does "
                               "not have; use loss_fn='chunked'")
        self.d_model = d_model
        self.n_layers = n_layers
        self.vocab_size = vocab_size
        self.lm_head_chunk_size = lm_head_chunk_size
        self.loss_fn = loss_fn
        self.aux_loss_weight = aux_loss_weight
        if d_ff is None:  # about 8/3 d_model, rounded up to a multiple of 128
            d_ff = -(-int(8 / 3 * d_model) // 128) * 128

        self.embed_tokens = nn.Embedding(vocab_size, d_model, padding_idx=padding_idx)
        self.embed_dropout = CounterDropout(dropout) if counter_dropout else nn.Dropout(dropout)
        self.layers = nn.ModuleList(
            DSALTTransformerBlock(d_model=d_model, n_heads=n_heads, n_min=n_min, n_max=n_max, k_lmk=k_lmk,
                                  max_seq_len=max_seq_len, d_ff=d_ff, dropout=dropout, yarn_scale=yarn_scale,
                                  layer_idx=i, n_kv_heads=n_kv_heads, qkv_bias=qkv_bias, rope_base=rope_base,
                                  post_norm=post_norm, layer_scale=layer_scale, residual_scale=residual_scale,
                                  fused_ffn=fused_ffn, activation=activation, counter_dropout=counter_dropout, norm=norm)
            for i in range(n_layers))
        self.final_norm = norm_class(norm)(d_model)
        self.lm_head = nn.Linear(d_model, vocab_size, bias=False)
        if tie_weights:
            self.lm_head.weight = self.embed_tokens.weight
        self._init_weights()

    @classmethod
    def from_config(cls, config) -> "DSALTLMHeadModel":
        """Build from a config object with ``to_dict()`` (the reference's DSALTConfig)."""
        return cls(**config.to_dict())

    def _init_weights(self) -> None:
        nn.init.normal_(self.embed_tokens.weight, std=0.02)
        deep = 0.02 / math.sqrt(2 * self.n_layers)
        for name, mod in self.named_modules():
            if not isinstance(mod, nn.Linear):
                continue
            nn.init.normal_(mod.weight, std=deep if ("out_proj" in name or "down_proj" in name) else 0.02)
            if mod.bias is not None:
                nn.init.zeros_(mod.bias)

    def quantize_fp8(self, lm_head: bool = True) -> "DSALTLMHeadModel":
        """The feed-forwards' projections and (``lm_head``) the head as frozen 8-bit layers, in place, for
        inference; the embedding, the attention and the norms stay as they are. On the GPU, widths that are
        multiples of 16 (else it raises and changes nothing)."""
        new = [(layer.ffn, *item) for layer in self.layers if type(layer.ffn) is SwiGLUFFN for item in layer.ffn._fp8_layers()]
        if lm_head and type(self.lm_head) is nn.Linear:
            new.append((self, "lm_head", FP8Linear.from_linear(self.lm_head)))
        for owner, name, layer in new:
            setattr(owner, name, layer)
        return self

    def _head(self, x: torch.Tensor) -> torch.Tensor:
        """The head's logits within a loss."""
        return self.lm_head(x) if type(self.lm_head) is FP8Linear else F.linear(x, self.lm_head.weight)

    def set_collect_last_P(self, on: bool) -> None:
        """Turn the attention modules' ``_last_P`` diagnostic on or off."""
        for layer in self.layers:
            layer.attn._collect_last_P = on

    @staticmethod
    def _to_autocast_dtype(x: torch.Tensor) -> torch.Tensor:
        dev = x.device.type
        if torch.is_autocast_enabled(dev):
            dt = torch.get_autocast_dtype(dev)
            if x.dtype != dt:
                return x.to(dt)
        return x

    def forward(self, input_ids: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                max_seqlen: int | None = None, labels: torch.Tensor | None = None,
                gradient_checkpointing: bool = False, padding_mask: torch.Tensor | None = None,
                teacher_logits: torch.Tensor | None = None, teacher_ids: torch.Tensor | None = None,
                temperature: float = 1.0, label_weight: float = 0.0) -> dict:
        """``teacher_logits`` and ``teacher_ids`` (input_ids' shape and K slots): the loss is the distillation
        loss of ``distill_loss`` with ``temperature`` and ``label_weight``; ``labels`` are then optional."""
        if (teacher_logits is None) != (teacher_ids is None):
            raise ValueError("teacher_logits and teacher_ids are given together")
        if teacher_ids is not None:  # the loss goes over chunks of all of them
            n = input_ids.numel()
            if (any(t.dim() < 1 or t.shape[:-1].numel() != n for t in (teacher_logits, teacher_ids))
                    or (labels is not None and labels.numel() != n)):
                got = [None if t is None else tuple(t.shape) for t in (teacher_logits, teacher_ids, labels)]
                raise _hip.DsaltError(f"teacher_logits, teacher_ids and labels must cover the {n} tokens (got {got})")
        with_loss = labels is not None or teacher_ids is not None
        if max_seqlen is None:
            max_seqlen = input_ids.shape[-1]
        seed = None
        if type(self.embed_dropout) is CounterDropout and self.training and self.embed_dropout.p > 0:
            seed = draw_seed(input_ids.device)
            x = self._to_autocast_dtype(self.embed_dropout(self.embed_tokens(input_ids), seed))
        else:
            x = self._to_autocast_dtype(self.embed_dropout(self.embed_tokens(input_ids)))
        cu_list = None
        if cu_seqlens is not None and not self._device_packing(cu_seqlens, x):
            cu_list = cu_seqlens.detach().cpu().tolist()
        if not with_loss and self._norms_fusable(x):
            # inference: each residual add runs in the pass of the norm that follows it
            delta = None
            for layer in self.layers:
                x, delta, _ = layer._forward_fused(x, delta, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen,
                                                   cu_list=cu_list)
            _, x = self.layers[-1]._sum_norm(x, delta, self.final_norm)
            return {"loss": None, "logits": self.lm_head(x), "aux_loss": None}
        aux = torch.zeros((), device=input_ids.device, dtype=x.dtype)
        joins = bool(self.layers) and all(type(layer) is DSALTTransformerBlock and layer.joins_branches
                                          and _block_train.plain(layer) for layer in self.layers)
        h = self.layers[0].attn_norm(x) if joins else None
        for i, layer in enumerate(self.layers):
            if joins:  # each block's last pass also forms the norm that the next block reads
                after = self.layers[i + 1].attn_norm if i + 1 < len(self.layers) else self.final_norm
                x, h, a = layer.join_branches(x, h, after, seed, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen,
                                              gradient_checkpointing=gradient_checkpointing, cu_list=cu_list)
            else:
                x, a = layer(x, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen,
                             gradient_checkpointing=gradient_checkpointing, cu_list=cu_list)
            if with_loss:  # the layers' auxiliary losses are only returned with a loss
                aux = aux + a
        x = h if joins else self.final_norm(x)
        if not with_loss:
            return {"loss": None, "logits": self.lm_head(x), "aux_loss": None}
        x, y = x.reshape(-1, self.d_model), None if labels is None else labels.reshape(-1).long()
        if teacher_ids is None:
            loss = _chunked_cross_entropy(x, self._head, y, self.lm_head_chunk_size)
        else:
            loss = _chunked_distillation(x, self._head, *(t.reshape(-1, t.shape[-1]) for t in (teacher_logits, teacher_ids)), y,
                                         temperature, label_weight, self.lm_head_chunk_size)
        return {"loss": loss + self.aux_loss_weight * aux, "logits": None, "aux_loss": aux.detach()}

    def _device_packing(self, cu_seqlens: torch.Tensor, x: torch.Tensor) -> bool:
        """Whether the layers need no host copy of cu_seqlens (a synchronisation): batches that no
        selection splits, without the ``_last_P`` diagnostic, on the HIP score route."""
        return (cu_seqlens.is_cuda and x.dim() == 2 and x.shape[0] <= _hip.SELECT_SPLIT_MIN
                and all((self.training or not getattr(layer.attn, "_collect_last_P", True))
                        and getattr(layer.attn, "_hip_scores", False) for layer in self.layers))

    def _norms_fusable(self, x: torch.Tensor) -> bool:
        """Whether every residual add and norm of the forward can run as dsalt_add_rms_norm
        passes (inference without autograd, 16-bit rows, norm weights of x's dtype), or, of LayerNorms,
        as dsalt_layer_norm passes (inference without autograd)."""
        if not self.layers:
            return False
        final = self.final_norm
        if not (DSALTTransformerBlock._layer_joins(x, x, final) if isinstance(final, LayerNorm)
                else type(final) is RMSENorm and _block_train.plain(final) and _hip.add_rms_norm_supported(x, final.weight)):
            return False
        if any(getattr(layer, "joins_branches", False) for layer in self.layers):
            return False
        return all(layer._norms_fusable(x, None, layer.attn_norm) and layer._norms_fusable(x, None, layer.ffn_norm)
                   for layer in self.layers)

    def num_parameters(self, trainable_only: bool = True) -> int:
        return sum(p.numel() for p in self.parameters() if p.requires_grad or not trainable_only)
