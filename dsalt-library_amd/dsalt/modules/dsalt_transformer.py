"""Pre-norm transformer block around DSALTAttention (dsalt/modules/dsalt_transformer.py).

The LM consumer of the attention path: x + attn(norm(x)), then x + ffn(norm(x)), with a
SwiGLU feed-forward. Parameter names and creation order follow the reference
(attn_norm, ffn_norm, attn, ffn; gate_proj, up_proj, down_proj) so state dicts load and
seeded initialisations agree. The attention runs on the HIP kernels; the projections are
torch (hipBLASLt GEMMs). On the GPU the FFN's gated product and each residual add with the
norm after it are HIP passes too, with autograd forward and backward (rows or modules that
those do not take run torch's ops).

Options beyond the reference, off by default: a feed-forward whose projections, activation and
product are one kernel (``gated_ffn``) and other activations; dropout whose mask is never
stored (``CounterDropout``); a norm after each branch, a learned layer scale and a residual
scale, joined to the residual stream in one pass (``branch_norm``); layer norms instead of RMS norms
(``LayerNorm``); a feed-forward whose projections are frozen 8-bit ones (``quantize_fp8``).
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
import torch.utils.checkpoint

from .. import _hip
from ..kernels import _block_train
from ..kernels.LayerNorm import LayerNorm
from ..kernels.RMSENorm import RMSENorm
from ..kernels.branch_norm import branch_norm
from ..kernels.dropout import counter_dropout, draw_seed
from ..kernels.fp8 import FP8Linear, fp8_matmul, fp8_quantize
from ..kernels.gated_ffn import _TORCH_ACT, gated_ffn, gated_ffn_supported
from .dsalt_attention import DSALTAttention


_NORMS = {"rms": RMSENorm, "layer": LayerNorm}


def norm_class(norm: str):
    """The module of a ``norm`` option."""
    if norm not in _NORMS:
        raise ValueError(f"norm must be one of {list(_NORMS)}, got {norm!r}")
    return _NORMS[norm]


class CounterDropout(nn.Module):
    """``nn.Dropout`` with ``counter_dropout``: no mask is stored. In training the call takes a seed
    (an int or an int64 GPU element) or draws one from torch's generator of x's GPU; ``offset``
    tells apart the places that share a seed. GPU tensors only."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        _hip.keep_threshold(p)  # refuses a probability outside [0, 1]
        self.p = p

    def forward(self, x: torch.Tensor, seed=None, offset: int = 0) -> torch.Tensor:
        if not self.training or self.p == 0:
            return x
        return counter_dropout(x, self.p, draw_seed(x.device) if seed is None else seed, offset)

    def extra_repr(self) -> str:
        return f"p={self.p}"


class SwiGLUFFN(nn.Module):
    """``down_proj(silu(gate_proj(x)) * up_proj(x))`` (dsalt_transformer.py:10-21). On the GPU
    the gated product is one HIP pass with torch's roundings (``dsalt_swiglu``), instead of
    torch's silu and product passes; with autograd, and projections that are plain nn.Linear
    modules, the whole is one function with a HIP pass for the product's gradients.

    ``activation``: "silu", "gelu" (erf), "gelu_tanh" or "relu". ``fused``: plain projections of
    16-bit operands (or fp32 ones under a 16-bit autocast) run as ``gated_ffn``, with and without
    autograd; others as above. ``counter_dropout``: the dropout is a ``CounterDropout``."""

    activation, fused = "silu", False  # of a module pickled without them

    def __init__(self, d_model: int, d_ff: int, dropout: float = 0.0, activation: str = "silu", fused: bool = False,
                 counter_dropout: bool = False):
        super().__init__()
        if activation not in _TORCH_ACT:
            raise ValueError(f"activation must be one of {list(_TORCH_ACT)}, got {activation!r}")
        self.gate_proj = nn.Linear(d_model, d_ff, bias=False)
        self.up_proj = nn.Linear(d_model, d_ff, bias=False)
        self.down_proj = nn.Linear(d_ff, d_model, bias=False)
        self.drop = CounterDropout(dropout) if counter_dropout else nn.Dropout(dropout)
        self.activation = activation
        self.fused = fused

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.drop(self.project(x))

    def quantize_fp8(self) -> "SwiGLUFFN":
        """The projections as frozen 8-bit ones (``FP8Linear``), in place, for inference: widths that are
        multiples of 16, weights on the GPU (else it raises and changes nothing). gate and up then share one
        quantisation of x."""
        for name, layer in self._fp8_layers():
            setattr(self, name, layer)
        return self

    def _fp8_layers(self) -> list:
        """The names of the plain projections, each with its 8-bit layer."""
        names = ("gate_proj", "up_proj", "down_proj")
        return [(n, FP8Linear.from_linear(getattr(self, n))) for n in names if type(getattr(self, n)) is nn.Linear]

    def project(self, x: torch.Tensor) -> torch.Tensor:
        """The feed-forward without its dropout."""
        if self.fused and self._one_kernel(x):
            return gated_ffn(x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, self.activation)
        if self._shared_rows(x):
            rows, dt = fp8_quantize(x), _block_train.autocast_dtype(x)
            g, u = (fp8_matmul(*rows, m.weight_q, m.weight_scale, m.bias, dt) for m in (self.gate_proj, self.up_proj))
        elif self.activation == "silu" and torch.is_grad_enabled() and _block_train.swiglu_supported(self, x):
            return _block_train.swiglu_ffn(self, x)
        else:
            g, u = self.gate_proj(x), self.up_proj(x)
        if self.activation != "silu":
            return self.down_proj(_TORCH_ACT[self.activation](g) * u)
        if not torch.is_grad_enabled() and _hip.swiglu_supported(g, u):
            h = _hip.swiglu(g, u)  # one pass, the same bits as the two torch ops below
        else:
            h = F.silu(g) * u
        return self.down_proj(h)

    def _shared_rows(self, x: torch.Tensor) -> bool:
        """Whether gate and up are 8-bit layers that quantise the same rows before their products."""
        lin = (self.gate_proj, self.up_proj)
        return (all(type(m) is FP8Linear for m in lin) and _block_train.plain(*lin)
                and not (torch.is_grad_enabled() and x.requires_grad)
                and x.shape[-1] > 0 and x.numel() // x.shape[-1] > _hip.FP8_FEW_ROWS)

    def _one_kernel(self, x: torch.Tensor) -> bool:
        lin = (self.gate_proj, self.up_proj, self.down_proj)
        return (all(type(m) is nn.Linear and m.bias is None for m in lin) and _block_train.plain(*lin)
                and _block_train.eager(x, *(m.weight for m in lin)) and gated_ffn_supported(x, *(m.weight for m in lin)))


class DSALTTransformerBlock(nn.Module):
    """RMSNorm -> DSALTAttention -> residual, RMSNorm -> SwiGLU -> residual
    (dsalt_transformer.py:24-88); ``gradient_checkpointing`` recomputes the attention and
    the FFN in the backward when training. ``_fuse_norms`` (default True): at inference
    without autograd, with 16-bit rows, a residual add and the norm after it run as one
    HIP pass (``dsalt_add_rms_norm``: the sum is torch's add bit for bit, the norm can
    differ from F.rms_norm in an output's last bit); with autograd, in fp32 or 16-bit, as one
    pass forward and one backward (``dsalt_norm_train``), which under autocast also writes
    the norm in the projections' type.

    ``post_norm`` (an RMSENorm of each branch's output: attn_post_norm, ffn_post_norm),
    ``layer_scale`` (a learned gate of each branch per channel, attn_gate and ffn_gate, that starts
    at this value), ``residual_scale`` and ``counter_dropout`` make a branch
    ``residual_scale * x + gate * post_norm(branch)`` on ``branch_norm``, which takes the
    feed-forward's dropout and the next norm along. ``fused_ffn``, ``activation``: see SwiGLUFFN.

    ``norm``: "rms", or "layer" for LayerNorm modules in the place of every RMSENorm. The attention's residual add and
    the layer norm after it are one pass forward and one backward (``add_layer_norm``); without autograd in the LM
    the feed-forward's add and the next block's norm too. With the options of ``branch_norm`` above, layer norms are
    passes of their own. Norms that are replaced or hooked are called as they are."""

    _fuse_norms = True
    joins_branches = False

    def __init__(self, d_model: int, n_heads: int, n_min: int, n_max: int, k_lmk: int, max_seq_len: int,
                 d_ff: int, dropout: float = 0.0, yarn_scale: float = 1.0, layer_idx: int = 0,
                 n_kv_heads: int | None = None, qkv_bias: bool = False, rope_base: float = 10000.0,
                 post_norm: bool = False, layer_scale: float | None = None, residual_scale: float = 1.0,
                 fused_ffn: bool = False, activation: str = "silu", counter_dropout: bool = False, norm: str = "rms"):
        super().__init__()
        Norm = norm_class(norm)
        self.layer_idx = layer_idx
        self.attn_norm = Norm(d_model)
        self.ffn_norm = Norm(d_model)
        self.attn = DSALTAttention(d_model=d_model, n_heads=n_heads, n_min=n_min, n_max=n_max, k_lmk=k_lmk,
                                   max_seq_len=max_seq_len, dropout=dropout, yarn_scale=yarn_scale,
                                   layer_idx=layer_idx, n_kv_heads=n_kv_heads, qkv_bias=qkv_bias,
                                   rope_base=rope_base)
        self.ffn = SwiGLUFFN(d_model=d_model, d_ff=d_ff, dropout=dropout, activation=activation, fused=fused_ffn,
                             counter_dropout=counter_dropout)
        self.residual_scale = residual_scale
        self.attn_post_norm = Norm(d_model) if post_norm else None
        self.ffn_post_norm = Norm(d_model) if post_norm else None
        self.attn_gate = nn.Parameter(torch.full((d_model,), float(layer_scale))) if layer_scale is not None else None
        self.ffn_gate = nn.Parameter(torch.full((d_model,), float(layer_scale))) if layer_scale is not None else None
        self.joins_branches = post_norm or layer_scale is not None or residual_scale != 1.0 or counter_dropout

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None, max_seqlen: int | None = None,
                gradient_checkpointing: bool = False, rope_cs: tuple | None = None,
                cu_list: list | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        if self.joins_branches:
            x, _, aux = self.join_branches(x, self.attn_norm(x), None, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen,
                                           gradient_checkpointing=gradient_checkpointing, rope_cs=rope_cs, cu_list=cu_list)
            return x, aux
        aux_box = []
        train_norms = torch.is_grad_enabled() and self._fuse_norms

        def attend(h, h_cast=None):
            more = {} if h_cast is None else {"_x_cast": h_cast}
            o, a = self.attn(h, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, rope_cs=rope_cs, cu_list=cu_list, **more)
            aux_box.append(a)
            return o

        recompute = gradient_checkpointing and self.training
        # under autocast the projections' operand is written by the norm itself
        cast = _block_train.autocast_dtype(x) if x.is_cuda else x.dtype
        cast = cast if cast != x.dtype and x.dtype == torch.float32 else None
        h_cast = None
        if train_norms and self._train_norm(x, None, self.attn_norm):
            if cast is not None and type(self.attn) is DSALTAttention and _block_train.plain(self.attn):
                x, h, h_cast = _block_train.add_norm(x, None, self.attn_norm, cast)
            else:
                x, h = _block_train.add_norm(x, None, self.attn_norm)
        else:
            h = self.attn_norm(x)
        x_attn = (torch.utils.checkpoint.checkpoint(attend, h, h_cast, use_reentrant=False) if recompute
                  else attend(h, h_cast))
        if self._norms_fusable(x, x_attn, self.ffn_norm):
            # the residual add and the FFN's norm in one HIP pass (inference)
            x, h = self._add_norm(x, x_attn, self.ffn_norm)
        elif train_norms and self._layer_joins(x, x_attn, self.ffn_norm):
            x, h = self.ffn_norm(x, x_attn, cast if self._plain_ffn() else None)
        elif train_norms and self._train_norm(x, x_attn, self.ffn_norm):
            low = (cast is not None and type(self.ffn) is SwiGLUFFN and _block_train.plain(self.ffn)
                   and _block_train.swiglu_supported(self.ffn, x))
            x, h = _block_train.add_norm(x, x_attn, self.ffn_norm, cast if low else None, low)
        else:
            x = x + x_attn
            h = self.ffn_norm(x)
        f = torch.utils.checkpoint.checkpoint(self.ffn, h, use_reentrant=False) if recompute else self.ffn(h)
        x = _block_train.residual_add(x, f) if train_norms else x + f
        return x, aux_box[0]

    def join_branches(self, x: torch.Tensor, h: torch.Tensor, next_norm: nn.Module | None, seed=None, cu_seqlens=None,
                      max_seqlen=None, gradient_checkpointing: bool = False, rope_cs=None, cu_list=None):
        """The block on the stream x and its norm h = attn_norm(x), each branch joined by
        ``branch_norm``: ``(x, next_norm(x), aux)`` (None without next_norm: the norm that reads
        the stream next). ``seed``: of the feed-forward's dropout, at offset layer_idx + 1."""
        recompute = gradient_checkpointing and self.training

        def run(fn, t):
            return torch.utils.checkpoint.checkpoint(fn, t, use_reentrant=False) if recompute else fn(t)

        o, aux = run(lambda t: self.attn(t, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, rope_cs=rope_cs, cu_list=cu_list), h)
        # the norm in the type that the feed-forward's projections compute in, where only they read it
        low = None if not self._plain_ffn() else _block_train.autocast_dtype(x) if x.dtype == torch.float32 else x.dtype
        x, h = self._join(x, o, self.attn_post_norm, self.attn_gate, self.ffn_norm, low)
        drop = self.ffn.drop if type(self.ffn) is SwiGLUFFN else None
        if type(drop) is CounterDropout and _block_train.plain(self.ffn, drop):
            f = run(self.ffn.project, h)
            p = drop.p if drop.training else 0.0
            if p > 0 and seed is None:
                seed = draw_seed(x.device)
            x, h = self._join(x, f, self.ffn_post_norm, self.ffn_gate, next_norm, None, p, seed)
        else:
            x, h = self._join(x, run(self.ffn, h), self.ffn_post_norm, self.ffn_gate, next_norm, None)
        return x, h, aux

    def _plain_ffn(self) -> bool:
        """Whether nothing but plain projections reads the feed-forward's operand."""
        if type(self.ffn) is not SwiGLUFFN:
            return False
        lin = (self.ffn.gate_proj, self.ffn.up_proj)
        return all(type(m) is nn.Linear for m in lin) and _block_train.plain(self.ffn, *lin)

    def _join(self, x, o, post, gate, norm, out_dtype, p: float = 0.0, seed=None):
        """x joined with the branch's output o, and its norm (in out_dtype; None: the sum's): norms that
        are replaced or hooked are called as they are. The sum has the type that x + o has: a
        16-bit stream beside an fp32 o (a replaced norm's, under autocast) goes on in fp32."""
        def inside(m):
            return m is None or (type(m) is RMSENorm and _block_train.plain(m))

        offset = self.layer_idx + 1
        if not inside(post):
            o, p, post = post(counter_dropout(o, p, seed, offset) if p > 0 else o), 0.0, None
        wide = torch.promote_types(x.dtype, o.dtype)
        if wide is not x.dtype:
            x = x.to(wide)

        def taken(w):
            return w if w is None or w.dtype is wide else w.float()

        n = norm if inside(norm) else None
        x, h = branch_norm(x, o, None if n is None else taken(n.weight),
                           post_weight=None if post is None else taken(post.weight), gate=taken(gate),
                           residual_scale=self.residual_scale, p=p, seed=seed, offset=offset,
                           eps=1e-6 if n is None else n.eps, post_eps=1e-6 if post is None else post.eps,
                           out_dtype=out_dtype if n is not None else None)
        return x, norm(x) if n is None and norm is not None else h

    @staticmethod
    def _train_norm(x: torch.Tensor, h: torch.Tensor | None, norm: nn.Module) -> bool:
        """Whether x (+ h) and the RMSENorm `norm` can run as one differentiable pass."""
        return (_block_train.eager(x, norm.weight) and type(norm) is RMSENorm and _block_train.plain(norm) and _hip.norm_train_supported(x, norm.weight)
                and norm.normalized_shape == (x.shape[-1],)
                and (h is None or _hip.norm_train_branch_supported(x, h)))

    @staticmethod
    def _layer_joins(x: torch.Tensor, h: torch.Tensor, norm: nn.Module) -> bool:
        """Whether x + h and the LayerNorm `norm` can run as one add_layer_norm pass."""
        return (type(norm) is LayerNorm and _block_train.plain(norm) and x.is_cuda and h.device == x.device and h.shape == x.shape
                and 1 <= x.shape[-1] <= _hip.LAYER_NORM_MAX_DIM and x.dtype in _hip._SCORE_DTYPES
                and (h.dtype is x.dtype or (x.dtype is torch.float32 and h.dtype in _hip._SCORE_DTYPES)))

    @staticmethod
    def _add_norm(x: torch.Tensor, h: torch.Tensor | None, norm: nn.Module):
        """``(x + h, norm(x + h))`` (without h: ``(None, norm(x))``) of norms that `_norms_fusable` takes."""
        if type(norm) is LayerNorm:
            return (None, norm(x)) if h is None else norm(x, h)
        return _hip.add_rms_norm(x, h, norm.weight, norm.eps)

    def _norms_fusable(self, x: torch.Tensor, h: torch.Tensor | None, norm: nn.Module) -> bool:
        """Whether x (+ h) and the RMSENorm `norm` can run as one dsalt_add_rms_norm pass:
        inference without autograd, 16-bit rows on the GPU, a weight of x's dtype; or the LayerNorm
        `norm` as one dsalt_layer_norm pass, without autograd."""
        if self.training or torch.is_grad_enabled() or not self._fuse_norms:
            return False
        if isinstance(norm, LayerNorm):
            return self._layer_joins(x, x if h is None else h, norm)
        if type(norm) is not RMSENorm or not _block_train.plain(norm):  # replaced or hooked: called as it is
            return False
        if h is not None and (h.shape != x.shape or h.dtype != x.dtype or not h.is_contiguous()
                              or h.data_ptr() % 16):
            return False
        return _hip.add_rms_norm_supported(x, norm.weight)

    def _forward_fused(self, x: torch.Tensor, delta: torch.Tensor | None, cu_seqlens=None, max_seqlen=None,
                       rope_cs=None, cu_list=None):
        """Inference forward that leaves its last residual add to the caller: returns
        (x + attention, the FFN output, aux - None on the packed path, where the attention
        makes no zero aux tensor), so that the next block's norm (or the final norm) takes
        that add in its own pass. `delta` is the previous block's pending FFN
        output (None for the first block). The caller checks `_norms_fusable` first."""
        x, h = self._sum_norm(x, delta, self.attn_norm)
        x_attn, aux = self.attn(h, cu_seqlens=cu_seqlens, max_seqlen=max_seqlen, rope_cs=rope_cs, cu_list=cu_list,
                                _need_aux=False)
        x, h = self._sum_norm(x, x_attn, self.ffn_norm)
        return x, self.ffn(h), aux

    def _sum_norm(self, x: torch.Tensor, h: torch.Tensor | None, norm: nn.Module):
        """``(x + h, norm(x + h))``, in one pass where the two go together: a replaced feed-forward's output may be
        of a wider type than the stream."""
        if self._norms_fusable(x, h, norm):
            x_sum, y = self._add_norm(x, h, norm)
            return x if x_sum is None else x_sum, y
        x = x if h is None else x + h
        return x, norm(x)
