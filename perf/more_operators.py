"""Operators around a block's projections and at the LM's end on one GPU: what they compute, over
the sizes that training, distillation and inference of this package's models meet.

Kinds of case (the ``kind`` of a case; ``*_train`` also returns every gradient):

* ``norm``, ``norm_train``: ``dsalt.kernels.layer_norm``, and with ``add`` ``add_layer_norm``: the
  residual sum and its layer norm.
* ``distill``, ``distill_train``: ``dsalt.kernels.distill_loss``: the loss of a student's logits against
  a teacher's top logits, and the labels' cross-entropy.
* ``matmul``: ``dsalt.kernels.fp8_matmul``: the product of two 8-bit matrices with a scale for each block
  of 128; ``linear``: ``dsalt.kernels.fp8_linear``, which quantises its 16-bit rows first.

With ``own`` False, ``run`` computes them in elementary torch operations in fp32, rounded
once at the end; with ``own`` True it calls the package.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsalt-library_amd"))

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
BLOCK = 128
FP8_MAX = 448.0  # of e4m3


def listed():
    return [
        # one token of an inference loop: latency
        {"name": "norm_token", "kind": "norm", "rows": 1, "d": 1024, "stream": "bf16", "dtype": "bf16", "out": "bf16", "add": True,
         "bias": True},
        # a short fp32 sequence of an odd width, trained
        {"name": "norm_train_odd", "kind": "norm_train", "rows": 300, "d": 511, "stream": "fp32", "dtype": "fp32", "out": "fp32",
         "add": False, "bias": True},
        # a mixed-precision training step over a ragged batch (2048 + 1777 + 600 + 2048 tokens): fp32 stream, bf16 branch
        {"name": "norm_train_ragged", "kind": "norm_train", "rows": 6473, "d": 1024, "stream": "fp32", "dtype": "bf16", "out": "bf16",
         "add": True, "bias": True},
        # wide rows in a 16-bit stream
        {"name": "norm_train_wide", "kind": "norm_train", "rows": 16384, "d": 4096, "stream": "bf16", "dtype": "bf16", "out": "bf16",
         "add": True, "bias": True},
        # the loss of one token over the LM's vocabulary: latency
        {"name": "distill_token", "kind": "distill", "rows": 1, "vocab": 32000, "k": 64, "dtype": "bf16", "tau": 1.0, "lam": 0.0,
         "labels": False},
        # a training step of a small model on a short ragged batch
        {"name": "distill_train_small", "kind": "distill_train", "rows": 575, "vocab": 500, "k": 16, "dtype": "fp32", "tau": 2.0,
         "lam": 0.5, "labels": True},
        # a training step over the ragged batch and the LM's vocabulary
        {"name": "distill_train_ragged", "kind": "distill_train", "rows": 6473, "vocab": 32000, "k": 64, "dtype": "bf16", "tau": 2.0,
         "lam": 0.5, "labels": True},
        # logits of one token: the weights' bytes count
        {"name": "linear_token", "kind": "linear", "rows": 1, "d": 1024, "n": 32000, "dtype": "bf16", "scales": "pow2"},
        # gate and up of a feed-forward over a packed batch of 4 x 2048 tokens
        {"name": "linear_packed", "kind": "linear", "rows": 8192, "d": 1024, "n": 5632, "dtype": "bf16", "scales": "pow2"},
        # a handful of tokens against weights whose scales are any fp32 values
        {"name": "matmul_rows23", "kind": "matmul", "rows": 23, "d": 2816, "n": 1024, "dtype": "bf16", "scales": "fp32"},
        # a ragged batch against odd widths, k ending inside a block
        {"name": "matmul_odd", "kind": "matmul", "rows": 6473, "d": 1360, "n": 1001, "dtype": "fp16", "scales": "fp32"},
        # the largest: gate and up of a wide block on 8 x 2048 tokens
        {"name": "matmul_wide", "kind": "matmul", "rows": 16384, "d": 2048, "n": 11008, "dtype": "bf16", "scales": "pow2"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm_train", "distill", "distill_train", "distill_train", "linear", "linear", "matmul",
                       "matmul"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind.startswith("norm"):
        stream = rng.choice([dtype, dtype, "fp32"])
        d = rng.choice([8 * _log_int(rng, 8, 1024), 8 * _log_int(rng, 8, 1024), _log_int(rng, 64, 8192)])
        rows = min(_log_int(rng, 1, 16384), 16384 * 4096 // d)
        return {"kind": kind, "rows": rows, "d": d, "stream": stream, "dtype": rng.choice([dtype, stream]),
                "out": rng.choice([dtype, stream]), "add": rng.random() < 0.6, "bias": rng.random() < 0.8}
    if kind.startswith("distill"):
        vocab = _log_int(rng, 500, 131072)
        rows = min(_log_int(rng, 1, 16384), 6473 * 32000 // vocab)
        labels = rng.random() < 0.7
        return {"kind": kind, "rows": rows, "vocab": vocab, "k": _log_int(rng, 4, 256), "dtype": rng.choice([dtype, "fp32"]),
                "tau": rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 3)]),
                "lam": rng.choice([0.0, 0.5, round(rng.uniform(0.0, 1.0), 3)]) if labels else 0.0, "labels": labels}
    d = rng.choice([128 * _log_int(rng, 1, 43), 16 * _log_int(rng, 4, 344)])
    n = rng.choice([8 * _log_int(rng, 8, 1376), _log_int(rng, 64, 11008)])
    rows = min(_log_int(rng, 1, 16384), 16384 * 2048 * 11008 // (d * n))
    return {"kind": kind, "rows": rows, "d": d, "n": n, "dtype": dtype, "scales": rng.choice(["pow2", "pow2", "fp32"])}


def _blocks(k):
    return -(-k // BLOCK)


def _quantise(x, tile, pow2):
    """(q e4m3 [n, k], scale [n or blocks of n, blocks of k]): the data that a program holds in 8 bits."""
    n, k = x.shape
    rows = BLOCK if tile else 1
    full = torch.zeros(-(-n // rows) * rows, _blocks(k) * BLOCK, device=x.device)
    full[:n, :k] = x
    amax = full.view(-1, rows, _blocks(k), BLOCK).abs().amax((1, 3))
    if pow2:
        m, e = torch.frexp(amax)
        scale = torch.ldexp(torch.ones_like(amax), torch.where(m <= FP8_MAX / 512, e - 9, e - 8))
    else:
        scale = amax / FP8_MAX
    scale = torch.where(amax > 0, scale, 1.0)
    full.view(-1, rows, _blocks(k), BLOCK).div_(scale[:, None, :, None]).clamp_(-FP8_MAX, FP8_MAX)
    return full[:n, :k].to(torch.float8_e4m3fn).contiguous(), scale.to(torch.float8_e8m0fnu) if pow2 else scale


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)

    s = {"case": case}
    kind, T = case["kind"], case["rows"]
    train = kind.endswith("_train")
    if kind.startswith("norm"):
        # a residual stream that has grown over some blocks, a branch output of unit scale, trained weights around 1
        d, st, out = case["d"], DTYPES[case["stream"]], DTYPES[case["out"]]
        s["x"] = normal(T, d, std=2.0, mean=0.3, dtype=st)
        s["h"] = normal(T, d) if case["add"] else None
        s["w"] = normal(d, std=0.25, mean=1.0, dtype=st)
        s["b"] = normal(d, std=0.1, dtype=st) if case["bias"] else None
        s["leaves"] = tuple(n for n in ("x", "h", "w", "b") if s[n] is not None)
        if train:
            s["dx_out"] = normal(T, d, std=0.1, dtype=st) if case["add"] else None
            s["dy"] = normal(T, d, std=0.1, dtype=out)
    elif kind.startswith("distill"):
        # a student that has learnt part of what the teacher knows: the teacher's top tokens (distinct, best
        # first) lie above the rest of the student's logits; some teachers' rows end before k slots,
        # and a tenth of the tokens are padding where there are labels
        V, K = case["vocab"], case["k"]
        step = torch.randint(1, max(2, V // K), (T, 1), generator=g, device=DEV)
        start = torch.randint(0, V, (T, 1), generator=g, device=DEV)
        slot = torch.arange(K, device=DEV)
        ids = (start + step * slot) % V
        top = 12.0 - 1.5 * torch.log1p(slot.float()) + normal(T, K, std=0.3, dtype=torch.float32)
        s["zt"] = top.sort(-1, descending=True).values
        logits = normal(T, V, std=2.0, dtype=torch.float32)
        s["logits"] = logits.scatter_add_(1, ids, 0.5 * s["zt"]).to(dt)
        kept = torch.randint(1, 4 * K + 1, (T, 1), generator=g, device=DEV)
        s["ids"] = torch.where(slot < kept, ids, -1)
        s["labels"] = None
        if case["labels"]:
            best = s["ids"][:, 0]
            other = torch.randint(0, V, (T,), generator=g, device=DEV)
            u = torch.rand(T, generator=g, device=DEV)
            s["labels"] = torch.where(u < 0.1, -100, torch.where(u < 0.5, other, best))
        s["leaves"] = ("logits",)
        if train:
            s["up"] = torch.full((), 0.25, device=DEV)  # one of four micro-batches
    else:
        # normalised rows with a few large channels, weights of the package's initialisation
        d, n = case["d"], case["n"]
        pow2 = case["scales"] == "pow2"
        x = normal(T, d, dtype=torch.float32) * torch.exp(0.5 * torch.randn(d, generator=g, device=DEV))
        s["w"], s["ws"] = _quantise(normal(n, d, std=0.02, dtype=torch.float32), True, pow2)
        if kind == "linear":
            s["x"] = x.to(dt)
        else:
            s["a"], s["as"] = _quantise(x, False, pow2)
    if train:
        for n in s["leaves"]:
            s[n].requires_grad_()
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- the package's calls ----------------------------------------------------------------
def _call_own(s):
    from dsalt import kernels

    c = s["case"]
    if c["kind"].startswith("norm"):
        out = DTYPES[c["out"]]
        if c["add"]:
            return kernels.add_layer_norm(s["x"], s["h"], s["w"], s["b"], eps=EPS, out_dtype=out)
        return (kernels.layer_norm(s["x"], s["w"], s["b"], eps=EPS, out_dtype=out),)
    if c["kind"].startswith("distill"):
        return (kernels.distill_loss(s["logits"], s["zt"], s["ids"], s["labels"], temperature=c["tau"], label_weight=c["lam"]),)
    if c["kind"] == "linear":
        return (kernels.fp8_linear(s["x"], s["w"], s["ws"]),)
    return (kernels.fp8_matmul(s["a"], s["as"], s["w"], s["ws"], out_dtype=DTYPES[c["dtype"]]),)


def _run_own(s):
    if not s["case"]["kind"].endswith("_train"):
        with torch.no_grad():
            return list(_call_own(s))
    outs = list(_call_own(s))
    ups = [s[n] for n in ("dx_out", "dy", "up") if s.get(n) is not None]
    grads = torch.autograd.grad(outs, [s[n] for n in s["leaves"]], ups)
    return [*(t.detach() for t in outs), *grads]


# ---- the plain forms ----------------------------------------------------------------------
def _plain_norm(s):
    c = s["case"]
    f32 = {n: s[n].detach().float() for n in ("x", "h", "w", "b", "dx_out", "dy") if s.get(n) is not None}
    z = f32["x"] + f32["h"] if "h" in f32 else f32["x"]
    zc = z - z.mean(-1, keepdim=True)
    r = torch.rsqrt(zc.square().mean(-1, keepdim=True) + EPS)
    n = zc * r
    y = n * f32["w"]
    if "b" in f32:
        y = y + f32["b"]
    outs = [z.to(s["x"].dtype)] if "h" in f32 else []
    outs.append(y.to(DTYPES[c["out"]]))
    if "dy" not in f32:
        return outs
    a = f32["dy"] * f32["w"]
    dz = r * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
    if "dx_out" in f32:
        dz = dz + f32["dx_out"]
    grads = {"x": dz, "h": dz, "w": (f32["dy"] * n).sum(0), "b": f32["dy"].sum(0)}
    return outs + [grads[m].to(s[m].dtype) for m in s["leaves"]]


def _plain_distill(s):
    c = s["case"]
    tau, lam = c["tau"], c["lam"]
    logits, V = s["logits"].detach().float(), c["vocab"]
    valid = (s["ids"] >= 0) & (s["ids"] < V)
    ids = torch.where(valid, s["ids"], 0)
    t = torch.where(valid, s["zt"].float() / tau, float("-inf"))
    tm = t.amax(-1, keepdim=True)
    te = torch.where(valid, torch.exp(t - tm), 0.0)
    log_p = torch.where(valid, t - tm - torch.log(te.sum(-1, keepdim=True)), 0.0)
    p = te / te.sum(-1, keepdim=True)
    q = logits / tau
    m = q.amax(-1, keepdim=True)
    q = q - m
    lse = torch.log(torch.exp(q).sum(-1, keepdim=True))
    rows = tau * tau * (1 - lam) * (p * (log_p - (q.gather(1, ids) - lse))).sum(-1)
    counted = torch.ones_like(rows, dtype=torch.bool)
    if s["labels"] is not None:
        counted = s["labels"] != -100
    if lam:
        label = torch.where(counted, s["labels"], 0)[:, None]
        m1 = logits.amax(-1, keepdim=True)
        lse1 = torch.log(torch.exp(logits - m1).sum(-1, keepdim=True))
        rows = rows + lam * (lse1 - (logits.gather(1, label) - m1))[:, 0]
    n = counted.sum().clamp(min=1).float()
    loss = torch.where(counted, rows, 0.0).sum() / n
    if "up" not in s:
        return [loss]
    w = (s["up"] / n * counted)[:, None]
    grad = torch.exp(q - lse).scatter_add_(1, ids, -p).mul_(tau * (1 - lam))
    if lam:
        grad += lam * torch.exp(logits - m1 - lse1)
        grad.scatter_add_(1, label, torch.full_like(lse1, -lam))
    return [loss, grad.mul_(w).to(s["logits"].dtype)]


def _spread(scale, rows, n, k):
    """The scale of every element of [n, k]; each row of `scale` serves `rows` of them."""
    return scale.float().repeat_interleave(rows, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_product(s):
    c = s["case"]
    T, d, n = c["rows"], c["d"], c["n"]
    if c["kind"] == "linear":
        # each block of 128 of a row over the power of two that brings its largest value to at most 448
        x = torch.nn.functional.pad(s["x"].float(), (0, _blocks(d) * BLOCK - d)).view(T, -1, BLOCK)
        amax = x.abs().amax(-1, keepdim=True)
        m, e = torch.frexp(amax)
        scale = torch.ldexp(torch.ones_like(amax), torch.where(m <= FP8_MAX / 512, e - 9, e - 8))
        scale = torch.where(amax > 0, scale, 1.0)
        a = ((x / scale).to(torch.float8_e4m3fn).float() * scale).view(T, -1)[:, :d]
    else:
        a = s["a"].float() * _spread(s["as"], 1, T, d)
    w = s["w"].float() * _spread(s["ws"], BLOCK, n, d)
    return [(a @ w.t()).to(DTYPES[c["dtype"]])]


def _run_plain(s):
    kind = s["case"]["kind"]
    with torch.no_grad():
        return _plain_norm(s) if kind.startswith("norm") else _plain_distill(s) if kind.startswith("distill") else _plain_product(s)


# ---- work ---------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    train, T = case["kind"].endswith("_train"), case["rows"]
    e = size[case["dtype"]]
    if case["kind"].startswith("norm"):
        n, s, o = T * case["d"], size[case["stream"]], size[case["out"]]
        # x, y and with the sum h and x_out; in training also their gradients
        return {"bytes": (2 if train else 1) * n * (s + o + (s + e if case["add"] else 0)), "flops": (20 if train else 8) * n}
    if case["kind"].startswith("distill"):
        n = T * case["vocab"]
        return {"bytes": (2 if train else 1) * e * n + T * case["k"] * 12, "flops": (10 if train else 4) * n}
    d, n = case["d"], case["n"]
    scales = (1 if case["scales"] == "pow2" else 4) * _blocks(d)
    rows = T * d * e if case["kind"] == "linear" else T * (d + scales)
    return {"bytes": rows + n * d + _blocks(n) * scales + T * n * e, "flops": 2 * T * n * d}


# ---- float64, from the definitions ----------------------------------------------------------
def _to_e4m3(v):
    """v rounded to the nearest e4m3 value (4 significant bits down to 2^-6, steps of 2^-9 below; ties to even)."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind, T = case["kind"], case["rows"]
    if kind in ("linear", "matmul"):
        total = torch.zeros(T, case["n"], dtype=torch.float64, device=DEV)
        ws = s["ws"].double().repeat_interleave(BLOCK, 0)[:case["n"]]
        for b in range(_blocks(case["d"])):
            part = slice(b * BLOCK, (b + 1) * BLOCK)
            if kind == "linear":
                x = s["x"][:, part].double()
                top = x.abs().amax(1, keepdim=True)
                sa = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, FP8_MAX) / FP8_MAX)))
                xb = _to_e4m3(x / sa)
            else:
                xb, sa = s["a"][:, part].double(), s["as"][:, b:b + 1].double()
            total += (xb * sa) @ (s["w"][:, part].double() * ws[:, b:b + 1]).t()
        return [total]
    w = {n: s[n].detach().double().requires_grad_() for n in s["leaves"]}
    if kind.startswith("norm"):
        z = w["x"] + w["h"] if case["add"] else w["x"]
        var, mean = torch.var_mean(z, 1, unbiased=False, keepdim=True)
        y = (z - mean) / torch.sqrt(var + EPS) * w["w"]
        outs = ([z] if case["add"] else []) + [y + w["b"] if case["bias"] else y]
        ups = [s[n].double() for n in ("dx_out", "dy") if s.get(n) is not None]
    else:
        F = torch.nn.functional
        keep = torch.arange(T, device=DEV) if s["labels"] is None else torch.nonzero(s["labels"] != -100)[:, 0]
        logits, ids, zt = w["logits"][keep], s["ids"][keep], s["zt"][keep].double()
        log_p = torch.log_softmax(zt.masked_fill(ids < 0, -1e300) / case["tau"], 1)
        log_q = torch.log_softmax(logits / case["tau"], 1).gather(1, ids.clamp(min=0))
        kl = torch.where(ids < 0, 0.0, log_p.exp() * (log_p - log_q)).sum()
        loss = (1 - case["lam"]) * case["tau"] ** 2 * kl
        if case["lam"]:
            loss = loss + case["lam"] * F.cross_entropy(logits, s["labels"][keep], reduction="sum")
        outs, ups = [loss / max(1, len(keep))], [s["up"].double()] if "up" in s else []
    if not kind.endswith("_train"):
        return [t.detach() for t in outs]
    grads = torch.autograd.grad(outs, [w[n] for n in s["leaves"]], ups)
    return [*(t.detach() for t in outs), *grads]
