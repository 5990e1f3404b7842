"""The block's feed-forward, dropout and branch operators on one GPU: what they compute, over
the sizes that training and inference of this package's blocks meet.

Kinds of case (the ``kind`` of a case; ``*_train`` also returns every gradient):

* ``ffn``, ``ffn_train``: ``dsalt.kernels.gated_ffn``, ``(act(x Wg^T) * (x Wu^T)) Wd^T``.
* ``dropout``, ``dropout_train``: ``dsalt.kernels.counter_dropout``, dropout whose mask is a
  function of the seed and the element's index.
* ``branch``, ``branch_train``: ``dsalt.kernels.branch_norm``: dropout and RMSNorm of a
  branch's output, its gate, the scaled residual sum and the RMSNorm of the sum.

With ``own`` False, ``run`` computes them in elementary torch operations in fp32, rounded
once at the end; with ``own`` True it calls the package.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsalt-library_amd"))

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _hidden(d):
    """Hidden width of the package's feed-forward: about 8/3 d, a multiple of 128."""
    return -(-int(8 / 3 * d) // 128) * 128


def listed():
    return [
        # one token through a full-width feed-forward: the weights' bytes and the launches count
        {"name": "ffn_token", "kind": "ffn", "rows": 1, "d": 1024, "f": 2816, "act": "silu", "dtype": "bf16"},
        # a handful of tokens, small width, the other 16-bit type and activation
        {"name": "ffn_rows23", "kind": "ffn", "rows": 23, "d": 512, "f": 1408, "act": "gelu_tanh", "dtype": "fp16"},
        # inference over a packed batch of the headline shape, 4 x 2048 tokens
        {"name": "ffn_packed", "kind": "ffn", "rows": 8192, "d": 1024, "f": 2816, "act": "silu", "dtype": "bf16"},
        # a training step of a small block on a short ragged batch (odd sizes all round)
        {"name": "ffn_train_small", "kind": "ffn_train", "rows": 575, "d": 264, "f": 712, "act": "gelu", "dtype": "fp16"},
        # a training step over a ragged batch of the block's usual width (2048 + 1777 + 600 + 2048 tokens)
        {"name": "ffn_train_ragged", "kind": "ffn_train", "rows": 6473, "d": 1024, "f": 2816, "act": "silu", "dtype": "bf16"},
        # the largest: a wide block on 8 x 2048 tokens
        {"name": "ffn_train_wide", "kind": "ffn_train", "rows": 16384, "d": 2048, "f": 5504, "act": "silu", "dtype": "bf16"},
        # embedding dropout of a short fp32 sequence, an odd number of elements
        {"name": "dropout_odd", "kind": "dropout", "n": 300 * 511 + 7, "p": 0.1, "offset": 3, "dtype": "fp32"},
        # dropout of a full batch's hidden states, forward and backward
        {"name": "dropout_train", "kind": "dropout_train", "n": 16384 * 2048, "p": 0.1, "offset": 0, "dtype": "bf16"},
        # one token of an inference loop, post-norm and layer scale: latency
        {"name": "branch_token", "kind": "branch", "rows": 1, "d": 1024, "stream": "bf16", "dtype": "bf16", "out": "bf16",
         "post": True, "pre": True, "gate": "channel", "scale": 1.0, "p": 0.0},
        # inference over a packed batch: sandwich norms without gate, scaled residual
        {"name": "branch_packed", "kind": "branch", "rows": 8192, "d": 1024, "stream": "bf16", "dtype": "bf16", "out": "bf16",
         "post": True, "pre": True, "gate": "none", "scale": 0.8, "p": 0.0},
        # a mixed-precision training step: fp32 stream, bf16 branch, dropout and layer scale
        {"name": "branch_train_ragged", "kind": "branch_train", "rows": 6473, "d": 1024, "stream": "fp32", "dtype": "bf16",
         "out": "bf16", "post": True, "pre": True, "gate": "channel", "scale": 1.0, "p": 0.1},
        # wide rows in a 16-bit stream, gated per token
        {"name": "branch_train_wide", "kind": "branch_train", "rows": 16384, "d": 4096, "stream": "bf16", "dtype": "bf16",
         "out": "bf16", "post": True, "pre": True, "gate": "token", "scale": 0.9, "p": 0.1},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "ffn_train", "ffn_train", "dropout", "dropout_train", "branch", "branch_train",
                       "branch_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind.startswith("ffn"):
        d = 8 * _log_int(rng, 8, 256)
        f = rng.choice([_hidden(d), 8 * _log_int(rng, d // 8, d // 2)])
        rows = _log_int(rng, 1, 16384)
        return {"kind": kind, "rows": rows, "d": d, "f": f, "dtype": dtype,
                "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"])}
    p = rng.choice([0.0, 0.05, 0.1, 0.1, 0.2, 0.5, round(rng.uniform(0.01, 0.95), 3)])
    if kind.startswith("dropout"):
        return {"kind": kind, "n": _log_int(rng, 4096, 16384 * 2048), "p": p, "offset": rng.randrange(1 << 40),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    stream = rng.choice([dtype, dtype, "fp32"])
    d = 8 * _log_int(rng, 8, 1024)
    rows = min(_log_int(rng, 1, 16384), 16384 * 4096 // d)
    return {"kind": kind, "rows": rows, "d": d, "stream": stream, "dtype": rng.choice([dtype, stream]),
            "out": rng.choice([dtype, stream]), "post": rng.random() < 0.7, "pre": rng.random() < 0.8,
            "gate": rng.choice(["none", "channel", "channel", "token"]),
            "scale": rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 3)]), "p": rng.choice([0.0, p])}


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)

    s = {"case": case}
    kind = case["kind"]
    train = kind.endswith("_train")
    if kind.startswith("ffn"):
        # normalised rows, weights of the package's initialisation, gradients of one scale
        T, d, f = case["rows"], case["d"], case["f"]
        s["x"] = normal(T, d)
        s["wg"], s["wu"], s["wd"] = normal(f, d, std=0.02), normal(f, d, std=0.02), normal(d, f, std=0.02)
        leaves = ("x", "wg", "wu", "wd")
        if train:
            s["dy"] = normal(T, d, std=0.1)
    else:
        s["seed"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), generator=g, device=DEV)
    if kind.startswith("dropout"):
        s["x"] = normal(case["n"])
        leaves = ("x",)
        if train:
            s["dy"] = normal(case["n"])
    if kind.startswith("branch"):
        # a residual stream that has grown over some blocks, a branch output of unit scale,
        # trained norm weights around 1, layer scales around 0.1 or token gates in (0, 1)
        T, d, st = case["rows"], case["d"], DTYPES[case["stream"]]
        s["x"], s["h"] = normal(T, d, std=2.0, dtype=st), normal(T, d)
        s["w_post"] = normal(d, std=0.25, mean=1.0, dtype=st) if case["post"] else None
        s["w"] = normal(d, std=0.25, mean=1.0, dtype=st) if case["pre"] else None
        s["gate"] = {"none": None, "channel": normal(d, std=0.05, mean=0.1, dtype=st),
                     "token": torch.sigmoid(normal(T, 1, dtype=torch.float32)).to(st)}[case["gate"]]
        leaves = tuple(n for n in ("x", "h", "w_post", "w", "gate") if s[n] is not None)
        if train:
            s["dx_out"] = normal(T, d, std=0.1, dtype=st)
            s["dy"] = normal(T, d, std=0.1, dtype=DTYPES[case["out"]]) if case["pre"] else None
    s["leaves"] = leaves
    if train:
        for n in leaves:
            s[n].requires_grad_()
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- the package's calls ----------------------------------------------------------------
def _call_own(s):
    from dsalt.kernels import branch_norm, counter_dropout, gated_ffn

    c = s["case"]
    if c["kind"].startswith("ffn"):
        return (gated_ffn(s["x"], s["wg"], s["wu"], s["wd"], activation=c["act"]),)
    if c["kind"].startswith("dropout"):
        return (counter_dropout(s["x"], c["p"], s["seed"], c["offset"]),)
    return branch_norm(s["x"], s["h"], s["w"], post_weight=s["w_post"], gate=s["gate"], residual_scale=c["scale"],
                       p=c["p"], seed=s["seed"], eps=EPS, out_dtype=DTYPES[c["out"]])


def _run_own(s):
    if not s["case"]["kind"].endswith("_train"):
        with torch.no_grad():
            return [t for t in _call_own(s) if t is not None]
    outs = [t for t in _call_own(s) if t is not None]
    ups = [s[n] for n in ("dx_out", "dy") if s.get(n) is not None]
    grads = torch.autograd.grad(outs, [s[n] for n in s["leaves"]], ups)
    return [*(t.detach() for t in outs), *grads]


# ---- the plain forms ----------------------------------------------------------------------
def _philox_bits(n, seed, offset):
    """The 16 random bits of each of n elements: Philox4x32 with 7 rounds (Salmon, Moraes, Dror
    and Shaw 2011), 8 elements per counter value, in int64 arithmetic on the seed's device."""
    m32 = 0xFFFFFFFF
    j = torch.arange((n + 7) // 8, device=seed.device)
    c0, c1 = j & m32, j >> 32
    c2, c3 = torch.full_like(j, offset & m32), torch.full_like(j, (offset >> 32) & m32)
    k0, k1 = seed & m32, (seed >> 32) & m32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits of the products, as int64
        c0, c1, c2, c3 = ((b >> 32) & m32) ^ c1 ^ k0, b & m32, ((a >> 32) & m32) ^ c3 ^ k1, a & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]


def _keep(shape, p, seed, offset):
    """The factor of each element: 65536 / t where kept, else 0."""
    t = round((1.0 - p) * 65536)
    n = math.prod(shape)
    return (_philox_bits(n, seed, offset) < t).to(torch.float32).mul_(65536 / t if t else 0.0).view(shape)


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        sg = torch.sigmoid(g)
        return g * sg, sg * (1 + g * (1 - sg))
    if name == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    c = (2 / math.pi) ** 0.5
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_ffn(s):
    c = s["case"]
    x, wg, wu, wd = (s[n].detach().float() for n in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    act, slope = _act(c["act"], g)
    a = act * u
    outs = [a @ wd.t()]
    if "dy" in s:
        dy = s["dy"].float()
        da = dy @ wd
        dg, du = da * u * slope, da * act
        outs += [dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ a]
    return [t.to(s["x"].dtype) for t in outs]


def _plain_dropout(s):
    c = s["case"]
    k = _keep(s["x"].shape, c["p"], s["seed"], c["offset"])
    return [(s[n].detach().float() * k).to(s["x"].dtype) for n in ("x", "dy") if n in s]


def _plain_branch(s):
    c = s["case"]
    f32 = {n: s[n].detach().float() for n in ("x", "h", "w", "w_post", "gate", "dx_out", "dy") if s.get(n) is not None}
    x, h, rs = f32["x"], f32["h"], c["scale"]
    keep = _keep(h.shape, c["p"], s["seed"], 0) if c["p"] else None
    hd = h if keep is None else h * keep
    n = hd
    if "w_post" in f32:
        rh = torch.rsqrt(hd.square().mean(-1, keepdim=True) + EPS)
        n = hd * rh * f32["w_post"]
    x_out = rs * x + (n * f32["gate"] if "gate" in f32 else n)
    outs = [x_out.to(s["x"].dtype)]
    if "w" in f32:
        r = torch.rsqrt(x_out.square().mean(-1, keepdim=True) + EPS)
        outs.append((x_out * r * f32["w"]).to(DTYPES[c["out"]]))
    if "dx_out" not in f32:
        return outs
    t, grads = f32["dx_out"], {}
    if "w" in f32:
        xh, a = x_out * r, f32["dy"] * f32["w"]
        t = t + r * (a - xh * (a * xh).mean(-1, keepdim=True))
        grads["w"] = (f32["dy"] * xh).sum(0)
    grads["x"] = rs * t
    dn = t
    if "gate" in f32:
        grads["gate"] = (t * n).sum(0) if c["gate"] == "channel" else (t * n).sum(-1, keepdim=True)
        dn = t * f32["gate"]
    if "w_post" in f32:
        hh, b = hd * rh, dn * f32["w_post"]
        grads["w_post"] = (dn * hh).sum(0)
        dn = rh * (b - hh * (b * hh).mean(-1, keepdim=True))
    grads["h"] = dn if keep is None else dn * keep
    return outs + [grads[n].to(s[n].dtype) for n in s["leaves"]]


def _run_plain(s):
    kind = s["case"]["kind"]
    with torch.no_grad():
        return _plain_ffn(s) if kind.startswith("ffn") else _plain_dropout(s) if kind.startswith("dropout") else _plain_branch(s)


# ---- work ---------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    train = case["kind"].endswith("_train")
    e = size[case["dtype"]]
    if case["kind"].startswith("ffn"):
        T, d, f = case["rows"], case["d"], case["f"]
        return {"bytes": e * ((4 if train else 2) * T * d + (6 if train else 3) * d * f),
                "flops": (18 if train else 6) * T * d * f}
    if case["kind"].startswith("dropout"):
        return {"bytes": (4 if train else 2) * e * case["n"], "flops": (2 if train else 1) * case["n"]}
    n, s, o = case["rows"] * case["d"], size[case["stream"]], size[case["out"]] if case["pre"] else 0
    # x, h, x_out, y; in training also their gradients
    return {"bytes": (2 if train else 1) * n * (2 * s + e + o), "flops": (30 if train else 10) * n}


# ---- float64, from the definitions ----------------------------------------------------------
def _mask64(n, p, seed, offset):
    """The dropout's factors from numpy's unsigned integers, as a float64 tensor on the GPU."""
    lo, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    j = np.arange(-(-n // 8), dtype=np.uint64)
    ctr = [j & lo, j >> sh, np.full_like(j, offset & 0xFFFFFFFF), np.full_like(j, offset >> 32)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(7):
        p0, p1 = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(p1 >> sh) ^ ctr[1] ^ np.uint64(key[0]), p1 & lo, (p0 >> sh) ^ ctr[3] ^ np.uint64(key[1]), p0 & lo]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack(ctr, 1).astype("<u4").reshape(-1).view("<u2")[:n]  # low half first
    t = int(np.rint((1.0 - p) * 65536))
    kept = torch.from_numpy(bits < t).to(DEV)
    return kept.double() * (65536 / t if t else 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    w = {n: s[n].detach().double().requires_grad_() for n in s["leaves"]}
    up = [s[n].double() for n in ("dx_out", "dy") if s.get(n) is not None]
    if case["kind"].startswith("ffn"):
        F = torch.nn.functional
        act = {"silu": F.silu, "relu": torch.relu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}
        outs = [(act[case["act"]](w["x"] @ w["wg"].t()) * (w["x"] @ w["wu"].t())) @ w["wd"].t()]
    elif case["kind"].startswith("dropout"):
        outs = [w["x"] * _mask64(case["n"], case["p"], int(s["seed"]), case["offset"])]
    else:
        b = w["h"]
        if case["p"]:
            b = b * _mask64(b.numel(), case["p"], int(s["seed"]), 0).view(b.shape)
        if case["post"]:
            b = b / torch.sqrt((b * b).mean(1, keepdim=True) + EPS) * w["w_post"]
        if case["gate"] != "none":
            b = b * w["gate"]
        z = case["scale"] * w["x"] + b
        outs = [z]
        if case["pre"]:
            outs.append(z / torch.sqrt((z * z).mean(1, keepdim=True) + EPS) * w["w"])
    if not case["kind"].endswith("_train"):
        return [t.detach() for t in outs]
    grads = torch.autograd.grad(outs, [w[n] for n in s["leaves"]], up)
    return [*(t.detach() for t in outs), *grads]
