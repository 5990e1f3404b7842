"""The transformer block's and the LM's options (fused feed-forward, counter-based dropout, post
norms, layer scale, residual scale): all of them in one run, against the same modules composed
from torch's ops, and what they leave as it was."""
import copy

import pytest
import torch
import torch.nn.functional as F

from dsalt import _hip
from dsalt.kernels import counter_dropout
from dsalt.kernels.gated_ffn import torch_gated_ffn
from dsalt.model import DSALTLMHeadModel
from dsalt.modules import CounterDropout, DSALTTransformerBlock, SwiGLUFFN

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
OPTIONS = dict(post_norm=True, layer_scale=0.2, residual_scale=0.9, fused_ffn=True, counter_dropout=True)
LENS = [200, 57, 131]
CU = [0, 200, 257, 388]


def block(dtype=FP, dropout=0.1, **kw):
    torch.manual_seed(5)
    b = DSALTTransformerBlock(128, 2, 4, 40, 4, 256, 264, dropout=dropout, layer_idx=2, **{**OPTIONS, **kw}).to(DEV, dtype).train()
    with torch.no_grad():
        for n, p in b.named_parameters():
            if "norm" in n or n.endswith("gate"):
                p.add_(0.2 * torch.randn(p.shape, device=DEV).to(dtype))
    return b


def composed(b, x, cu, seed, autocast=None):
    """The block's formulas in torch's ops, around the same attention module."""
    def rms(t, norm):
        return F.rms_norm(t.float(), (t.shape[-1],), norm.weight.float(), norm.eps)

    def join(x, o, post, gate):
        n = rms(o, post) if post is not None else o.float()
        n = n if gate is None else gate.float() * n
        return (b.residual_scale * x.float() + n).to(x.dtype)

    o, aux = b.attn(rms(x, b.attn_norm).to(x.dtype), cu_seqlens=cu, max_seqlen=256)
    x = join(x, o, b.attn_post_norm, b.attn_gate)
    h = rms(x, b.ffn_norm).to(x.dtype)
    f = torch_gated_ffn(h, b.ffn.gate_proj.weight, b.ffn.up_proj.weight, b.ffn.down_proj.weight, b.ffn.activation)
    if b.training and b.ffn.drop.p > 0:
        f = counter_dropout(f, b.ffn.drop.p, seed, b.layer_idx + 1)
    return join(x, f, b.ffn_post_norm, b.ffn_gate), aux


@pytest.mark.parametrize("dtype,autocast", [(FP, None), (BF, None), (HF, None), (FP, BF)])
@pytest.mark.parametrize("activation,extra", [("silu", {}), ("gelu_tanh", {}), ("relu", {"post_norm": False}),
                                              ("gelu", {"layer_scale": None, "residual_scale": 1.0})])
def test_block(dtype, autocast, activation, extra):
    print(f"block options {dtype} autocast={autocast} {activation} {extra}", flush=True)
    b = block(dtype, activation=activation, **extra)
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    x = torch.randn(CU[-1], 128, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(dtype)
    dy = torch.randn(CU[-1], 128, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(dtype)
    seed = torch.tensor([9], device=DEV)
    got, want = [], []
    for out in (got, want):
        xi = x.clone().requires_grad_()
        b.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=autocast or BF, enabled=autocast is not None):
            if out is got:
                y, _, _ = b.join_branches(xi, b.attn_norm(xi), None, seed, cu_seqlens=cu, max_seqlen=256)
            else:
                y, _ = composed(b, xi, cu, seed)
        y.backward(dy)
        out += [("y", y.detach()), ("x", xi.grad)] + [(n, p.grad) for n, p in b.named_parameters() if p.grad is not None]
    assert [n for n, _ in got] == [n for n, _ in want]
    # both sides round at every op's output in the compute dtype: some ten roundings in a chain
    # of up to half a step each, which add up like a random walk; windows and landmarks are
    # whole-number decisions on roundings that the two sides' norms may take differently, in
    # a few rows
    u = torch.finfo(autocast or dtype).eps / 2 if (autocast or dtype) != FP else 2.0 ** -11  # fp32 attention computes in fp16
    # relu's slope jumps: the two sides' h differ by a rounding, g = h Wg^T then by about u of its
    # scale s, and of gates with density 1 / (s sqrt(2 pi)) at 0 a share of 2 u / sqrt(2 pi) < u lies
    # within u s of it. Where the slopes differ the whole gradient of that gate does, in u of all
    # gates against the half that pass: sqrt(2 u) of its norm
    tol = 24 * u + ((2 * u) ** 0.5 if activation == "relu" else 0.0)
    for (n, a), (_, c) in zip(got, want):
        assert a.dtype == c.dtype and a.shape == c.shape, n
        err, size = float((a.float() - c.float()).norm()), float(c.float().norm())
        assert err <= tol * size + 1e-6, (n, err / max(size, 1e-12), u)


def test_ffn_fused_against_separate():
    for dtype in (BF, HF):
        torch.manual_seed(1)
        ffn = SwiGLUFFN(128, 264, fused=True, activation="gelu").to(DEV, dtype)
        x = torch.randn(3, 41, 128, device=DEV).to(dtype).requires_grad_()
        y = ffn(x)
        want = torch_gated_ffn(x.double(), *(m.weight.double() for m in (ffn.gate_proj, ffn.up_proj, ffn.down_proj)), "gelu")
        assert float((y.double() - want).norm()) <= 4 * torch.finfo(dtype).eps / 2 * float(want.norm())
        hooked = copy.deepcopy(ffn)
        calls = []
        hooked.up_proj.register_forward_hook(lambda *a: calls.append(1))
        assert float((hooked(x).double() - want).norm()) <= 8 * torch.finfo(dtype).eps / 2 * float(want.norm()) and calls
    ffn = SwiGLUFFN(128, 264, fused=True).to(DEV)  # fp32 projections run as without the option
    x = torch.randn(9, 128, device=DEV)
    other = SwiGLUFFN(128, 264).to(DEV)
    other.load_state_dict(ffn.state_dict())
    assert torch.equal(ffn(x), other(x))


def test_defaults_have_no_new_parameters():
    a = DSALTTransformerBlock(128, 2, 4, 40, 4, 256, 264)
    assert not a.joins_branches and not any("post_norm" in n or n.endswith("_gate") for n, _ in a.named_parameters())
    names = {n for n, _ in DSALTTransformerBlock(128, 2, 4, 40, 4, 256, 264, **OPTIONS).named_parameters()}
    assert names - {n for n, _ in a.named_parameters()} == {"attn_post_norm.weight", "ffn_post_norm.weight", "attn_gate", "ffn_gate"}
    with pytest.raises(ValueError, match="activation"):
        SwiGLUFFN(64, 64, activation="tanh")
    with pytest.raises(ValueError, match="probability"):
        CounterDropout(1.5)


def test_counter_dropout_module():
    m = CounterDropout(0.25).to(DEV)
    x = torch.randn(1000, device=DEV)
    assert m.eval()(x) is x
    m.train()
    torch.manual_seed(3)
    a = m(x)
    b = m(x)
    torch.manual_seed(3)
    assert torch.equal(m(x), a) and not torch.equal(a, b)
    assert torch.equal(m(x, 7, 2), counter_dropout(x, 0.25, 7, 2))
    with pytest.raises(_hip.DsaltError):
        m(x.cpu(), 1)


def test_replaced_and_hooked_norms_are_called():
    b = block(dropout=0.0, fused_ffn=False)
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    x = torch.randn(CU[-1], 128, device=DEV)
    with torch.no_grad():
        want, _ = b(x, cu_seqlens=cu, max_seqlen=256)
        calls = []
        for n in (b.attn_post_norm, b.ffn_norm, b.ffn_post_norm):
            n.register_forward_hook(lambda m, i, o: calls.append(m))
        got, _ = b(x, cu_seqlens=cu, max_seqlen=256)
    assert [id(c) for c in calls] == [id(n) for n in (b.attn_post_norm, b.ffn_norm, b.ffn_post_norm)]
    assert float((got - want).norm()) <= 16 * 2.0 ** -11 * float(want.norm())


def lm(**kw):
    torch.manual_seed(2)
    return DSALTLMHeadModel(vocab_size=500, d_model=128, n_layers=3, n_heads=2, n_min=4, n_max=40, k_lmk=4, max_seq_len=256,
                            **{**OPTIONS, "dropout": 0.1, **kw}).to(DEV)


def test_lm_training_step():
    """Loss and gradients of a step: the same with the same torch seed, with checkpointing, and not
    with another seed; every parameter gets a finite gradient."""
    m = lm().train()
    ids = torch.randint(0, 500, (CU[-1],), device=DEV)
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)

    def step(seed, **kw):
        torch.manual_seed(seed)
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=BF):
            loss = m(ids, cu_seqlens=cu, max_seqlen=256, labels=ids, **kw)["loss"]
        loss.backward()
        return loss.detach(), {n: p.grad for n, p in m.named_parameters() if p.grad is not None}

    a, b, c, d = step(1), step(1), step(2), step(1, gradient_checkpointing=True)
    assert torch.equal(a[0], b[0]) and not torch.equal(a[0], c[0]) and torch.equal(a[0], d[0])
    for n in a[1]:
        assert torch.isfinite(a[1][n]).all(), n
        assert torch.equal(a[1][n], b[1][n]) and torch.equal(a[1][n], d[1][n]), n
    missing = [n for n, p in m.named_parameters() if n not in a[1]]
    assert not missing, missing


@pytest.mark.parametrize("dtype", [FP, BF])
def test_lm_inference_takes_the_next_norms_along(dtype):
    """The LM's loop is join_branches of every layer with the norm that follows it, to the bit; and each
    layer by itself gives the same stream, whose norm differs by the stream's rounding alone.
    (Compared layer by layer on the same input: behind a norm that differs in its last bit a
    landmark near a tie may be another one, and every later query of the sequence sees it.)"""
    m = lm().to(dtype).eval()
    m.set_collect_last_P(False)
    ids = torch.randint(0, 500, (CU[-1],), device=DEV)
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        got = m(ids, cu_seqlens=cu, max_seqlen=256)["logits"]
        x = m.embed_tokens(ids)
        h = m.layers[0].attn_norm(x)
        for i, layer in enumerate(m.layers):
            after = m.layers[i + 1].attn_norm if i + 1 < len(m.layers) else m.final_norm
            alone, none, _ = layer.join_branches(x, h, None, cu_seqlens=cu, max_seqlen=256)
            x, h, _ = layer.join_branches(x, h, after, cu_seqlens=cu, max_seqlen=256)
            assert none is None and torch.equal(alone, x)
            want = after(x).double()
            u = torch.finfo(dtype).eps / 2
            # y's own rounding and that of the stream on the other side, whose rms moves less
            assert bool(((h.double() - want).abs() <= (4 * u + 2.0 ** -20) * want.abs() + 2.0 ** -18).all())
        assert torch.equal(got, m.lm_head(h))
        assert torch.equal(got, m(ids, cu_seqlens=cu, max_seqlen=256)["logits"])


def test_lm_inference_in_a_graph():
    """The LM with every option, captured and replayed over new tokens, with eager calls between."""
    m = lm().to(BF).eval()
    m.set_collect_last_P(False)
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    batches = [torch.randint(0, 500, (CU[-1],), device=DEV) for _ in range(4)]
    ids = batches[0].clone()
    with torch.no_grad():
        want = [m(b, cu_seqlens=cu, max_seqlen=256)["logits"] for b in batches]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(ids, cu_seqlens=cu, max_seqlen=256)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(ids, cu_seqlens=cu, max_seqlen=256)["logits"]
        for i, b in enumerate(batches):
            print(f"lm graph replay {i}", flush=True)
            ids.copy_(b)
            graph.replay()
            assert torch.equal(out, want[i])
            assert torch.equal(m(batches[i - 1], cu_seqlens=cu, max_seqlen=256)["logits"], want[i - 1])


def test_counter_dropout_draws_anew_on_every_replay():
    m = CounterDropout(0.25).train()
    x = torch.ones(4096, device=DEV)
    m(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x)
    seen = []
    for i in range(4):
        print(f"dropout replay {i}", flush=True)
        graph.replay()
        seen.append(out.clone())
        m(x)  # an eager draw between
        # 4096 draws of a share of 3/4: five standard deviations of sqrt(3 / 16 / 4096)
        assert abs(float((out != 0).float().mean()) - 0.75) <= 5 * (3 / 16 / 4096) ** 0.5
    assert all(not torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])


def test_unpacked_input_and_odd_widths():
    """[1, T, d] input (whose attention takes no dropout of its own); a hidden width that the fused
    feed-forward does not take runs as separate projections."""
    for d_ff in (264, 260):
        torch.manual_seed(5)
        b = DSALTTransformerBlock(128, 2, 4, 40, 4, 256, d_ff, dropout=0.0, layer_idx=1, **OPTIONS).to(DEV, BF).train()
        b.ffn.drop.p = 0.1
        x = torch.randn(1, 150, 128, device=DEV, dtype=BF, requires_grad=True)
        res = []
        for checkpoint in (False, True):
            torch.manual_seed(9)
            y, _ = b(x, gradient_checkpointing=checkpoint)
            res.append((y, *torch.autograd.grad(y.float().square().sum(), [x, *b.parameters()], allow_unused=True)))
        assert y.shape == x.shape
        for p, q in zip(*res):
            assert (p is None and q is None) or (torch.isfinite(p).all() and torch.equal(p, q))
        missing = [n for (n, _), g in zip(b.named_parameters(), res[0][2:]) if g is None]
        assert not [n for n in missing if "ffn" in n or "gate" in n and "win" not in n or "norm" in n], missing


class Widened(torch.nn.Module):
    """A module's result in fp32, as torch's normalisations give it under autocast."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x).float()


REPLACED = {"attn_post_norm": lambda b: torch.nn.LayerNorm(128), "ffn_post_norm": lambda b: torch.nn.LayerNorm(128),
            "ffn": lambda b: Widened(copy.deepcopy(b.ffn))}


@pytest.mark.parametrize("which", list(REPLACED))
@pytest.mark.parametrize("stream,weights,autocast", [(BF, FP, BF), (HF, FP, HF), (BF, BF, None), (FP, FP, BF)])
def test_replaced_modules_that_return_fp32(which, stream, weights, autocast):
    """A replaced norm or feed-forward that returns fp32 beside a 16-bit stream: the sum is fp32, as
    torch's addition promotes it. Values and gradients against the composition in torch's ops."""
    print(f"replaced {which} {stream} {weights} {autocast}", flush=True)
    b = block(weights, dropout=0.0)
    setattr(b, which, REPLACED[which](b).to(DEV))
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    x, dy = (torch.randn(CU[-1], 128, device=DEV, generator=torch.Generator(DEV).manual_seed(s)).to(stream) for s in (1, 2))

    def norm(m, t):  # LayerNorm in fp32 where the run is without autocast
        if type(m) is not torch.nn.LayerNorm:
            return F.rms_norm(t.float(), (128,), m.weight.float(), m.eps)
        return F.layer_norm(t.float(), (128,), m.weight.float(), m.bias.float(), m.eps)

    def composed_run(xi):
        o, _ = b.attn(norm(b.attn_norm, xi).to(xi.dtype), cu_seqlens=cu, max_seqlen=256)
        z = b.residual_scale * xi.float() + b.attn_gate.float() * norm(b.attn_post_norm, o)
        if which != "attn_post_norm":
            z = z.to(xi.dtype)
        f = b.ffn(norm(b.ffn_norm, z).to(autocast or weights))
        return b.residual_scale * z.float() + b.ffn_gate.float() * norm(b.ffn_post_norm, f)

    if weights != FP:  # without autocast LayerNorm's input has its weight's type
        for n in ("attn_post_norm", "ffn_post_norm"):
            m = getattr(b, n)
            if type(m) is torch.nn.LayerNorm:
                m.forward = lambda t, m=m: F.layer_norm(t.float(), (128,), m.weight, m.bias, m.eps)
    res = []
    for fn in (lambda xi: b(xi, cu_seqlens=cu, max_seqlen=256)[0], composed_run):
        xi = x.clone().requires_grad_()
        b.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=autocast or BF, enabled=autocast is not None):
            y = fn(xi)
        y.backward(dy.to(y.dtype))
        res.append([("y", y.detach()), ("x", xi.grad)] + [(n, p.grad) for n, p in b.named_parameters() if p.grad is not None])
    assert res[0][0][1].dtype == FP and [n for n, _ in res[0]] == [n for n, _ in res[1]]
    u = torch.finfo(autocast or weights).eps / 2  # test_block's count of roundings
    for (n, a), (_, c) in zip(*res):
        assert a.dtype == c.dtype, n
        err, size = float((a.float() - c.float()).norm()), float(c.float().norm())
        assert err <= 24 * u * size + 1e-6, (n, err / max(size, 1e-12), u)


@pytest.mark.parametrize("which", ["attn_post_norm", "ffn_post_norm"])
def test_lm_with_replaced_norms_under_autocast(which):
    m = lm().train()
    for layer in m.layers:
        setattr(layer, which, torch.nn.LayerNorm(128).to(DEV))
    ids = torch.randint(0, 500, (CU[-1],), device=DEV)
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    with torch.autocast("cuda", dtype=BF):
        loss = m(ids, cu_seqlens=cu, max_seqlen=256, labels=ids)["loss"]
    loss.backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())
    with torch.no_grad(), torch.autocast("cuda", dtype=BF):
        assert bool(torch.isfinite(m.eval()(ids, cu_seqlens=cu, max_seqlen=256)["logits"]).all())


@pytest.mark.parametrize("fused", [False, True])
def test_projections_without_a_weight(fused):
    """A projection replaced by a module that has no weight of its own is called as it is, in training too."""
    torch.manual_seed(1)
    ffn = SwiGLUFFN(64, 128, fused=fused).to(DEV)
    x = torch.randn(5, 64, device=DEV, requires_grad=True)
    want, = torch.autograd.grad(ffn(x).sum(), x)
    ffn.up_proj = Widened(ffn.up_proj)
    got, = torch.autograd.grad(ffn(x).sum(), x)
    # fp32 sums of 64 and 128 terms in another order on either side
    assert float((got - want).norm()) <= 2.0 ** -17 * float(want.norm())


@pytest.mark.parametrize("how", ["replaced", "hooked", "projection replaced", "projection hooked"])
def test_feed_forward_sees_the_stream_type(how):
    """Under autocast an fp32 stream's norm is rounded for the feed-forward only where plain projections,
    which round it themselves, are all that reads it."""
    b = block(FP, dropout=0.0, fused_ffn=False)
    seen = []
    if how == "replaced":
        b.ffn = Widened(b.ffn)
        target = b.ffn
    else:
        target = b.ffn if how == "hooked" else b.ffn.up_proj
        if how == "projection replaced":
            target = b.ffn.up_proj = Widened(b.ffn.up_proj)
    target.register_forward_pre_hook(lambda m, i: seen.append(i[0].dtype))
    cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
    x = torch.randn(CU[-1], 128, device=DEV)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), torch.autocast("cuda", dtype=BF):
            b(x, cu_seqlens=cu, max_seqlen=256)
    assert seen == [FP, FP]


def test_norms_and_gates_of_another_type():
    """Post norms and gates in the other 16-bit type than the stream's are read at their own value."""
    b = block(BF, dropout=0.0)
    with torch.no_grad():
        for n in ("attn_post_norm", "ffn_post_norm"):
            getattr(b, n).weight.data = getattr(b, n).weight.data.to(HF)
        b.ffn_gate.data = b.ffn_gate.data.to(HF)
        cu = torch.tensor(CU, dtype=torch.int32, device=DEV)
        x = torch.randn(CU[-1], 128, device=DEV).to(BF)
        got, _ = b(x, cu_seqlens=cu, max_seqlen=256)
        for n in ("attn_post_norm", "ffn_post_norm"):
            getattr(b, n).weight.data = getattr(b, n).weight.data.float()
        b.ffn_gate.data = b.ffn_gate.data.float()
        assert got.dtype == BF and torch.equal(got, b(x, cu_seqlens=cu, max_seqlen=256)[0])
