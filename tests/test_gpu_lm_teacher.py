"""The LM's options on layer norm, distillation and 8-bit layers, each alone and as they are used together:
a teacher whose feed-forwards and head run in 8 bits answers, a student with layer norms learns from it."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from dsalt import DsaltError
from dsalt.kernels import FP8Linear, LayerNorm, add_layer_norm, distill_loss, fp8_linear, fp8_quantize
from dsalt.model import DSALTLMHeadModel
from dsalt.modules import DSALTTransformerBlock, SwiGLUFFN

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


def lm(seed=0, **kw):
    torch.manual_seed(seed)
    kw = dict(vocab_size=500, d_model=128, n_layers=2, n_heads=2, n_min=4, n_max=40, k_lmk=4, max_seq_len=256, **kw)
    model = DSALTLMHeadModel(**kw).to(DEV)
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, LayerNorm):
                m.weight.normal_(1.0, 0.2)
                m.bias.normal_(0.0, 0.2)
    model.set_collect_last_P(False)
    return model


def packed(seed, lens=(37, 100, 9, 61)):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 500, (sum(lens),), generator=g).to(DEV)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    return ids, cu


class TorchNorm(nn.Module):
    """A LayerNorm's values in torch's ops, as a module that no pass of the package takes in."""

    def __init__(self, norm):
        super().__init__()
        self.norm = norm
        self.eps, self.normalized_shape, self.weight, self.bias = norm.eps, norm.normalized_shape, norm.weight, norm.bias

    def forward(self, x):
        return F.layer_norm(x.float(), self.normalized_shape, self.weight.float(), self.bias.float(), self.eps).to(x.dtype)


def with_torch_norms(model):
    for layer in model.layers:
        layer.attn_norm, layer.ffn_norm = TorchNorm(layer.attn_norm), TorchNorm(layer.ffn_norm)
        layer._fuse_norms = False
    model.final_norm = TorchNorm(model.final_norm)
    return model


@pytest.mark.parametrize("more", [{}, {"post_norm": True, "layer_scale": 0.5}, {"fused_ffn": True, "activation": "gelu"}])
def test_layer_norm_model_trains(more):
    """Loss and gradients of a model with layer norms, against the same model with torch's norms (fp32: sums
    in another order, through two blocks)."""
    ids, cu = packed(1)
    y = torch.roll(ids, -1)
    a, b = lm(norm="layer", **more), with_torch_norms(lm(norm="layer", **more))
    assert {n for n, _ in a.named_parameters() if "norm" in n and n.endswith("bias")} >= {"final_norm.bias", "layers.0.ffn_norm.bias"}
    out = []
    for m in (a, b):
        m.train()
        loss = m(ids, cu_seqlens=cu, labels=y)["loss"]
        loss.backward()
        out.append((loss, {n.replace(".norm.", "."): p.grad for n, p in m.named_parameters()}))
    assert abs(float(out[0][0] - out[1][0])) < 1e-4
    for n, g in out[0][1].items():
        w = out[1][1][n]
        assert float((g - w).norm()) <= 5e-3 * float(w.norm()) + 1e-6, n  # the attention computes in fp16


@pytest.mark.parametrize("dtype", [BF, FP])
def test_layer_norm_model_answers(dtype):
    ids, cu = packed(2)
    a, b = lm(norm="layer").to(dtype).eval(), with_torch_norms(lm(norm="layer").to(dtype).eval())
    with torch.no_grad():
        u, v = (m(ids, cu_seqlens=cu)["logits"].float() for m in (a, b))
        single = a(ids[:37], cu_seqlens=cu[:2])["logits"].float()
    # roundings of 2^-9 at some ten places of the bf16 stream (two blocks) that the passes place otherwise
    assert float((u - v).norm() / v.norm()) < (10 * 2.0 ** -9 if dtype is BF else 1e-3)
    assert float((single - u[:37]).norm() / single.norm()) < (10 * 2.0 ** -9 if dtype is BF else 1e-3)


def test_layer_norm_block_under_autocast():
    """An fp32 stream with 16-bit branches: the add takes the branch as it is, the norm comes out in the projections'
    type; gradients against torch's norms."""
    x = torch.randn(60, 128, device=DEV)
    cu = torch.tensor([0, 25, 60], dtype=torch.int32, device=DEV)
    grads = []
    for torch_norms in (False, True):
        torch.manual_seed(3)
        block = DSALTTransformerBlock(128, 2, 4, 40, 4, 256, 192, norm="layer").to(DEV).train()
        if torch_norms:
            block.attn_norm, block.ffn_norm, block._fuse_norms = TorchNorm(block.attn_norm), TorchNorm(block.ffn_norm), False
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=BF):
            out, _ = block(leaf, cu_seqlens=cu)
        out.square().sum().backward()
        grads.append((out.detach(), leaf.grad))
    for u, v in zip(*grads):
        assert u.dtype == FP and float((u - v).norm() / v.norm()) < 2e-2  # bf16 products on both sides


def test_norm_option_is_checked():
    for cls in (lambda n: lm(norm=n), lambda n: DSALTTransformerBlock(64, 2, 4, 40, 4, 256, 96, norm=n)):
        with pytest.raises(ValueError, match="norm must be"):
            cls("batch")


@pytest.mark.parametrize("labels,lam", [(False, 0.0), (True, 0.0), (True, 0.4)])
@pytest.mark.parametrize("chunk", [2048, 50])
def test_distilled_loss_is_that_of_the_logits(labels, lam, chunk):
    """The chunked loss and every gradient equal those of distill_loss on the model's own logits."""
    ids, cu = packed(4)
    T = ids.numel()
    g = torch.Generator(device=DEV).manual_seed(9)
    zt = torch.randn(T, 12, device=DEV, generator=g) * 2
    ti = torch.rand(T, 500, device=DEV, generator=g).topk(12).indices
    y = torch.roll(ids, -1) if labels else None
    if labels:
        y[::7] = -100
    model = lm(lm_head_chunk_size=chunk).train()
    out = model(ids, cu_seqlens=cu, labels=y, teacher_logits=zt, teacher_ids=ti, temperature=2.0, label_weight=lam)
    assert out["logits"] is None
    out["loss"].backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    logits = model(ids, cu_seqlens=cu)["logits"]
    want = distill_loss(logits, zt, ti, y, temperature=2.0, label_weight=lam)
    want.backward()
    assert abs(float(out["loss"] - want)) < 1e-5 * max(1.0, float(want))
    for n, p in model.named_parameters():
        assert float((got[n] - p.grad).norm()) <= 1e-3 * float(p.grad.norm()) + 1e-7, n
    with pytest.raises(ValueError, match="together"):
        model(ids, cu_seqlens=cu, teacher_ids=ti)


@pytest.mark.parametrize("rows", [1, 20, 33, 300])
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_quantised_feed_forward(rows, activation):
    """One quantisation serves gate and up; with a hook, or few rows, the layers run by themselves: the same bits."""
    torch.manual_seed(5)
    ffn = SwiGLUFFN(128, 352, activation=activation).to(DEV, BF).eval().quantize_fp8()
    assert all(type(m) is FP8Linear for m in (ffn.gate_proj, ffn.up_proj, ffn.down_proj))
    x = torch.randn(rows, 128, device=DEV, dtype=BF)
    with torch.no_grad():
        got = ffn(x)
        calls = []
        ffn.gate_proj.register_forward_hook(lambda *a: calls.append(1))
        assert torch.equal(ffn(x), got) and len(calls) == 1
        act = F.silu if activation == "silu" else F.gelu
        g, u = (fp8_linear(x, m.weight_q, m.weight_scale) for m in (ffn.gate_proj, ffn.up_proj))
        assert torch.equal(got, fp8_linear(act(g) * u, ffn.down_proj.weight_q, ffn.down_proj.weight_scale))
    with pytest.raises(DsaltError, match="inference"):
        ffn(x.requires_grad_())


def test_quantised_model():
    """Logits of the quantised model against the model's own; its loss, its state, autocast, and training refused."""
    ids, cu = packed(6)
    model, full = lm().to(BF).eval(), lm().to(BF).eval()
    keys = set(model.state_dict())
    model.quantize_fp8()
    assert type(model.lm_head) is FP8Linear and "lm_head.weight" in keys and "lm_head.weight_bits" in model.state_dict()
    with torch.no_grad():
        u, v = (m(ids, cu_seqlens=cu)["logits"].float() for m in (model, full))
        # e4m3 operands: 2^-4 at most, 2^-5.8 in the mean square, of each factor of three products in a row
        assert float((u - v).norm() / v.norm()) < 3 * 2 * 2.0 ** -4
        loss = model(ids, cu_seqlens=cu, labels=torch.roll(ids, -1))["loss"]
        assert abs(float(loss) - float(F.cross_entropy(u, torch.roll(ids, -1)))) < 2e-2  # bf16 logits
        wide = lm().eval().quantize_fp8(lm_head=False)
        assert type(wide.lm_head) is nn.Linear
        with torch.autocast("cuda", dtype=BF):
            assert bool(torch.isfinite(wide(ids, cu_seqlens=cu)["logits"]).all())
        torch.manual_seed(1)
        other = lm(seed=8).to(BF).eval().quantize_fp8()
        other.load_state_dict(model.state_dict())
        assert torch.equal(other(ids, cu_seqlens=cu)["logits"].float(), u)
    with pytest.raises(DsaltError, match="inference"):
        model(ids, cu_seqlens=cu, labels=ids)


def test_teacher_and_student():
    """A run of all of it: the teacher's top logits in 8 bits, then training steps of the student under autocast; the
    same through a captured graph, replayed, with eager steps between."""
    ids, cu = packed(7)
    teacher = lm(seed=1, norm="layer").to(BF).eval().quantize_fp8()
    student = lm(seed=2, norm="layer", activation="gelu", fused_ffn=True).train()
    y = torch.roll(ids, -1)
    y[36] = y[136] = -100

    def answer():
        with torch.no_grad():
            return teacher(ids, cu_seqlens=cu)["logits"].float().topk(16)

    zt, ti = answer()
    q, s = fp8_quantize(torch.randn(40, 128, device=DEV))
    assert q.shape == (40, 128) and s.shape == (40, 1)

    def step():
        for p in student.parameters():
            p.grad = None
        with torch.autocast("cuda", dtype=BF):
            out = student(ids, cu_seqlens=cu, labels=y, teacher_logits=zt, teacher_ids=ti, temperature=2.0, label_weight=0.5)
        out["loss"].backward()
        return out["loss"].detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    eager_loss = step()
    eager = {n: p.grad.clone() for n, p in student.named_parameters()}
    assert bool(torch.isfinite(eager_loss)) and all(bool(torch.isfinite(g).all()) and bool(g.any()) for g in eager.values())
    with torch.no_grad():
        student.eval()
        logits = student(ids, cu_seqlens=cu)["logits"]
        student.train()
    # the attention selects and computes otherwise in training (soft windows): the loss is of the same size only
    near = distill_loss(logits, zt, ti, y, temperature=2.0, label_weight=0.5)
    assert 0.5 * float(near) < float(eager_loss) < 2 * float(near)
    for p in student.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    captured = {n: p.grad for n, p in student.named_parameters()}
    for k in range(3):
        ids.copy_(packed(20 + k)[0])
        y.copy_(torch.roll(ids, -1))
        new = answer()
        zt.copy_(new[0])
        ti.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        kept, grads = loss.clone(), {n: g.clone() for n, g in captured.items()}
        assert torch.equal(kept, step())
        for n, p in student.named_parameters():
            assert torch.equal(grads[n], p.grad), n
