"""Calls of the layer norm, the distillation loss and the 8-bit products that their documentation allows
besides the plain ones: one tensor in two places, tensors made under inference_mode, threads at once, inside
torch.compile, under checkpointing."""
import threading

import pytest
import torch
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

import dsalt
from dsalt.kernels import FP8Linear, add_layer_norm, distill_loss, fp8_linear, fp8_quantize, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, FP])
def test_gradients_of_both_sides_are_their_own(dtype):
    x, h = (torch.randn(40, 64, device=DEV, dtype=dtype).requires_grad_() for _ in range(2))
    for i, f in enumerate((lambda a, y: a.sum() + (y * y).sum(), lambda a, y: a.sum(), lambda a, y: y.sum())):
        x.grad = h.grad = None
        f(*add_layer_norm(x, h)).backward()
        assert x.grad.data_ptr() != h.grad.data_ptr(), i
        assert torch.equal(x.grad, h.grad), i


def test_one_tensor_in_two_places():
    """fp32 throughout: sums of 64 products, 64 eps relative to their terms' magnitudes (below 100 each)."""
    tol = 64 * torch.finfo(FP).eps * 100
    x = torch.randn(40, 64, device=DEV).requires_grad_()
    w = torch.randn(64, device=DEV).requires_grad_()
    dy = torch.randn(40, 64, device=DEV)
    z, y = add_layer_norm(x, x, w, w)
    got = torch.autograd.grad([z, y], [x, w], [dy, dy])
    z = x.double() * 2
    want = torch.autograd.grad([z, F.layer_norm(z, (64,), w.double(), w.double())], [x, w], [dy.double(), dy.double()])
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= tol
    v = torch.randn(64, device=DEV).requires_grad_()
    got, = torch.autograd.grad(layer_norm(v, v, v), v, dy[0])
    u = v.detach().double().requires_grad_()
    want, = torch.autograd.grad(F.layer_norm(u, (64,), u, u), u, dy[0].double())
    assert (got - want).abs().max() <= tol


def test_a_model_that_teaches_itself():
    """Teacher and student one tensor, a slot for every token: no loss and no gradient but roundings (300
    terms of at most one, eps each)."""
    s = torch.randn(50, 300, device=DEV).requires_grad_()
    ids = torch.arange(300, device=DEV).expand(50, 300)
    loss = distill_loss(s, s, ids)
    loss.backward()
    eps = torch.finfo(FP).eps
    assert abs(loss.item()) <= 300 * eps and s.grad.abs().max() <= 300 * eps


@pytest.mark.parametrize("labels", [False, True])
def test_teacher_under_inference_mode(labels):
    s = torch.randn(50, 300, device=DEV).requires_grad_()
    with torch.inference_mode():
        z, ids = torch.randn(50, 300, device=DEV).topk(8)
        y = torch.randint(0, 300, (50,), device=DEV) if labels else None
    kw = {"temperature": 2.0, "label_weight": 0.3 if labels else 0.0}
    loss = distill_loss(s, z, ids, y, **kw)
    plain = distill_loss(s, z.clone(), ids.clone(), None if y is None else y.clone(), **kw)
    assert torch.equal(loss, plain)
    got, want = (torch.autograd.grad(v, s)[0] for v in (loss, plain))
    assert torch.equal(got, want)
    g, = torch.autograd.grad(distill_loss(s, z, ids, y, **kw), s, create_graph=True)
    g.square().sum().backward()
    assert s.grad.isfinite().all()


def test_frozen_parts_under_inference_mode():
    x = torch.randn(40, 64, device=DEV, dtype=BF).requires_grad_()
    with torch.inference_mode():
        h, w = torch.randn(40, 64, device=DEV, dtype=BF), torch.randn(64, device=DEV)
        lin = FP8Linear.from_linear(torch.nn.Linear(64, 48).to(DEV))
    dy = torch.randn(40, 64, device=DEV, dtype=BF)
    got = torch.autograd.grad(add_layer_norm(x, h, w)[1], x, dy)[0]
    assert torch.equal(got, torch.autograd.grad(add_layer_norm(x, h.clone(), w.clone())[1], x, dy)[0])
    assert lin(x.detach()).isfinite().all()
    bias = torch.zeros(64, device=DEV).requires_grad_()  # of rows that are an inference tensor
    got, = torch.autograd.grad(layer_norm(h, None, bias), bias, dy)
    assert torch.equal(got, torch.autograd.grad(layer_norm(h.clone(), None, bias), bias, dy)[0])


def test_change_in_place_is_noticed():
    z, ids = torch.randn(50, 4, device=DEV), torch.randint(0, 300, (50, 4), device=DEV)
    s = torch.randn(50, 300, device=DEV).requires_grad_() * 1
    loss = distill_loss(s, z, ids)
    s.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    x = torch.randn(4, 64, device=DEV).requires_grad_() * 1
    y = layer_norm(x)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def operands(seed, rows):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    return {"x": rnd(rows, 256), "h": rnd(rows, 256), "w": rnd(256), "head": rnd(520, 256), "z": rnd(rows, 8),
            "ids": torch.randint(0, 520, (rows, 8), device=DEV, generator=g)}


def chain(x, h, w, t):
    """The operators as a model chains them: a norm, a frozen 8-bit layer beside, a loss."""
    s, y = add_layer_norm(x, h, w)
    with torch.no_grad():
        frozen = fp8_linear(y, *fp8_quantize(t["head"], tile=True))
    return s, frozen, distill_loss(F.linear(layer_norm(y), t["head"]), t["z"], t["ids"], temperature=2.0)


def step(t, fn=chain):
    leaves = [t[n].clone().requires_grad_() for n in ("x", "h", "w")]
    s, frozen, loss = fn(*leaves, t)
    return [s.detach(), frozen, loss.detach(), *torch.autograd.grad([s, loss], leaves, [torch.ones_like(s), torch.ones_like(loss)])]


def test_threads_with_streams_of_their_own():
    """Four threads, each on its own stream with its own operands, get what one thread gets."""
    cases = [operands(i, rows) for i, rows in enumerate((3, 40, 300, 900))]
    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = step(cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # a thread's failure is the test's
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_inside_compile_and_checkpoint():
    t = operands(9, 50)
    want = step(t)
    for fn in (torch.compile(chain, backend="eager"), lambda *a: checkpoint(chain, *a, use_reentrant=False)):
        assert all(torch.equal(p, q) for p, q in zip(step(t, fn), want))


@pytest.mark.parametrize("checkpointing", [False, True])
@pytest.mark.parametrize("autocast", [False, True])
def test_student_of_a_quantised_teacher(checkpointing, autocast):
    """A teacher in 8 bits answers under inference_mode; the student's step runs and fills its gradients."""
    torch.manual_seed(5)
    kw = dict(vocab_size=160, d_model=128, n_layers=2, n_heads=2, n_min=4, n_max=16, k_lmk=4, max_seq_len=64, norm="layer")
    teacher = dsalt.DSALTLMHeadModel(**kw).to(DEV, BF).eval()
    student = dsalt.DSALTLMHeadModel(**kw).to(DEV, FP if autocast else BF).train()
    ids = torch.randint(0, 160, (1, 40), device=DEV)
    with torch.inference_mode():
        z, top = teacher.quantize_fp8()(ids)["logits"].topk(8)
    with torch.autocast("cuda", BF, enabled=autocast):
        out = student(ids, teacher_logits=z, teacher_ids=top, temperature=2.0, labels=ids, label_weight=0.2,
                      gradient_checkpointing=checkpointing)
    out["loss"].backward()
    for n in ("embed_tokens", "final_norm", "lm_head"):
        assert all(p.grad is not None and p.grad.isfinite().all() for p in getattr(student, n).parameters()), n
