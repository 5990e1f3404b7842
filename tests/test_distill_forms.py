"""The distillation loss on the CPU: its torch form at the edges, and the LM's use of it."""
import ctypes

import pytest
import torch

import dsalt._hip as hip
from dsalt.kernels import distill_loss
from dsalt.kernels.distill import torch_distill_loss
from dsalt.model import DSALTLMHeadModel


def operands(rows=5, V=11, K=3, seed=1):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn(rows, V, generator=g).requires_grad_()
    z, ids = torch.randn(rows, K, generator=g), torch.randint(0, V, (rows, K), generator=g)
    return s, z, ids, torch.randint(0, V, (rows,), generator=g)


@pytest.mark.parametrize("tau", [0.25, 1.0, 2.0])
def test_teacher_of_lowest_values(tau):
    """All slots alike have 1 / K each, also where the logits over the temperature are past fp32's range."""
    s, z, ids, _ = operands()
    z[1], z[2, 1:] = torch.finfo(torch.float32).min, torch.finfo(torch.float32).min
    got = torch_distill_loss(s, z, ids, None, (tau, 0.0, -100, "none"))
    want = torch_distill_loss(s.double(), z.double(), ids, None, (tau, 0.0, -100, "none"))
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("tau", [1e-39, 2.0 ** -64, 2.0 ** 63, 1e20, 1e39])
def test_temperatures_past_fp32(tau):
    """A temperature whose inverse or square fp32 does not hold is refused (the first term would be NaN)."""
    s, z, ids, _ = operands()
    with pytest.raises(ValueError, match="temperature"):
        distill_loss(s, z, ids, temperature=tau)
    args = hip.DistillArgs(rows=4, logits_stride=100, teacher_stride=8, ids_stride=8, ignore_index=-100, vocab=100, k=8, teacher_dtype=2,
                           reduction=1, temperature=2.0, workspace_bytes=1 << 30)
    for i, n in enumerate(("logits", "teacher", "ids", "loss", "workspace")):
        setattr(args, n, 0x10000000 + i * 0x100000)
    for t, code in ((tau, 1), (2.0 ** -63, 0), (2.0 ** 62, 0)):
        args.temperature = t
        assert hip.lib().dsalt_distill_check(ctypes.byref(args), 0) == code


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_do_not_count_have_no_gradient(bad):
    """Whatever they hold, in the loss, its gradient and a graph of the gradient."""
    s, z, ids, y = operands()
    y[1], y[3] = -100, 11
    want, = torch.autograd.grad(torch_distill_loss(s, z, ids, y, (2.0, 0.5, -100, "mean")), s)
    rows = s.detach().clone()
    rows[1, 4], rows[3] = bad, bad
    z[3, 0] = bad
    leaf = rows.requires_grad_()
    loss = torch_distill_loss(leaf, z, ids, y, (2.0, 0.5, -100, "mean"))
    got, = torch.autograd.grad(loss, leaf, create_graph=True)
    assert bool(torch.isfinite(loss)) and torch.equal(got, want) and not got[1].any() and not got[3].any()
    second, = torch.autograd.grad(got.square().sum(), leaf)
    assert bool(torch.isfinite(second).all())


def test_labels_alone():
    """label_weight 1: the cross-entropy, also where the student cannot say what the teacher does."""
    s, z, ids, y = operands()
    ids[:, 0] = (y + 1) % 11
    rows = s.detach().clone()
    rows[torch.arange(5), ids[:, 0]] = float("-inf")
    leaf = rows.requires_grad_()
    got = torch_distill_loss(leaf, z, ids, y, (2.0, 1.0, -100, "mean"))
    want = torch.nn.functional.cross_entropy(leaf, y)
    torch.testing.assert_close(got, want)
    torch.testing.assert_close(*(torch.autograd.grad(t, leaf)[0] for t in (got, want)))


@pytest.mark.parametrize("mask", [-1e30, torch.finfo(torch.float32).min])
def test_student_masks(mask):
    """A mask that leaves nothing of a row is a uniform softmax, and beside other logits has no share."""
    s, z, ids, y = operands()
    rows = s.detach().clone()
    rows[1], rows[2, 5:] = mask, mask
    ids, y = ids % 5, y % 5
    leaf = rows.requires_grad_()
    opts = (0.25, 0.5, -100, "sum")
    got, want = (torch_distill_loss(t, z, ids, y, opts) for t in (leaf, leaf.double()))
    torch.testing.assert_close(got.double(), want)
    torch.testing.assert_close(*(torch.autograd.grad(t, leaf)[0] for t in (got, want)))


def lm():
    """The LM without blocks, whose attention the CPU does not have: embedding, norm, head and loss."""
    torch.manual_seed(3)
    model = DSALTLMHeadModel(vocab_size=11, d_model=32, n_layers=1, n_heads=2, n_min=2, n_max=8, k_lmk=2, max_seq_len=64,
                             lm_head_chunk_size=3)
    model.layers = torch.nn.ModuleList()
    return model


def test_model_checks_as_the_loss_does():
    """On the CPU too: values and operands are refused, no gradient goes to the teacher."""
    _, z, ids, y = operands()
    model, tokens = lm(), torch.arange(5)
    kw = dict(teacher_logits=z.requires_grad_(), teacher_ids=ids)
    for bad in (dict(label_weight=0.5), dict(labels=y, label_weight=1.5), dict(temperature=0.0), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            model(tokens, **kw, **bad)
    for bad in (dict(teacher_ids=ids.float()), dict(teacher_ids=ids[:, :2]), dict(labels=y[:, None].expand(5, 2))):
        with pytest.raises(hip.DsaltError):
            model(tokens, **{**kw, **bad})
    out = model(tokens, labels=y, temperature=2.0, label_weight=0.5, **kw)
    out["loss"].backward()
    assert z.grad is None and bool(model.final_norm.weight.grad.any())
    logits = model(tokens)["logits"]
    want = torch_distill_loss(logits, z.detach(), ids, y, (2.0, 0.5, -100, "mean"))
    torch.testing.assert_close(out["loss"], want)


def test_model_refuses_teachers_of_other_lengths():
    """Rows of a teacher or labels beyond the tokens, also where they end on a chunk of the head."""
    _, z, ids, y = operands(rows=6)
    model, tokens = lm(), torch.arange(3)
    for n in (2, 4, 6):
        with pytest.raises(hip.DsaltError, match="tokens"):
            model(tokens, teacher_logits=z[:n], teacher_ids=ids[:n])
        with pytest.raises(hip.DsaltError, match="tokens"):
            model(tokens, teacher_logits=z[:3], teacher_ids=ids[:3], labels=y[:n])
    assert bool(torch.isfinite(model(tokens, teacher_logits=z[:3], teacher_ids=ids[:3], labels=y[:3])["loss"]))
    assert bool(torch.isfinite(model(tokens[None], teacher_logits=z[None, :3], teacher_ids=ids[None, :3])["loss"]))


def test_model_averages_over_the_rows_that_count():
    """Labels that are no token count for nothing in the model's mean, as in the loss of its logits."""
    _, z, ids, y = operands(rows=7)
    y[1], y[3], y[4] = -100, 11, -3
    model, tokens = lm(), torch.arange(7)
    got = model(tokens, teacher_logits=z, teacher_ids=ids, labels=y, temperature=2.0, label_weight=0.5)["loss"]
    want = torch_distill_loss(model(tokens)["logits"], z, ids, y, (2.0, 0.5, -100, "mean"))
    torch.testing.assert_close(got, want)
