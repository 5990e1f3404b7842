"""distill_loss (one pass over the logits forward, one backward) against float64 autograd."""
import pytest
import torch

from dsalt import DsaltError
from dsalt.kernels import distill_loss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def inputs(lead, V, K, dtype=FP, t_dtype=FP, labels=True, seed=0, ints=torch.int64, holes=True):
    g = torch.Generator(device=DEV).manual_seed(seed + V)
    s = (torch.randn(*lead, V, device=DEV, generator=g) * 3).to(dtype)
    z = (torch.randn(*lead, K, device=DEV, generator=g) * 2 + 4).to(t_dtype)
    ids = torch.rand(*lead, V, device=DEV, generator=g).topk(min(K, V), -1).indices
    ids = torch.cat([ids, torch.full((*lead, K - ids.shape[-1]), -1, device=DEV)], -1)
    if holes:
        gone = torch.rand(*lead, K, device=DEV, generator=g)
        ids = torch.where(gone < 0.1, -1, torch.where(gone < 0.15, V + 5, ids))
        z = torch.where(gone > 0.95, float("-inf"), z)
    y = None
    if labels:
        y = torch.randint(0, V, lead, device=DEV, generator=g)
        if lead[0] > 2:
            y[::3] = ids[::3, ..., 0].clamp(0, V - 1)  # a label that is also a slot
            y[1] = -100
        y = y.to(ints)
    return s, z, ids.to(ints), y


def reference(s, z, ids, y, tau, lam, reduction="mean", up=None):
    """Loss and gradient in float64, row by row from the definition."""
    s = s.detach().double().reshape(-1, s.shape[-1]).requires_grad_()
    z, ids = z.double().reshape(s.shape[0], -1), ids.reshape(s.shape[0], -1)
    rows, counted = [], 0
    for r in range(s.shape[0]):
        if y is not None:
            label = int(y.reshape(-1)[r])
            if not 0 <= label < s.shape[1]:
                rows.append(s.new_zeros(()))
                continue
        counted += 1
        on = (ids[r] >= 0) & (ids[r] < s.shape[1]) & (z[r] > float("-inf"))
        loss = s.new_zeros(())
        if bool(on.any()) and lam < 1:
            log_p = torch.log_softmax(z[r][on] / tau, 0)
            log_q = torch.log_softmax(s[r] / tau, 0)[ids[r][on].long()]
            loss = loss + (1 - lam) * tau ** 2 * (log_p.exp() * (log_p - log_q)).sum()
        if lam:
            loss = loss - lam * torch.log_softmax(s[r], 0)[label]
        rows.append(loss)
    rows = torch.stack(rows) if rows else s.sum(-1)
    loss = rows if reduction == "none" else rows.sum() / (max(counted, 1) if reduction == "mean" else 1)
    g = None
    if loss.requires_grad:
        g, = torch.autograd.grad(loss, s, torch.ones_like(loss) if up is None else up.double().reshape(loss.shape))
    return loss.detach(), g, max(counted, 1) if reduction == "mean" else 1


def compare(s, z, ids, y, tau=1.0, lam=0.0, reduction="mean", up=None):
    leaf = s.detach().requires_grad_()
    kw = dict(temperature=tau, label_weight=lam, reduction=reduction)
    loss = distill_loss(leaf, z, ids, y, **kw)
    with torch.no_grad():
        assert torch.equal(distill_loss(s, z, ids, y, **kw), loss)
    g, = torch.autograd.grad(loss, leaf, torch.ones_like(loss) if up is None else up)
    want, w_g, n = reference(s, z, ids, y, tau, lam, reduction, up)
    assert loss.dtype == FP and g.dtype == s.dtype and g.shape == s.shape
    # Exponents are differences of logits of up to 40 in units of 1 / tau, each off by 2^-24 of them, from
    # four roundings; sums of V terms run in trees and lanes of at most V / 64 terms a lane, and the losses
    # of rows are summed alike: 2^-16 of the magnitudes (tau^2 times a log of up to 60) covers them.
    scale = max(tau * tau, 1.0) * 60 / min(tau, 1.0)
    assert bool(((loss.double() - want.reshape(loss.shape)).abs() <= 2.0 ** -16 * scale * (1 if reduction != "sum" else s[..., 0].numel())).all()), \
        (loss, want)
    if w_g is None:
        assert not g.any()
        return loss, g
    # the gradient's terms are probabilities (of relative error 2^-18 as above) times tau and the upstream
    umax = 1.0 if up is None else float(up.abs().max())
    tol = torch.finfo(s.dtype).eps / 2 * w_g.abs() + 2.0 ** -17 * max(tau, 1.0) * umax / n + (2.0 ** -25 if s.dtype == HF else 0.0)
    err = (g.double().reshape(w_g.shape) - w_g).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    return loss, g


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 63, 64, 65, 500, 2047, 2048, 2049, 4100, 32000, 50257])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_vocabularies(V, dtype):
    compare(*inputs((7,), V, 5, dtype), tau=1.5, lam=0.3)


@pytest.mark.parametrize("tau,lam,labels", [(1.0, 0.0, False), (1.0, 0.0, True), (1.0, 0.4, True), (2.0, 0.0, False), (2.0, 0.5, True),
                                            (0.5, 0.25, True), (3.7, 1.0, True), (1.0, 1.0, True)])
@pytest.mark.parametrize("V", [300, 5003])
def test_weights(tau, lam, labels, V):
    compare(*inputs((9,), V, 8, labels=labels), tau=tau, lam=lam)


@pytest.mark.parametrize("dtype", [FP, BF, HF])
@pytest.mark.parametrize("t_dtype", [FP, BF, HF])
@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_types(dtype, t_dtype, ints):
    compare(*inputs((6,), 777, 12, dtype, t_dtype, ints=ints), tau=2.0, lam=0.5)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 16, 17, 63, 130, 600])
def test_rows(rows):
    """One row to more than slices are made for, of long rows and of short ones."""
    for V in (9001, 40):
        compare(*inputs((rows,), V, 6, BF), tau=2.0, lam=0.5)


@pytest.mark.parametrize("K", [1, 2, 63, 64, 65, 200, 1024])
def test_slots(K):
    compare(*inputs((5,), 3001, K), tau=1.3, lam=0.2)
    compare(*inputs((5,), 1025, K), tau=1.3, lam=0.2)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("labels", [False, True])
def test_reductions(reduction, labels):
    s, z, ids, y = inputs((3, 4), 130, 6, labels=labels)
    up = torch.randn(3, 4, device=DEV) if reduction == "none" else torch.tensor(-2.5, device=DEV)
    loss, _ = compare(s, z, ids, y, tau=2.0, lam=0.5 if labels else 0.0, reduction=reduction, up=up)
    assert loss.shape == ((3, 4) if reduction == "none" else ())


def test_rows_without_teacher_or_label():
    """No slots (ids -1, logits -inf): only the labels' term; no label: nothing, whatever the row holds."""
    s, z, ids, y = inputs((8,), 90, 4, holes=False)
    ids[2] = -1
    z[3] = float("-inf")
    y[5], y[6] = 90, -7
    compare(s, z, ids, y, tau=2.0, lam=0.5)
    s[5] = float("nan")
    s[1] = float("inf")
    loss, g = compare(s, z, ids, y, tau=2.0, lam=0.5)
    assert bool(torch.isfinite(loss)) and not g[5].any() and not g[1].any()
    loss, g = compare(s[2:3], z[2:3], ids[2:3], None)
    assert loss == 0 and not g.any()
    loss, g = compare(s, z, ids, torch.full_like(y, -100), tau=2.0, lam=0.5)
    assert loss == 0 and not g.any()


def test_masked_logits():
    """A padded vocabulary: logits of -inf or the type's lowest value have no probability and no gradient."""
    for low in (float("-inf"), torch.finfo(BF).min):
        for V, cut in ((600, 500), (40000, 33333)):
            s, z, ids, y = inputs((4,), V, 6, BF, holes=False)
            ids, y = ids % cut, y % cut
            s[:, cut:] = low
            s[:, :3] = low
            ids, y = ids.clamp(min=3), y.clamp(min=3)
            y[1] = 4
            _, g = compare(s, z, ids, y, tau=2.0, lam=0.5)
            assert not g[:, cut:].any() and bool(torch.isfinite(g).all())


def test_teacher_where_the_student_cannot():
    """A student's -inf at a teacher's token is an infinite loss with a finite gradient."""
    s, z, ids, _ = inputs((3,), 50, 4, labels=False, holes=False)
    s[1, ids[1, 2]] = float("-inf")
    leaf = s.requires_grad_()
    rows = distill_loss(leaf, z, ids, reduction="none")
    g, = torch.autograd.grad(rows.sum(), leaf)
    assert rows[1] == float("inf") and bool(torch.isfinite(rows[[0, 2]]).all()) and bool(torch.isfinite(g).all())


@pytest.mark.parametrize("where", ["student", "teacher"])
def test_nan_stays_in_its_row(where):
    s, z, ids, y = inputs((5,), 3000, 4, holes=False)
    (s if where == "student" else z)[2, 1] = float("nan")
    leaf = s.requires_grad_()
    rows = distill_loss(leaf, z, ids, y, label_weight=0.5, reduction="none")
    g, = torch.autograd.grad(rows.sum(), leaf)
    assert bool(torch.isnan(rows[2])) and bool(torch.isfinite(rows[[0, 1, 3, 4]]).all())
    assert bool(torch.isnan(g[2]).any()) and bool(torch.isfinite(g[[0, 1, 3, 4]]).all())


def test_ids_that_repeat():
    """Slots of one id add up, in the loss and in the gradient, the same bits on every call."""
    s, z, ids, y = inputs((6,), 4000, 40, holes=False)
    ids[:, 20:] = ids[:, :20]
    ids[0] = ids[0, 0]
    y[0], y[2] = ids[0, 0], ids[2, 3]
    _, g = compare(s, z, ids, y, tau=2.0, lam=0.5)
    for _ in range(5):
        assert torch.equal(compare(s, z, ids, y, tau=2.0, lam=0.5)[1], g)


def test_strides():
    """Rows of a padded vocabulary, expanded teachers, transposed ids, misaligned bases: the contiguous bits."""
    s, z, ids, y = inputs((6,), 1001, 6, BF)
    want = distill_loss(s.clone().requires_grad_(), z, ids, y, temperature=2.0, label_weight=0.5)
    wide = torch.zeros(6, 1030, device=DEV, dtype=BF)
    wide[:, 5:1006] = s
    for S in (wide[:, 5:1006], s.t().contiguous().t()):
        for T, I in ((z, ids), (z.t().contiguous().t(), ids.t().contiguous().t())):
            loss, _ = compare(S, T, I, y, tau=2.0, lam=0.5)
            assert abs(float(loss - want)) < 1e-4
    compare(s, z[:1].expand(6, 6), ids[:1].expand(6, 6), y.view(6, 1).expand(6, 2)[:, 1], tau=2.0, lam=0.5)


def test_extreme_logits():
    """Logits of thousands, and temperatures far from 1."""
    s, z, ids, y = inputs((4,), 700, 5, holes=False)
    for S in (s * 1000, s + 60000.0):
        loss, g = distill_loss(S, z, ids, y, label_weight=0.5), None
        want, _, _ = reference(S, z, ids, y, 1.0, 0.5)
        assert abs(float(loss) - float(want)) <= 2.0 ** -20 * float(S.abs().max()) * 4
    compare(s, z, ids, y, tau=50.0, lam=0.5)


def test_no_rows():
    s, z, ids, y = inputs((0,), 20, 3)
    assert distill_loss(s, z, ids, y) == 0 and distill_loss(s, z, ids, y, reduction="none").shape == (0,)
    leaf = s.requires_grad_()
    g, = torch.autograd.grad(distill_loss(leaf, z, ids, y, reduction="sum"), leaf)
    assert g.shape == (0, 20)


def test_differences_and_second_order():
    s, z, ids, y = inputs((3,), 30, 4, holes=False)
    leaf = s.clone().requires_grad_()
    kw = dict(temperature=2.0, label_weight=0.5)
    g, = torch.autograd.grad(distill_loss(leaf, z, ids, y, **kw), leaf, create_graph=True)
    for i, j in ((0, 0), (0, int(ids[0, 0])), (2, int(y[2]))):
        f = []
        for step in (1e-5, -1e-5):
            t = s.double().clone()
            t[i, j] += step
            f.append(reference(t, z, ids, y, 2.0, 0.5)[0])
        assert abs(float((f[0] - f[1]) / 2e-5) - float(g[i, j])) < 1e-5  # fp32 arithmetic on values of order 1
    g2, = torch.autograd.grad(g.square().sum(), leaf)
    ref = s.double().requires_grad_()
    on = (y >= 0)
    log_p = torch.log_softmax(z.double() / 2, -1)
    rows = 0.5 * 4 * (log_p.exp() * (log_p - torch.log_softmax(ref / 2, -1).gather(1, ids))).sum(-1)
    rows = rows - 0.5 * torch.log_softmax(ref, -1).gather(1, y.clamp(min=0)[:, None])[:, 0]
    w, = torch.autograd.grad((rows * on).sum() / on.sum(), ref, create_graph=True)
    w2, = torch.autograd.grad(w.square().sum(), ref)
    assert float((g2 - w2).norm() / w2.norm()) < 1e-4


def test_captured_and_replayed():
    s, z, ids, y = inputs((40,), 6000, 7, BF)
    leaf = s.clone().requires_grad_()

    def step():
        loss = distill_loss(leaf, z, ids, y, temperature=2.0, label_weight=0.5)
        return loss.detach(), *torch.autograd.grad(loss, leaf)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        new = inputs((40,), 6000, 7, BF, seed=20 + k)
        with torch.no_grad():
            for a, b in zip((leaf, z, ids, y), new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


def test_offsets_past_32_bits():
    """Rows whose bytes lie past 4 GiB, forward and backward."""
    V, rows = 131072, 16384 + 3
    s = torch.zeros(rows, V, device=DEV, dtype=BF)
    small, z, ids, y = inputs((3,), V, 4, BF, holes=False)
    y[1] = 17
    s[-3:] = small
    Z, I = torch.zeros(rows, 4, device=DEV), torch.full((rows, 4), -1, device=DEV)
    Z[-3:], I[-3:] = z, ids
    Y = torch.full((rows,), -100, device=DEV)
    Y[-3:] = y
    a, b = s.requires_grad_(), small.clone().requires_grad_()
    la, lb = (distill_loss(*t, temperature=2.0, label_weight=0.5) for t in ((a, Z, I, Y), (b, z, ids, y)))
    ga, = torch.autograd.grad(la, a)
    gb, = torch.autograd.grad(lb, b)
    assert abs(float(la - lb)) <= 2.0 ** -18 * float(lb)
    # rows that are cut otherwise sum in another order: a bf16 step of the largest
    assert float((ga[-3:].float() - gb.float()).abs().max()) <= 2.0 ** -8 * float(gb.abs().max()) and not ga[:-3].any()


def test_transforms_and_autocast():
    s, z, ids, y = inputs((5,), 60, 4)
    want = distill_loss(s, z, ids, y, label_weight=0.5, reduction="none")
    got = torch.vmap(lambda *t: distill_loss(*t, label_weight=0.5, reduction="none"))(s, z, ids, y)
    torch.testing.assert_close(got, want)
    with torch.autocast("cuda", dtype=BF):
        assert torch.equal(distill_loss(s, z, ids, y, label_weight=0.5, reduction="none"), want)
    torch.testing.assert_close(torch.compile(lambda *t: distill_loss(*t, label_weight=0.5, reduction="none") + 1)(s, z, ids, y), want + 1)


def test_refusals():
    s, z, ids, y = inputs((4,), 20, 3)
    for call in (lambda: distill_loss(s.double(), z, ids), lambda: distill_loss(s, z, ids[:, :2]), lambda: distill_loss(s, z[:3], ids[:3]),
                 lambda: distill_loss(s, z, ids.float()), lambda: distill_loss(s, z, ids, y[:2]), lambda: distill_loss(s, z.cpu(), ids),
                 lambda: distill_loss(s, z[:, :0], ids[:, :0]), lambda: distill_loss(s[:, :0], z, ids),
                 lambda: distill_loss(s, z.repeat(1, 400), ids.repeat(1, 400)), lambda: distill_loss(s, z, ids, y.bool())):
        with pytest.raises(DsaltError):
            call()
    for kw in (dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(label_weight=-0.1),
               dict(label_weight=1.5), dict(reduction="max")):
        with pytest.raises(ValueError):
            distill_loss(s, z, ids, y, **kw)
    with pytest.raises(ValueError, match="labels"):
        distill_loss(s, z, ids, label_weight=0.5)


@pytest.mark.parametrize("V", [100, 5000])
def test_rows_of_the_lowest_value(V):
    """A mask of the type's lowest value that leaves nothing: all logits are equal, the softmax is 1 / V."""
    s, z, ids, y = inputs((4,), V, 4, FP, holes=False)
    s[:] = torch.finfo(FP).min
    compare(s, z, ids, y, tau=2.0, lam=0.5)


@pytest.mark.parametrize("V", [1, 100, 4096, 4097, 8200, 32000, 65536, 65537, 70001])
@pytest.mark.parametrize("tau,lam", [(1.0, 0.0), (2.0, 0.5), (3.0, 0.5), (1.0, 1.0)])
@pytest.mark.parametrize("dtype", [FP, BF])
def test_lone_row(V, tau, lam, dtype):
    """One row, which one workgroup ends, or slices do: every reduction, a row that starts off 16 bytes."""
    s, z, ids, y = inputs((1,), V, 66, dtype)
    for reduction in ("mean", "sum", "none"):
        up = torch.tensor([1.7] if reduction == "none" else 1.7, device=DEV)
        compare(s, z, ids, y, tau=tau, lam=lam, reduction=reduction, up=up)
    wide = torch.zeros(1, V + 3, device=DEV, dtype=dtype)
    wide[:, 3:] = s
    want = distill_loss(s, z, ids, y, temperature=tau, label_weight=lam)
    got = distill_loss(wide[:, 3:], z, ids, y, temperature=tau, label_weight=lam)
    # the same terms in another order: 2^-16 of a log of up to 60, as above
    assert abs(got - want) <= 2.0 ** -16 * 60 * max(tau * tau, 1.0)


@pytest.mark.parametrize("V", [100, 32000, 70001])
def test_lone_row_that_does_not_count(V):
    s, z, ids, y = inputs((1,), V, 5)
    for labels in (torch.full_like(y, -100), torch.full_like(y, V)):
        loss, g = compare(s, z, ids, labels, tau=2.0, lam=0.5)
        assert loss == 0 and not g.any()
    loss, g = compare(s, z, torch.full_like(ids, -1), None)
    assert loss == 0 and not g.any()
    s[0, 3] = float("nan")
    leaf = s.detach().requires_grad_()
    loss = distill_loss(leaf, z, ids, y, label_weight=0.5)
    g, = torch.autograd.grad(loss, leaf)
    assert loss.isnan() and g.isnan().all()
