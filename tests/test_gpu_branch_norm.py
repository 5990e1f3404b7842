"""branch_norm (dropout, norm, gate and scaled residual sum of a branch, and the next norm, one
pass forward and one backward) against float64 autograd."""
import itertools

import numpy as np
import pytest
import torch

from dsalt import _hip
from dsalt.kernels import _block_train, branch_norm, counter_dropout
from dsalt.kernels.RMSENorm import RMSENorm
from philox_reference import keep_mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NAMES = ("x", "h", "weight", "post_weight", "gate")


def inputs(lead, d, xd, hd, od, post=True, pre=True, gate="channel", wd=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + d)
    wd = xd if wd is None else wd

    def rnd(dt, *s, std=1.0, mean=0.0):
        return (torch.randn(*s, device=DEV, generator=g) * std + mean).to(dt)

    t = {"x": rnd(xd, *lead, d, std=2.0), "h": rnd(hd, *lead, d), "weight": rnd(wd, d, std=0.25, mean=1.0) if pre else None,
         "post_weight": rnd(wd, d, std=0.25, mean=1.0) if post else None,
         "gate": {"none": None, "channel": rnd(wd, d, std=0.5, mean=0.5), "token": rnd(wd, *lead, 1)}[gate]}
    return t, rnd(xd, *lead, d), rnd(od, *lead, d)


def reference(t, p, seed, offset, rs, eps, dz, dy):
    w = {n: v.detach().double().requires_grad_() for n, v in t.items() if v is not None}
    n = w["h"]
    th = _hip.keep_threshold(p)
    if th < 65536:
        keep = torch.from_numpy(keep_mask(n.numel(), p, seed, offset)).view(n.shape).to(n.device)
        n = torch.where(keep, n * (65536.0 / max(th, 1)), 0.0)
    if "post_weight" in w:
        n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + eps) * w["post_weight"]
    z = rs * w["x"] + (w["gate"] * n if "gate" in w else n)
    outs, ups = [z], [dz]
    if "weight" in w:
        outs.append(z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps) * w["weight"])
        ups.append(dy)
    pairs = [(o, u.double()) for o, u in zip(outs, ups) if u is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(w.values()), [u for _, u in pairs], allow_unused=True)
    return [o.detach() for o in outs], dict(zip(w, grads))


def close(got, want, dtype, what, rows_summed=1):
    """One rounding to the dtype, plus fp32 arithmetic: a row's sums of d <= 8192 terms and the
    column sums stay within 2^-18 of the largest magnitudes they are formed from (2^-24 a
    term's rounding; sums run over at most 64 terms a lane, then in trees), which the row's
    or column's largest value stands for."""
    assert got.dtype == dtype and got.shape == want.shape, what
    err = (got.double() - want).abs()
    scale = want.abs().max() * rows_summed ** 0.5
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -18 * scale + (2.0 ** -25 if dtype == HF else 0.0)
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


def run(t, dz, dy, **kw):
    leaves = {n: v.detach().clone().requires_grad_() for n, v in t.items() if v is not None}
    outs = [o for o in branch_norm(leaves["x"], leaves["h"], leaves.get("weight"), post_weight=leaves.get("post_weight"),
                                   gate=leaves.get("gate"), **kw) if o is not None]
    pairs = [(o, u) for o, u in zip(outs, (dz, dy)) if u is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [u for _, u in pairs], allow_unused=True)
    return [o.detach() for o in outs], dict(zip(leaves, grads))


def compare(t, dz, dy, rs=0.75, p=0.2, seed=77, offset=5, eps=1e-6, od=None):
    kw = dict(residual_scale=rs, p=p, seed=seed, offset=offset, eps=eps, out_dtype=od)
    outs, grads = run(t, dz, dy, **kw)
    w_outs, w_grads = reference(t, p, seed, offset, rs, eps, dz, dy)
    for n, a, b in zip(("x_out", "y"), outs, w_outs):
        close(a, b, t["x"].dtype if n == "x_out" or od is None else od, n)
    rows = t["x"].numel() // t["x"].shape[-1]
    for n, g in grads.items():
        if w_grads[n] is None:
            assert g is None or not bool(g.any()), n
            continue
        close(g, w_grads[n], t[n].dtype, "d" + n, 1 if n in ("x", "h") else max(1, rows / 64))
    with torch.no_grad():
        bare = branch_norm(t["x"], t["h"], t["weight"], post_weight=t["post_weight"], gate=t["gate"], **kw)
    assert all(torch.equal(a, b) for a, b in zip(outs, bare))
    return outs, grads


@pytest.mark.parametrize("xd,hd,od,wd", [(FP, BF, BF, FP), (FP, HF, FP, FP), (FP, FP, FP, FP), (FP, FP, HF, FP), (FP, BF, HF, FP),
                                         (BF, BF, BF, BF), (BF, BF, BF, FP), (HF, HF, HF, HF), (HF, HF, HF, FP)])
@pytest.mark.parametrize("rows,d", [(1, 8), (3, 512), (5, 520), (3101, 1024), (7, 1032), (2, 2056), (1601, 4096), (3, 4104), (513, 8192)])
def test_types_and_sizes(rows, d, xd, hd, od, wd):
    print(f"branch_norm {rows}x{d} {xd} {hd} {od} {wd}", flush=True)
    t, dz, dy = inputs((rows,), d, xd, hd, od, wd=wd)
    compare(t, dz, dy, od=od)


@pytest.mark.parametrize("post,pre,gate,p", list(itertools.product((True, False), (True, False), ("none", "channel", "token"),
                                                                   (0.0, 0.3))))
def test_forms(post, pre, gate, p):
    for rows, d in ((37, 200), (9, 1536)):
        print(f"branch_norm form post={post} pre={pre} gate={gate} p={p} {rows}x{d}", flush=True)
        t, dz, dy = inputs((rows,), d, FP, BF, BF, post, pre, gate)
        compare(t, dz, dy if pre else None, p=p, od=BF)
        compare(t, dz, None, p=p, od=BF)  # only the stream's gradient
        if pre:
            compare(t, None, dy, p=p, od=BF)  # only the norm's


def test_leading_dimensions_strides_and_alignment():
    t, dz, dy = inputs((3, 4), 136, BF, BF, BF, gate="token")
    want = run(t, dz, dy, p=0.2, seed=3)
    compare(t, dz, dy)
    for n in ("x", "h"):
        off = torch.zeros(t[n].numel() + 3, device=DEV, dtype=BF)[3:].view(3, 4, 136)
        off.copy_(t[n])
        wide = torch.zeros(3, 4, 272, device=DEV, dtype=BF)[..., ::2]
        wide.copy_(t[n])
        for v in (off, wide):
            got = run({**t, n: v}, dz.transpose(0, 1).contiguous().transpose(0, 1), dy.expand(3, 4, 136), p=0.2, seed=3)
            assert all(torch.equal(a, b) for a, b in zip(got[0], want[0]))
            assert all(torch.equal(got[1][k], want[1][k]) for k in want[1])


def test_offsets_past_32_bits():
    """More than 2^31 elements and 2^32 bytes a tensor: rows at both ends equal those of a call of
    their own."""
    rows, d = 262207, 8192
    print(f"branch_norm {rows}x{d}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(4)
    x, h, dz, dy = (torch.randn(rows, d, device=DEV, generator=g, dtype=BF) for _ in range(4))
    w, post, gate = (torch.rand(s, device=DEV, generator=g) for s in ((d,), (d,), (rows, 1)))

    def call(at):
        t = {"x": x[at], "h": h[at], "weight": w, "post_weight": post, "gate": gate[at]}
        outs, grads = run(t, dz[at], dy[at], residual_scale=0.75)
        return [*outs, grads["x"], grads["h"], grads["gate"]]

    whole = call(slice(None))
    for at in (slice(0, 5), slice(rows - 70, rows)):
        for n, a, b in zip(("x_out", "y", "dx", "dh", "dgate"), whole, call(at)):
            assert torch.equal(a[at], b), (n, at)


def test_no_rows():
    t, dz, dy = inputs((0,), 64, FP, BF, BF)
    outs, grads = run(t, dz, dy, out_dtype=BF)
    assert outs[0].shape == (0, 64) and outs[1].dtype == BF
    assert all(not bool(grads[n].any()) for n in ("weight", "post_weight", "gate"))


def test_rows_of_zeros_and_dropped_rows():
    """A branch that is all zero or all dropped leaves the scaled residual; its norm divides by
    sqrt(eps), never by 0."""
    t, dz, dy = inputs((6,), 72, FP, FP, FP)
    t["h"][2] = 0
    t["x"][4] = 0
    compare(t, dz, dy, p=0.0)
    outs, grads = run(t, dz, dy, p=1.0, seed=1, residual_scale=0.5)
    assert torch.equal(outs[0], 0.5 * t["x"]) and not bool(grads["h"].any())


def test_nan_stays_in_its_row():
    t, dz, dy = inputs((9,), 1536, BF, BF, BF)
    outs, grads = run(t, dz, dy, p=0.1, seed=2)
    t2 = {**t, "h": t["h"].clone()}
    t2["h"][3] = float("nan")
    o2, g2 = run(t2, dz, dy, p=0.1, seed=2)
    keep = [r for r in range(9) if r != 3]
    for a, b in (*zip(o2, outs), (g2["x"], grads["x"]), (g2["h"], grads["h"])):
        assert torch.equal(a[keep], b[keep]) and bool(a[3].isnan().any())


def test_nan_without_a_norm_gradient():
    """Only x_out's gradient: it passes whatever the stream holds."""
    t, dz, dy = inputs((5,), 200, FP, FP, FP, post=False, gate="none")
    t["x"][1] = float("nan")
    t["x"][2, 3] = float("inf")
    _, grads = run(t, dz, None, residual_scale=0.5)
    assert torch.equal(grads["x"], 0.5 * dz) and torch.equal(grads["h"], dz)


def test_equals_the_parts():
    """Dropout alone in the branch, no gate and scale 1: x_out has the bits of counter_dropout and
    the add; without dropout either, those of the block's add + norm pass."""
    t, _, _ = inputs((50,), 256, FP, FP, FP, post=False, gate="none")
    x, h = t["x"], t["h"]
    x_out, _ = branch_norm(x, h, p=0.3, seed=4, offset=2)
    assert torch.equal(x_out, x + counter_dropout(h, 0.3, 4, 2))
    norm = RMSENorm(256).to(DEV)
    s, y = _block_train.add_norm(x, h, norm)
    got = branch_norm(x, h, norm.weight, eps=norm.eps)
    assert torch.equal(got[0], s)
    close(got[1].detach(), y.detach().double(), FP, "y")


def test_second_order():
    t, dz, dy = inputs((5,), 64, FP, FP, FP)
    leaves = [t[n].detach().clone().requires_grad_() for n in NAMES]
    wide = [v.detach().double().requires_grad_() for v in leaves]
    out = []
    for ls, up in ((leaves, (dz, dy)), (wide, (dz.double(), dy.double()))):
        if ls is leaves:
            x_out, y = branch_norm(ls[0], ls[1], ls[2], post_weight=ls[3], gate=ls[4], residual_scale=0.5)
        else:
            nrm = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w
            x_out = 0.5 * ls[0] + ls[4] * nrm(ls[1], ls[3])
            y = nrm(x_out, ls[2])
        g = torch.autograd.grad((x_out, y), ls, up, create_graph=True)
        out.append(torch.autograd.grad(sum(v.square().sum() for v in g), ls))
    for a, b in zip(*out):
        # some tens of fp32 roundings in a row, over sums of at most 320 terms
        assert float((a.double() - b).norm()) <= 2.0 ** -17 * float(b.norm())


def test_changed_in_place_is_refused():
    for i, n in enumerate(("x", "h", "post_weight")):
        t, dz, dy = inputs((4,), 64, FP, FP, FP)
        ls = {k: v.detach().clone().requires_grad_() for k, v in t.items()}
        x_out, y = branch_norm(ls["x"], ls["h"], ls["weight"], post_weight=ls["post_weight"], gate=ls["gate"])
        with torch.no_grad():
            ls[n].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad((x_out, y), list(ls.values()), (dz, dy))
    x_out.add_(1)  # the stream may be modified in place


@pytest.mark.parametrize("rows,d", [(40, 256), (40, 2048)])
def test_streams_and_graph(rows, d):
    t, dz, dy = inputs((rows,), d, FP, BF, BF)
    seed = torch.tensor([12], device=DEV)
    leaves = {n: v.detach().clone().requires_grad_() for n, v in t.items()}

    def step():
        x_out, y = branch_norm(leaves["x"], leaves["h"], leaves["weight"], post_weight=leaves["post_weight"],
                               gate=leaves["gate"], residual_scale=0.75, p=0.2, seed=seed, offset=5, out_dtype=BF)
        return x_out.detach(), y.detach(), *torch.autograd.grad((x_out, y), list(leaves.values()), (dz, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    outs, grads = run(t, dz, dy, residual_scale=0.75, p=0.2, seed=12, offset=5, out_dtype=BF)
    assert all(torch.equal(a, b) for a, b in zip(other, (*outs, *grads.values())))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for s in (5, -9, 2 ** 60):
        new, nz, ny = inputs((rows,), d, FP, BF, BF, seed=abs(s) % 100)
        with torch.no_grad():
            for n in leaves:
                leaves[n].copy_(new[n])
            dz.copy_(nz)
            dy.copy_(ny)
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        outs, grads = run(new, nz, ny, residual_scale=0.75, p=0.2, seed=s, offset=5, out_dtype=BF)
        assert all(torch.equal(a, b) for a, b in zip(got, (*outs, *grads.values()))), s


def test_partial_gradients():
    t, dz, dy = inputs((70,), 136, FP, BF, BF)
    _, want = run(t, dz, dy, p=0.2, seed=1, out_dtype=BF)
    for need in range(1, 32):
        ls = {n: t[n].detach().clone().requires_grad_(bool(need >> i & 1)) for i, n in enumerate(NAMES)}
        x_out, y = branch_norm(ls["x"], ls["h"], ls["weight"], post_weight=ls["post_weight"], gate=ls["gate"], p=0.2, seed=1,
                               out_dtype=BF)
        outs = [(o, u) for o, u in ((x_out, dz), (y, dy)) if o.requires_grad]
        live = [n for n in NAMES if ls[n].requires_grad]
        for n, g in zip(live, torch.autograd.grad([o for o, _ in outs], [ls[n] for n in live], [u for _, u in outs])):
            assert torch.equal(g, want[n]), (need, n)


def test_refusals_on_gpu():
    t, _, _ = inputs((4,), 64, BF, BF, BF)
    x, h, w = t["x"], t["h"], t["weight"]
    for args, kw in (((x, h[:, :56]), {}), ((x, h.half()), {}), ((x, h, w.half()), {}), ((x, h, w[:8]), {}),
                     ((x, h, w), {"out_dtype": FP}), ((x, h), {"gate": x}), ((x, h), {"gate": w[:8]}),
                     ((x[:, :12].contiguous(), h[:, :12].contiguous()), {}), ((x.double(), h.double()), {}),
                     ((x, h), {"p": 0.1, "seed": torch.tensor([1])}), ((x, h.cpu()), {}),
                     ((x.new_zeros(2, 8200), x.new_zeros(2, 8200)), {})):
        with pytest.raises(_hip.DsaltError):
            branch_norm(*args, **kw)
    for kw in ({"p": 0.1}, {"p": -1.0}, {"p": 0.1, "seed": 1, "offset": -1}):
        with pytest.raises(ValueError):
            branch_norm(x, h, **kw)


@pytest.mark.parametrize("only", ["x_out", "y"])
def test_second_order_of_one_output(only):
    """A graph of the backward where one output has no gradient: float64's double backward, through
    fp32 operations (2^-18 of the largest value, as close() counts them, twice over)."""
    t, dz, dy = inputs((6,), 64, FP, FP, FP)
    up = dz if only == "x_out" else dy
    res = []
    for dt in (FP, torch.float64):
        w = {n: v.detach().to(dt).requires_grad_() for n, v in t.items()}
        if dt is FP:
            x_out, y = branch_norm(w["x"], w["h"], w["weight"], post_weight=w["post_weight"], gate=w["gate"], residual_scale=0.5)
        else:
            n = w["h"] * torch.rsqrt(w["h"].square().mean(-1, keepdim=True) + 1e-6) * w["post_weight"]
            x_out = 0.5 * w["x"] + w["gate"] * n
            y = x_out * torch.rsqrt(x_out.square().mean(-1, keepdim=True) + 1e-6) * w["weight"]
        first, = torch.autograd.grad(x_out if only == "x_out" else y, w["h"], up.to(dt), create_graph=True)
        res.append(torch.autograd.grad(first.square().sum(), (w["h"], w["post_weight"])))
    for a, b in zip(*res):
        assert bool(((a.double() - b).abs() <= 2.0 ** -17 * b.abs().max()).all())


def test_stream_and_branch_one_tensor():
    """x given as h too: its gradient is the sum of both."""
    t, dz, dy = inputs((5,), 72, BF, BF, BF)
    x = t["x"].clone().requires_grad_()
    outs = branch_norm(x, x, t["weight"], gate=t["gate"])
    got, = torch.autograd.grad(outs, x, (dz, dy))
    two = {n: t["x"].clone().requires_grad_() for n in ("x", "h")}
    parts = torch.autograd.grad(branch_norm(two["x"], two["h"], t["weight"], gate=t["gate"]), (two["x"], two["h"]), (dz, dy))
    assert torch.equal(got, parts[0] + parts[1])


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("d", [8, 1032, 8192])
def test_one_dimensional_stream(gate, d):
    """x [d]: one row, whose token gate is [1]."""
    for xd, hd in ((FP, BF), (HF, HF)):
        print(f"branch_norm [{d}] gate={gate} {xd}", flush=True)
        t, dz, dy = inputs((), d, xd, hd, hd, gate=gate)
        outs, grads = compare(t, dz, dy, od=hd)
        assert outs[0].shape == outs[1].shape == (d,)
        assert gate == "none" or grads["gate"].shape == ((1,) if gate == "token" else (d,))
        two = run({n: v if v is None or n in ("weight", "post_weight") or gate == "channel" and n == "gate" else v[None]
                   for n, v in t.items()}, dz[None], dy[None], residual_scale=0.75, p=0.2, seed=77, offset=5, out_dtype=hd)
        assert all(torch.equal(a, b[0]) for a, b in zip(outs, two[0]))
        assert all(torch.equal(grads[n], two[1][n].view(grads[n].shape)) for n in grads)


@pytest.mark.parametrize("rows", [0, 1, 700])
def test_backward_entry_without_dy(rows):
    """The C entry with d_weight wanted and no gradient of y: zeros, whatever the stream and the buffer
    held; the other results as without d_weight."""
    print(f"branch_norm backward without dy {rows}", flush=True)
    t, dz, _ = inputs((rows,), 136, FP, BF, BF)
    if rows:
        t["x"][0, 3] = float("inf")
    opts = (0.5, 0.0, 0, 1e-6, 1e-6, BF)
    _, _, stats = _hip.branch_norm(*t.values(), opts, None, True)
    want = _hip.branch_norm_bwd(*t.values(), opts, None, stats, dz, None, (True, True, False, True, True))
    ws = torch.empty(max(16, _hip.lib().dsalt_branch_norm_workspace_size(rows, 136)), device=DEV, dtype=torch.uint8)
    got = [torch.full_like(v, 7.0) for v in t.values()]
    _hip._call("dsalt_branch_norm_bwd", _hip._branch_pack(
        *t.values(), opts, None, rstd=stats.data_ptr(), rstd_post=stats.data_ptr() + 4 * rows, dx_out=dz.data_ptr(), dy=0,
        grads=[g.data_ptr() for g in got], ws=(ws.data_ptr(), ws.numel())), dz.device)
    assert not bool(got[2].any())
    for i in (0, 1, 3, 4):
        assert torch.equal(got[i], want[i]), i


class Tagged(torch.Tensor):
    """A tensor subclass with nothing of its own."""


@pytest.mark.parametrize("p", [0.0, 0.2])
def test_transforms_tracing_and_subclasses(p):
    """What an autograd function with a HIP kernel does not know runs as torch's ops: the kernels' values
    within their fp32 roundings."""
    t, dz, dy = inputs((6,), 64, FP, FP, FP, gate="token")
    ts = tuple(t.values())

    def call(x, h, w, post, gate):
        return branch_norm(x, h, w, post_weight=post, gate=gate, residual_scale=0.75, p=p, seed=5, offset=2)

    with torch.no_grad():
        want = call(*ts)
    _, grads = run(t, dz, dy, residual_scale=0.75, p=p, seed=5, offset=2)
    got = torch.func.grad(lambda ts: sum((o * u).sum() for o, u in zip(call(*ts), (dz, dy))))(ts)
    for n, g in zip(NAMES, got):
        close(g, grads[n].double(), FP, n, 6)
    vs = tuple(torch.randn_like(v) for v in ts)
    _, tangents = torch.func.jvp(call, ts, vs)
    # sum of outputs' tangents against the upstream gradients = sum of the gradients against the tangents
    a = sum(float((o.double() * u.double()).sum()) for o, u in zip(tangents, (dz, dy)))
    parts = [(grads[n].double() * v.double()) for n, v in zip(NAMES, vs)]
    assert abs(a - sum(float(q.sum()) for q in parts)) <= 2.0 ** -18 * sum(float(q.abs().sum()) for q in parts)
    for o, w in zip(torch.jit.trace(call, ts)(*ts), want):
        close(o, w.double(), FP, "traced")
    for o, w in zip(call(ts[0].as_subclass(Tagged), *ts[1:]), want):
        assert type(o) is Tagged
        close(o.as_subclass(torch.Tensor), w.double(), FP, "subclass")
    # each example a row [d] with a gate [1]: the mask of one row for all of them
    rows = torch.func.vmap(call, in_dims=(0, 0, None, None, 0))(*ts)
    with torch.no_grad():
        for i in range(6):
            for o, w in zip(rows, call(ts[0][i], ts[1][i], ts[2], ts[3], ts[4][i])):
                close(o[i], w.double(), FP, "vmap")


@pytest.mark.parametrize("gate", ["channel", "token"])
def test_against_differences(gate):
    """The kernels' gradients along random directions against central differences of the float64
    function, which are off by h^2 / 6 of its third derivative (h = 1e-5: below 1e-8 of the size)."""
    t, dz, dy = inputs((7,), 72, FP, FP, FP, gate=gate)
    _, grads = run(t, dz, dy, residual_scale=0.75, p=0.2, seed=3, offset=1)
    keep = torch.from_numpy(keep_mask(7 * 72, 0.2, 3, 1)).view(7, 72).to(DEV).double() * (65536 / _hip.keep_threshold(0.2))

    def value(ts):
        nrm = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w
        x_out = 0.75 * ts["x"] + ts["gate"] * nrm(ts["h"] * keep, ts["post_weight"])
        return float((x_out * dz.double()).sum() + (nrm(x_out, ts["weight"]) * dy.double()).sum())

    g = torch.Generator(device=DEV).manual_seed(1)
    base = {n: v.double() for n, v in t.items()}
    for n in NAMES:
        v = torch.randn(t[n].shape, generator=g, device=DEV, dtype=torch.float64)
        hi, lo = (value({**base, n: base[n] + s * 1e-5 * v}) for s in (1, -1))
        parts = grads[n].double() * v
        # fp32 gradients: a few 2^-24 of each, over sums of up to 504 terms
        assert abs(float(parts.sum()) - (hi - lo) / 2e-5) <= 2.0 ** -18 * float(parts.abs().sum()) + 1e-6, n
