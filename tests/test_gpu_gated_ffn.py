"""gated_ffn (both projections, activation and product in one kernel, with its backward) against
float64, at the edges of its tiles and variants, with error bounds that follow the roundings."""
import pytest
import torch
import torch.nn.functional as F

from dsalt import _hip
from dsalt.kernels import gated_ffn
from dsalt.kernels.gated_ffn import torch_gated_ffn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
ACTS = ("silu", "gelu", "gelu_tanh", "relu")


def inputs(rows, d, f, e, dtype, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * rows + f)

    def rnd(*s, std=1.0):
        return (torch.randn(*s, device=DEV, generator=g) * std).to(dtype)

    return (rnd(rows, d, std=scale), rnd(f, d, std=d ** -0.5), rnd(f, d, std=d ** -0.5), rnd(e, f, std=f ** -0.5),
            rnd(rows, e, std=0.25))


def act64(name, g):
    g = g.detach().requires_grad_()
    v = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu}[name](g)
    s, = torch.autograd.grad(v.sum(), g)
    return v.detach(), s


def reference(x, wg, wu, wd, dy, act, dtype):
    """Float64 results and a bound of each one's error. A rounding to the dtype is off by at most
    half a step (u relative), an fp32 sum of K products by at most (K + 8) 2^-24 of the sum of
    their magnitudes. Carried to first order through the formulas; |act'| <= 1.13, |act''| <= 0.81
    (GELU's, the largest), relu's slope is open where g is within its error of 0. 1 % more
    for the products of errors; fp16's smallest step 2^-25 absolute."""
    u = torch.finfo(dtype).eps / 2
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    gam = lambda k: (k + 8) * 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == HF else 0.0
    g, p = x @ wg.t(), x @ wu.t()
    eg, ep = gam(x.shape[1]) * (x.abs() @ wg.abs().t()), gam(x.shape[1]) * (x.abs() @ wu.abs().t())
    v, s = act64(act, g)
    a = v * p
    ea = u * a.abs() + 1.13 * eg * p.abs() + v.abs() * ep + 2.0 ** -20 * (a.abs() + p.abs() * g.abs()) + tiny
    y = a @ wd.t()
    ey = u * y.abs() + (gam(a.shape[1]) * a.abs() + ea) @ wd.abs().t()
    k = 2.0 ** -12 if dtype == BF else 2.0 ** -16  # g and u as they are kept, in 12 or 16 significant bits
    eg, ep = eg + k * g.abs(), ep + k * p.abs()
    da, eda = dy @ wd, gam(dy.shape[1]) * (dy.abs() @ wd.abs())
    dg, du = da * p * s, da * v
    open_ = (0.81 * eg if act != "relu" else (g.abs() <= eg).double()) + 2.0 ** -20 * (1 + g.abs())
    edg = u * dg.abs() + eda * p.abs() * s.abs() + da.abs() * (ep * s.abs() + p.abs() * open_) + tiny
    edu = u * du.abs() + eda * v.abs() + da.abs() * (1.13 * eg + 2.0 ** -20 * g.abs()) + tiny
    f, T = wg.shape[0], x.shape[0]
    dx = dg @ wg + du @ wu
    edx = u * dx.abs() + (gam(2 * f) * dg.abs() + edg) @ wg.abs() + (gam(2 * f) * du.abs() + edu) @ wu.abs()
    res = {"y": (y, ey), "dx": (dx, edx)}
    for n, m, em in (("dwg", dg, edg), ("dwu", du, edu)):
        w = m.t() @ x
        res[n] = (w, u * w.abs() + (gam(T) * m.abs() + em).t() @ x.abs())
    w = dy.t() @ a
    res["dwd"] = (w, u * w.abs() + dy.abs().t() @ (gam(T) * a.abs() + ea))
    return {n: (w, 1.01 * e + tiny) for n, (w, e) in res.items()}


def check(got, want, dtype, what):
    """Every element within its bound; and all of them together within two half-steps of their norm:
    a rounding's error is spread evenly over a half-step to either side, so its norm is at most
    1 / sqrt(3) of one, and that of two in a chain, which do not line up, sqrt(2 / 3)."""
    ref, bound = want
    assert got.shape == ref.shape and got.dtype == dtype, what
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), (what, float((err / bound.clamp(min=1e-30)).max()))
    if ref.numel() > 64:
        tiny = 2.0 ** -25 * ref.numel() ** 0.5 if dtype == HF else 0.0
        assert float(err.norm()) <= torch.finfo(dtype).eps * float(ref.norm()) + tiny, (what, float(err.norm() / ref.norm()))


def run(x, wg, wu, wd, dy, act):
    leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*leaves, activation=act)
    return dict(zip(("y", "dx", "dwg", "dwu", "dwd"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,d,f,e", [
    (1, 8, 8, 8), (1, 72, 136, 40), (2, 128, 64, 264), (7, 64, 200, 8), (16, 520, 24, 56), (17, 72, 136, 40), (31, 8, 520, 16),
    (33, 64, 64, 64), (64, 264, 104, 128), (65, 56, 128, 72), (127, 128, 384, 120), (128, 192, 256, 128), (129, 200, 264, 136),
    (257, 320, 72, 328), (513, 72, 520, 64), (700, 264, 712, 264)])
def test_against_float64(rows, d, f, e, dtype):
    act = ACTS[(rows + d) % 4]
    print(f"gated_ffn {rows} x {d} -> {f} -> {e} {dtype} {act}", flush=True)
    x, wg, wu, wd, dy = inputs(rows, d, f, e, dtype)
    ref = reference(x, wg, wu, wd, dy, act, dtype)
    got = run(x, wg, wu, wd, dy, act)
    for n in ref:
        check(got[n], ref[n], dtype, (n, act))
    with torch.no_grad():
        check(gated_ffn(x, wg, wu, wd, activation=act), ref["y"], dtype, "y without a graph")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [3, 200])
def test_activations(act, rows):
    print(f"gated_ffn activation {act} {rows}", flush=True)
    x, wg, wu, wd, dy = inputs(rows, 64, 128, 64, BF, seed=5, scale=4.0)
    ref, got = reference(x, wg, wu, wd, dy, act, BF), run(x, wg, wu, wd, dy, act)
    for n in ref:
        check(got[n], ref[n], BF, (n, act))


# sizes that between them take every tile shape, with whole tiles only, with tiles split along k
# besides whole ones and with split ones only, in each of the five products
@pytest.mark.parametrize("rows,d,f", [
    (2049, 512, 1408), (1500, 1024, 2816), (74, 64, 64), (3062, 2344, 64), (8579, 904, 712), (3298, 1952, 2496),
    (846, 520, 3504), (9414, 888, 2672), (3684, 2200, 2440), (7748, 2216, 1504), (2629, 784, 3176), (9228, 472, 848),
    (2378, 1560, 1712), (1383, 1480, 3120), (7376, 1776, 536), (7355, 2264, 1848)])
def test_larger(rows, d, f):
    dtype = (BF, HF)[rows % 2]
    print(f"gated_ffn {rows} x {d} x {f} {dtype}", flush=True)
    x, wg, wu, wd, dy = inputs(rows, d, f, d, dtype)
    ref, got = reference(x, wg, wu, wd, dy, "silu", dtype), run(x, wg, wu, wd, dy, "silu")
    for n in ref:
        check(got[n], ref[n], dtype, n)
    with torch.no_grad():
        check(gated_ffn(x, wg, wu, wd), ref["y"], dtype, "y without a graph")


# and those that the plan's constants, refitted, moved to other shapes or splits
@pytest.mark.parametrize("rows,d,f", [
    (9680, 2024, 400), (8080, 152, 3256), (9408, 200, 3840), (8361, 424, 3576), (1627, 1192, 3728), (3415, 2376, 608),
    (1500, 512, 1408), (3000, 768, 2048), (5452, 656, 3632), (7836, 880, 3168),
    (5407, 1224, 2440), (6843, 280, 3904), (8368, 1040, 2848), (4510, 680, 3544), (4022, 1952, 1864)])
def test_larger_splits(rows, d, f):
    test_larger(rows, d, f)


def test_offsets_past_32_bits():
    """Every buffer of rows and hidden columns is larger than 2^32 bytes: the last rows against
    float64, and the weights' gradients, by their norm, against float64 sums over pieces."""
    rows, d, f, piece = 270001, 64, 8192, 4096
    print(f"gated_ffn {rows} x {d} x {f}", flush=True)
    x, wg, wu, wd, dy = inputs(rows, d, f, d, BF)
    got = run(x, wg, wu, wd, dy, "silu")
    last = reference(x[-257:], wg, wu, wd, dy[-257:], "silu", BF)
    check(got["y"][-257:], last["y"], BF, "y")
    check(got["dx"][-257:], last["dx"], BF, "dx")
    want = {n: 0 for n in ("dwg", "dwu", "dwd")}
    for i in range(0, rows, piece):
        ref = reference(x[i:i + piece], wg, wu, wd, dy[i:i + piece], "silu", BF)
        want = {n: w + ref[n][0] for n, w in want.items()}
    for n, w in want.items():
        assert float((got[n].double() - w).norm()) <= torch.finfo(BF).eps * float(w.norm()), n


def test_against_differences():
    """dx against central differences of the float64 function along random directions: the
    difference is off by h^2 / 6 of its third derivative, the gradient by its roundings."""
    x, wg, wu, wd, dy = inputs(9, 64, 72, 64, HF, seed=3)
    got = run(x, wg, wu, wd, dy, "gelu")
    ts = [t.double() for t in (x, wg, wu, wd)]
    g = torch.Generator(device=DEV).manual_seed(1)
    for i, n in enumerate(("dx", "dwg", "dwu", "dwd")):
        v = torch.randn(ts[i].shape, generator=g, device=DEV, dtype=torch.float64)
        step = 1e-4
        hi, lo = (torch_gated_ffn(*[t + s * step * v if j == i else t for j, t in enumerate(ts)], "gelu") for s in (1, -1))
        want = float(((hi - lo) / (2 * step) * dy.double()).sum())
        have, size = float((got[n].double() * v).sum()), float((got[n].double().abs() * v.abs()).sum())
        assert abs(have - want) <= 4 * 2.0 ** -11 * size + 1e-5, (n, have, want)


def test_strides_views_and_alignment():
    x, wg, wu, wd, dy = inputs(150, 72, 136, 40, BF)
    want = run(x, wg, wu, wd, dy, "silu")
    wide = torch.zeros(150, 3 * 72 + 8, device=DEV, dtype=BF)
    both = torch.cat([wg, wu])  # gate and up as rows of one matrix
    for lo in (0, 72, 144):
        for shift in (0, 8, 3):  # 16-byte aligned columns and ones that are not
            if lo + shift + 72 > wide.shape[1]:
                continue
            xv = wide[:, lo + shift:lo + shift + 72]
            xv.copy_(x)
            got = run_views(xv, both[:136], both[136:], wd.t().contiguous().t(), dy.t().contiguous().t())
            for n, t in got.items():
                assert torch.equal(t, want[n]), (n, lo, shift)
    # leading dimensions, an expanded gradient, a transposed one
    x3 = x.view(3, 50, 72).requires_grad_()
    y = gated_ffn(x3, wg, wu, wd)
    assert y.shape == (3, 50, 40) and torch.equal(y.detach().view(150, 40), want["y"])
    dx, = torch.autograd.grad(y.sum(), x3)
    one = run(x, wg, wu, wd, torch.ones_like(dy), "silu")
    assert torch.equal(dx.view(150, 72), one["dx"])


def run_views(x, wg, wu, wd, dy):
    ts = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    y = gated_ffn(*ts)
    return dict(zip(("y", "dx", "dwg", "dwu", "dwd"), (y.detach(), *torch.autograd.grad(y, ts, dy))))


def test_no_rows():
    x, wg, wu, wd, dy = inputs(0, 64, 72, 40, BF)
    got = run(x, wg, wu, wd, dy, "silu")
    assert got["y"].shape == (0, 40) and got["dx"].shape == (0, 64)
    assert all(bool((got[n] == 0).all()) for n in ("dwg", "dwu", "dwd"))
    assert gated_ffn(x.view(2, 0, 64), wg, wu, wd).shape == (2, 0, 40)


@pytest.mark.parametrize("rows", [5, 140])
def test_nan_and_infinity_stay_in_their_rows(rows):
    x, wg, wu, wd, dy = inputs(rows, 72, 136, 40, BF)
    clean = run(x, wg, wu, wd, dy, "silu")
    x2 = x.clone()
    x2[1] = float("nan")
    x2[3, 5] = float("inf")
    got = run(x2, wg, wu, wd, dy, "silu")
    keep = [r for r in range(rows) if r not in (1, 3)]
    for n in ("y", "dx"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
        assert bool(got[n][1].isnan().all()) and not bool(got[n][3].isfinite().all())
    # a weight's NaN row reaches its own column of the hidden activation only
    wg2 = wg.clone()
    wg2[7] = float("nan")
    wd2 = wd.clone()
    wd2[:, 7] = 0
    got = run(x, wg2, wu, wd2, dy, "silu")
    assert bool(got["dwu"][7].isnan().all()) and bool(got["dwu"][8].isfinite().all())


@pytest.mark.parametrize("need", range(1, 16))
def test_partial_gradients(need):
    """Any set of inputs that require gradients: the same bits as all of them."""
    x, wg, wu, wd, dy = inputs(70, 72, 136, 40, BF)
    want = run(x, wg, wu, wd, dy, "gelu")
    ts = [t.detach().clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, wg, wu, wd))]
    y = gated_ffn(*ts, activation="gelu")
    live = [i for i in range(4) if need >> i & 1]
    for i, g in zip(live, torch.autograd.grad(y, [ts[i] for i in live], dy)):
        assert torch.equal(g, want[("dx", "dwg", "dwu", "dwd")[i]])


def test_autocast():
    x, wg, wu, wd, dy = (t.float() for t in inputs(70, 72, 136, 40, BF))
    want = run(*(t.to(BF) for t in (x, wg, wu, wd, dy)), "silu")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    with torch.autocast("cuda", dtype=BF):
        y = gated_ffn(*leaves)
    assert y.dtype == BF and torch.equal(y, want["y"])
    for n, g in zip(("dx", "dwg", "dwu", "dwd"), torch.autograd.grad(y, leaves, dy.to(BF))):
        assert g.dtype == torch.float32 and torch.equal(g, want[n].float()), n
    with torch.autocast("cuda", dtype=BF):  # a backward inside one of another dtype
        y = gated_ffn(*leaves)
        with torch.autocast("cuda", dtype=HF):
            dx, = torch.autograd.grad(y, leaves[:1], dy.to(BF))
    assert torch.equal(dx, want["dx"].float())


def test_second_order():
    """The graph of the backward is torch's: its gradients against float64 double backward, within
    the roundings of five 16-bit ops in a row."""
    ts = [t.detach().requires_grad_() for t in inputs(6, 64, 72, 64, HF, seed=9)[:4]]
    dy = inputs(6, 64, 72, 64, HF, seed=9)[4]
    got, want = [], []
    for fn, leaves, up, out in ((gated_ffn, ts, dy, got), (None, [t.detach().double().requires_grad_() for t in ts], dy.double(), want)):
        y = fn(*leaves, "gelu") if fn else torch_gated_ffn(*leaves, "gelu")
        gx, = torch.autograd.grad(y, leaves[0], up, create_graph=True)
        out += torch.autograd.grad(gx.double().square().sum(), leaves)
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= 8 * 2.0 ** -11 * float(b.norm())
    wd_only = ts[3].detach().clone().requires_grad_()
    up = dy.clone().requires_grad_()
    g, = torch.autograd.grad(gated_ffn(ts[0].detach(), ts[1].detach(), ts[2].detach(), wd_only), wd_only, up, create_graph=True)
    assert torch.autograd.grad(g.sum(), up)[0].shape == up.shape


def test_changed_in_place_is_refused():
    x, wg, wu, wd, dy = inputs(20, 64, 72, 40, BF)
    for i in range(4):
        ts = [t.detach().clone().requires_grad_() for t in (x, wg, wu, wd)]
        y = gated_ffn(*ts)
        with torch.no_grad():
            ts[i].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y, ts, dy)
    # a weight that no wanted gradient reads may change, as with linears
    wd1 = wd.detach().clone().requires_grad_()
    y = gated_ffn(x, wg, wu, wd1)
    with torch.no_grad():
        wd1.add_(1)
    torch.autograd.grad(y, wd1, dy)
    y = gated_ffn(x.clone().requires_grad_(), wg, wu, wd)
    y.add_(1)  # the output may be modified in place


def test_streams_and_graph():
    """Another stream; a captured forward and backward replayed over new inputs, with eager work
    between the replays, against eager results."""
    x, wg, wu, wd, dy = inputs(90, 72, 136, 40, BF)
    want = run(x, wg, wu, wd, dy, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, wg, wu, wd, dy, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)
    leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu, wd)]
    up = dy.clone()

    def step():
        y = gated_ffn(*leaves)
        return y.detach(), *torch.autograd.grad(y, leaves, up)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        new = inputs(90, 72, 136, 40, BF, seed=20 + seed)
        with torch.no_grad():
            for a, b in zip((*leaves, up), new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(*new, "silu")
        for a, n in zip(outs, ("y", "dx", "dwg", "dwu", "dwd")):
            assert torch.equal(a, eager[n]), (seed, n)


def test_runs_agree():
    """Sums run in a fixed order: the same bits on every call."""
    args = inputs(1030, 264, 712, 264, BF)
    a, b = run(*args, "silu"), run(*args, "silu")
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_refusals_on_gpu():
    x, wg, wu, wd, _ = inputs(4, 64, 72, 40, BF)
    for args in ((x.float(), wg, wu, wd), (x, wg.half(), wu, wd), (x[:, :60], wg[:, :60], wu[:, :60], wd), (x, wg, wu[:64], wd),
                 (x, wg, wu, wd[:, :64]), (x, wg, wu, wd.cpu()), (x.float(), wg.float(), wu.float(), wd.float())):
        with pytest.raises(_hip.DsaltError):
            gated_ffn(*args)
    with pytest.raises(ValueError, match="activation"):
        gated_ffn(x, wg, wu, wd, activation="tanh")


@pytest.mark.parametrize("rows", [5, 150])
def test_one_tensor_in_several_places_and_two_backwards(rows):
    """x a row, w_gate used as w_up and w_down too: the gradients add up; a graph kept for a second
    backward gives the same."""
    x, wg, _, _, dy = inputs(rows, 64, 64, 64, HF, seed=2)
    print(f"gated_ffn one weight three times {rows}", flush=True)
    apart = run(x, wg, wg, wg, dy, "silu")
    a, w = x.clone().requires_grad_(), wg.clone().requires_grad_()
    y = gated_ffn(a, w, w, w)
    first = torch.autograd.grad(y, (a, w), dy, retain_graph=True)
    second = torch.autograd.grad(y, (a, w), dy)
    assert torch.equal(y, apart["y"]) and torch.equal(first[0], apart["dx"])
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    total = apart["dwg"].double() + apart["dwu"].double() + apart["dwd"].double()
    # autograd's two additions in fp16: a half-step each, of sums within the magnitudes' sum
    bound = 2 * 2.0 ** -11 * 1.01 * sum(apart[n].double().abs() for n in ("dwg", "dwu", "dwd")) + 2.0 ** -24
    assert bool(((first[1].double() - total).abs() <= bound).all())
    one = gated_ffn(x[0], wg, wg, wg)
    assert one.shape == (64,) and torch.equal(one, gated_ffn(x[:1], wg, wg, wg)[0])


def test_two_graphs_and_eager_calls_in_turn():
    """Two captured forward passes of unlike sizes (split products, so that each has a workspace),
    replayed in turn with eager calls between."""
    cases = [inputs(300, 512, 1408, 512, BF), inputs(90, 1024, 2816, 1024, BF)]
    graphs, outs = [], []
    with torch.no_grad():
        want = [gated_ffn(x, wg, wu, wd) for x, wg, wu, wd, _ in cases]
        for x, wg, wu, wd, _ in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(gated_ffn(x, wg, wu, wd))
            graphs.append(g)
        for turn in range(4):
            print(f"gated_ffn replay {turn}", flush=True)
            for i in (0, 1) if turn % 2 else (1, 0):
                outs[i].zero_()
                graphs[i].replay()
                x, wg, wu, wd, _ = cases[1 - i]
                assert torch.equal(gated_ffn(x, wg, wu, wd), want[1 - i])
            for got, ref in zip(outs, want):
                assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("rows,d,f", [(20, 72, 136), (150, 72, 136), (575, 264, 712), (1500, 512, 1408), (8579, 904, 712), (2049, 2048, 1408)])
def test_weights_of_different_row_strides(rows, d, f, dtype):
    """Each weight a column slice of a wider matrix of its own: the bits of contiguous weights, with w_up's
    stride above and below w_gate's. Sizes with whole and with split tiles of every shape."""
    x, wg, wu, wd, dy = inputs(rows, d, f, d, dtype)
    want = run(x, wg, wu, wd, dy, "silu")

    def wider(t, more):  # NaN beside it: what is read of it shows
        w = torch.full((t.shape[0], t.shape[1] + more), float("nan"), device=DEV, dtype=dtype)
        w[:, 8:8 + t.shape[1]] = t
        return w[:, 8:8 + t.shape[1]]

    for more in ((0, 16, 8), (64, 8, 24), (8, 1024, 16)):
        print(f"gated_ffn strides {rows} x {d} x {f} + {more} {dtype}", flush=True)
        ws = [wider(w, m) if m else w for w, m in zip((wg, wu, wd), more)]
        assert [w.stride(0) for w in ws] == [d + more[0], d + more[1], f + more[2]]
        got = run_views(x, *ws, dy)
        for n in want:
            assert torch.equal(got[n], want[n]), (more, n)


@pytest.mark.parametrize("rows", [25, 97])
@pytest.mark.parametrize("dtype,lowest,up,scale", [(BF, -10.0, 1.0, 1.0), (HF, -5.5, 2.0 ** 14, 2.0 ** 10)], ids=["bf16", "fp16"])
def test_gelu_of_far_negative_gates(dtype, lowest, up, scale, rows):
    """GELU and its slope where phi(g) is small, each element by itself: g and u are single products, y, dx
    and the inner gradients single ones of what was rounded, so that a relative bound holds: half a
    step, plus 2^-15 for an exp of exponents up to 72, rounded to 2^-24 of that three times, and the
    sum of slope's two terms, of which the smaller is at most a sixteenth. fp16's u and dy keep the
    values above its smallest normal one."""
    print(f"gated_ffn gelu tail {rows} {dtype}", flush=True)
    g = torch.linspace(lowest, -4.0, rows, device=DEV).to(dtype)
    x = torch.zeros(rows, 8, device=DEV, dtype=dtype)
    x[:, 0], x[:, 1] = g, up
    wg, wu, wd = (torch.zeros(8, 8, device=DEV, dtype=dtype) for _ in range(3))
    wg[0, 0] = wu[0, 1] = wd[0, 0] = 1
    dy = torch.zeros_like(x)
    dy[:, 0] = scale
    got = run(x, wg, wu, wd, dy, "gelu")
    z = g.double()
    phi = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    slope = phi + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5
    bound = torch.finfo(dtype).eps / 2 + 2.0 ** -15
    for n, have, want in (("y", got["y"][:, 0], z * phi * up), ("dg", got["dx"][:, 0], scale * up * slope),
                          ("du", got["dx"][:, 1], scale * z * phi)):
        assert float(want.abs().min()) > torch.finfo(dtype).tiny and float(want.abs().max()) < torch.finfo(dtype).max
        assert bool(((have.double() - want).abs() <= bound * want.abs()).all()), (n, float((have.double() / want - 1).abs().max()))


def test_transforms_and_tracing():
    """What an autograd function with a HIP kernel does not know runs as torch's ops."""
    x, wg, wu, wd, dy = inputs(12, 64, 72, 40, HF)
    ref = reference(x, wg, wu, wd, dy, "silu", HF)
    got = torch.func.grad(lambda t: (gated_ffn(t, wg, wu, wd).float() * dy.float()).sum())(x)
    want = run(x, wg, wu, wd, dy, "silu")
    # some five fp16 roundings in a chain on torch's side, two on the kernels', each half a step at most
    near = lambda a, b: float((a.double() - b.double()).norm()) <= 7 * 2.0 ** -11 * float(b.double().norm())
    assert near(got, want["dx"])
    assert near(torch.jit.trace(lambda t: gated_ffn(t, wg, wu, wd), (x,), check_trace=False)(x), ref["y"][0])
    assert near(torch.func.vmap(lambda t: gated_ffn(t, wg, wu, wd))(x.view(3, 4, 64)).view(12, 40), ref["y"][0])
    v = torch.randn(12, 64, device=DEV).to(HF)
    _, tangent = torch.func.jvp(lambda t: gated_ffn(t, wg, wu, wd), (x,), (v,))
    size = float((want["dx"].double() * v.double()).abs().sum())
    assert abs(float((tangent.double() * dy.double()).sum() - (want["dx"].double() * v.double()).sum())) <= 7 * 2.0 ** -11 * size


@pytest.mark.parametrize("rows", [5, 140])
def test_frozen_inference_tensors(rows):
    """Weights and rows loaded under inference_mode, which count no versions, beside a trainable down
    projection: as linears, which save neither."""
    x, wg, wu, wd, dy = inputs(rows, 64, 72, 40, BF)
    want = run(x, wg, wu, wd, dy, "silu")
    with torch.inference_mode():
        frozen = [t.clone() for t in (x, wg, wu)]
    w = wd.clone().requires_grad_()
    y = gated_ffn(*frozen, w)
    assert torch.equal(y, want["y"]) and torch.equal(torch.autograd.grad(y, w, dy)[0], want["dwd"])
    y = gated_ffn(*frozen, w)
    up = dy.clone().requires_grad_()
    g, = torch.autograd.grad(y, w, up, create_graph=True)
    assert torch.autograd.grad(g.sum(), up)[0].shape == up.shape
    gate = wg.clone().requires_grad_()
    for graph in (False, True):
        g, = torch.autograd.grad(gated_ffn(x, gate, frozen[2], wd), gate, dy, create_graph=graph)
        # with a graph the backward is torch's, with some five roundings to bf16 in a chain
        assert torch.equal(g, want["dwg"]) if not graph else float((g - want["dwg"]).norm()) <= 7 * 2.0 ** -8 * float(g.norm())
    with pytest.raises(RuntimeError, match="[Ii]nference"):  # a gradient that reads them is refused by torch
        gated_ffn(x.clone().requires_grad_(), *frozen[1:], wd)
    with torch.inference_mode():
        assert torch.equal(gated_ffn(*frozen, wd), want["y"])
