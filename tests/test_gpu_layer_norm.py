"""layer_norm and add_layer_norm (one pass forward and one backward) against float64 autograd."""
import pytest
import torch

from dsalt import DsaltError, _hip
from dsalt.kernels import LayerNorm, add_layer_norm, layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def inputs(lead, d, xd, hd, od, add=True, weight=True, bias=True, wd=None, seed=0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed + d)
    wd = xd if wd is None else wd

    def rnd(dt, *s, std=1.0, mean=0.0):
        return (torch.randn(*s, device=DEV, generator=g) * std + mean).to(dt)

    t = {"x": rnd(xd, *lead, d, std=2.0, mean=mean), "h": rnd(hd, *lead, d) if add else None,
         "weight": rnd(wd, d, std=0.25, mean=1.0) if weight else None, "bias": rnd(wd, d, std=0.5) if bias else None}
    return t, rnd(xd, *lead, d) if add else None, rnd(od, *lead, d)


def reference(t, dz, dy, eps):
    w = {n: v.detach().double().requires_grad_() for n, v in t.items() if v is not None}
    z = w["x"] + w["h"] if "h" in w else w["x"] * 1
    zc = z - z.mean(-1, keepdim=True)
    n = zc / torch.sqrt(zc.square().mean(-1, keepdim=True) + eps)
    y = n * w.get("weight", 1.0) + w.get("bias", 0.0)
    pairs = [(o, u.double()) for o, u in ((z, dz if "h" in w else None), (y, dy)) if u is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(w.values()), [u for _, u in pairs], allow_unused=True)
    return ([z.detach()] if "h" in w else []) + [y.detach()], dict(zip(w, grads)), n.detach()


def close(got, want, dtype, what, scale):
    """One rounding to the dtype, and fp32 arithmetic: sums of d <= 8192 or of `rows` terms run over at
    most 64 terms a lane, then in trees, each rounding at most 2^-24 of what is summed, so that a result
    is within 2^-18 of `scale`, the largest magnitude it is formed from."""
    assert got.dtype == dtype and got.shape == want.shape, what
    err = (got.double() - want).abs()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -18 * scale + (2.0 ** -25 if dtype == HF else 0.0)
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


def run(t, dz, dy, eps, od):
    leaves = {n: v.detach().clone().requires_grad_() for n, v in t.items() if v is not None}
    wb = leaves.get("weight"), leaves.get("bias")
    outs = (layer_norm(leaves["x"], *wb, eps, od),) if t["h"] is None else add_layer_norm(leaves["x"], leaves["h"], *wb, eps, od)
    pairs = [(o, u) for o, u in zip(outs, (dy,) if t["h"] is None else (dz, dy)) if u is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [u for _, u in pairs], allow_unused=True)
    return [o.detach() for o in outs], dict(zip(leaves, grads))


def compare(t, dz, dy, eps=1e-5, od=None):
    od = t["x"].dtype if od is None else od
    outs, grads = run(t, dz, dy, eps, od)
    w_outs, w_grads, n = reference(t, dz, dy, eps)
    z = w_outs[0] if t["h"] is not None else t["x"].double()
    zmax = z.abs().max()
    # the centred row carries z's own magnitude, over its deviation
    rmax = (1 / torch.sqrt(z.var(-1, unbiased=False) + eps)).max() if z.numel() else 0.0
    amax = max(float(n.abs().max()), float(zmax * rmax))
    wmax = 1.0 if t["weight"] is None else t["weight"].double().abs().max()
    for name, a, b in zip(("x_out", "y") if t["h"] is not None else ("y",), outs, w_outs):
        close(a, b, t["x"].dtype if name == "x_out" else od, name, zmax if name == "x_out" else amax * wmax + b.abs().max())
    rows = max(z.numel() // z.shape[-1], 1)
    gmax = 0.0 if dy is None else dy.double().abs().max()
    for name, g in grads.items():
        if g is None:
            assert w_grads[name] is None or not w_grads[name].any(), name
            continue
        if name in ("x", "h"):
            scale = rmax * gmax * wmax * (1 + amax * amax) + (0.0 if dz is None else dz.double().abs().max())
        else:
            scale = rows ** 0.5 * gmax * (1 + amax)
        close(g, w_grads[name], t[name].dtype, name, scale)


@pytest.mark.parametrize("d", [1, 2, 7, 8, 63, 64, 100, 511, 512, 513, 1000, 1024, 1031, 2048, 2056, 4096, 4099, 8184, 8191, 8192])
@pytest.mark.parametrize("add", [False, True])
def test_widths(d, add):
    compare(*inputs((5,), d, BF, BF, BF, add=add))
    compare(*inputs((37,), d, FP, FP, FP, add=add))


@pytest.mark.parametrize("xd,hd,od", [(BF, BF, BF), (HF, HF, HF), (FP, FP, FP), (FP, BF, BF), (FP, HF, HF), (FP, BF, HF), (FP, FP, BF)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("d", [72, 75])
def test_types(xd, hd, od, wide, d):
    compare(*inputs((3, 11), d, xd, hd, od, wd=FP if wide else None), od=od)
    compare(*inputs((3, 11), d, xd, hd, od, add=False, wd=FP if wide else None), od=od)


@pytest.mark.parametrize("rows", [1, 7, 8, 9, 300, 5000])
@pytest.mark.parametrize("d", [264, 1024])
def test_rows(rows, d):
    compare(*inputs((rows,), d, FP, BF, BF), od=BF)


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("add", [False, True])
def test_without_weight_or_bias(weight, bias, add):
    compare(*inputs((20,), 96, BF, BF, BF, add=add, weight=weight, bias=bias))


@pytest.mark.parametrize("which", ["dz", "dy"])
@pytest.mark.parametrize("xd", [BF, FP])
def test_one_upstream_gradient(which, xd):
    t, dz, dy = inputs((20,), 96, xd, xd, xd)
    compare(t, dz if which == "dz" else None, dy if which == "dy" else None)


def test_mean_far_from_zero():
    """The variance of rows whose mean is a thousand deviations away: a sum of squares would lose it."""
    compare(*inputs((64,), 1024, FP, FP, FP, add=False, mean=2000.0))


def test_constant_rows_and_large_eps():
    """A row of one value (also d = 1) has no deviation: y = bias, its gradient is finite."""
    t, dz, dy = inputs((6,), 40, FP, FP, FP, add=False)
    t["x"][:] = 3.0
    outs, grads = run(t, dz, dy, 1e-5, FP)
    assert torch.equal(outs[0], t["bias"].expand(6, 40)) and bool(torch.isfinite(grads["x"]).all())
    compare(*inputs((6,), 40, FP, FP, FP, add=False), eps=0.5)


def test_nonfinite_rows_stay_in_their_rows():
    t, dz, dy = inputs((9,), 136, BF, BF, BF)
    t["x"][2, 5], t["h"][4, 0] = float("nan"), float("inf")
    outs, grads = run(t, dz, dy, 1e-5, BF)
    bad = torch.zeros(9, dtype=torch.bool, device=DEV)
    bad[2] = bad[4] = True
    assert bool(torch.isnan(outs[1][bad]).all()) and bool(torch.isfinite(outs[1][~bad]).all())
    assert bool(torch.isfinite(grads["x"][~bad]).all())


def test_empty():
    for lead in ((0,), (3, 0)):
        t, dz, dy = inputs(lead, 24, BF, BF, BF)
        outs, grads = run(t, dz, dy, 1e-5, BF)
        assert outs[0].shape == outs[1].shape == (*lead, 24)
        assert not grads["weight"].any() and not grads["bias"].any() and grads["x"].shape == (*lead, 24)


def test_strides_and_alignment():
    """Transposed, sliced and misaligned operands give the bits of their contiguous copies."""
    t, dz, dy = inputs((16,), 88, BF, BF, BF)
    flat = torch.empty(16 * 88 + 1, device=DEV, dtype=BF)
    odd = flat[1:].view(16, 88).copy_(t["x"])
    assert odd.data_ptr() % 16
    wide = torch.empty(16, 100, device=DEV, dtype=BF)
    sliced = wide[:, 3:91].copy_(t["x"])
    turned = t["x"].t().contiguous().t()
    want, wg = run(t, dz, dy, 1e-5, BF)
    for x in (odd, sliced, turned):
        got = add_layer_norm(x, t["h"], t["weight"], t["bias"])
        assert all(torch.equal(a, b) or float((a.float() - b.float()).abs().max()) <= 2.0 ** -6 for a, b in zip(got, want))
    leaf = sliced.clone().requires_grad_()
    h = t["h"].clone().requires_grad_()
    outs = add_layer_norm(leaf, h, t["weight"], t["bias"])
    g = torch.autograd.grad(outs, (leaf, h), (dz.t().contiguous().t(), dy.expand(16, 88)))
    assert torch.equal(g[0], wg["x"]) and torch.equal(g[1], wg["h"])


def test_second_order_and_differences():
    """The gradient against differences of float64's function, and a gradient of the gradient."""
    for add, xd in ((True, FP), (False, FP), (True, BF)):
        t, dz, dy = inputs((4,), 24, xd, xd, xd, add=add, seed=3)
        leaves = [v.clone().requires_grad_() for v in t.values() if v is not None]
        ref = [v.detach().double().requires_grad_() for v in leaves]

        def plain(*a):
            z, rest = (a[0] + a[1], a[2:]) if add else (a[0], a[1:])
            return torch.nn.functional.layer_norm(z, (24,), rest[0], rest[1], 1e-5)

        got = add_layer_norm(*leaves)[1] if add else layer_norm(*leaves)
        g1 = torch.autograd.grad(got, leaves, dy, create_graph=True)
        w1 = torch.autograd.grad(plain(*ref), ref, dy.double(), create_graph=True)
        g2 = torch.autograd.grad(sum(g.float().square().sum() for g in g1), leaves[:-1])  # the gradient does not depend on the bias
        w2 = torch.autograd.grad(sum(g.square().sum() for g in w1), ref[:-1])
        tol = 0.1 if xd == BF else 1e-3
        for a, b in zip(g2, w2):
            assert float((a.double() - b).norm() / b.norm()) < tol
    x = torch.randn(3, 10, dtype=torch.float64)
    w, b = torch.randn(10, dtype=torch.float64), torch.randn(10, dtype=torch.float64)
    dy = torch.randn(3, 10, dtype=torch.float64)
    leaf = x.float().to(DEV).requires_grad_()
    g, = torch.autograd.grad(layer_norm(leaf, w.float().to(DEV), b.float().to(DEV)), leaf, dy.float().to(DEV))
    step = 1e-6
    for i, j in ((0, 0), (1, 4), (2, 9)):
        hi, lo = x.clone(), x.clone()
        hi[i, j] += step
        lo[i, j] -= step
        f = [(torch.nn.functional.layer_norm(t, (10,), w, b, 1e-5) * dy).sum() for t in (hi, lo)]
        # differences of step 1e-6 in float64: 1e-9; fp32 arithmetic on values of order one: 1e-5
        assert abs(float((f[0] - f[1]) / (2 * step)) - float(g[i, j])) < 1e-4


def test_captured_and_replayed():
    """A training pass in a graph, replayed on new inputs between eager work, gives the eager bits."""
    t, dz, dy = inputs((33,), 200, FP, BF, BF)
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}

    def step():
        outs = add_layer_norm(*leaves.values(), out_dtype=BF)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, list(leaves.values()), (dz, dy))]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        new, _, _ = inputs((33,), 200, FP, BF, BF, seed=10 + k)
        with torch.no_grad():
            for n, v in leaves.items():
                v.copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        kept = [g.clone() for g in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


def test_streams():
    t, dz, dy = inputs((300,), 1024, BF, BF, BF)
    want = run(t, dz, dy, 1e-5, BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, dz, dy, 1e-5, BF)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[0], want[0])) and all(torch.equal(got[1][n], want[1][n]) for n in want[1])


def test_offsets_past_32_bits():
    """Rows whose bytes lie past 4 GiB."""
    rows, d = (1 << 31) // 4096 + 9, 4096
    x = torch.zeros(rows, d, device=DEV, dtype=BF)
    w = torch.linspace(0.5, 1.5, d, device=DEV)
    last = torch.randn(9, d, device=DEV).to(BF)
    x[-9:] = last
    with torch.no_grad():
        y = layer_norm(x, w)
        assert torch.equal(y[-9:], layer_norm(last, w)) and not y[:-9].any()


def test_module():
    m = LayerNorm(96).to(DEV)
    with torch.no_grad():
        m.weight.normal_(1.0, 0.2)
        m.bias.normal_()
    x, h = torch.randn(5, 96, device=DEV), torch.randn(5, 96, device=DEV)
    want = torch.nn.functional.layer_norm(x.double(), (96,), m.weight.double(), m.bias.double(), m.eps)
    torch.testing.assert_close(m(x).double(), want, rtol=1e-5, atol=1e-5)
    s, y = m(x, h.to(BF), out_dtype=BF)
    assert s.dtype == FP and y.dtype == BF and torch.equal(s, x + h.to(BF))
    assert m(x.to(BF)).dtype == BF
    half = LayerNorm(96, bias=False).to(DEV, BF)
    assert half(x).dtype == FP and half.bias is None


def test_transforms_and_compile():
    """vmap, forward mode and torch.compile give torch's values."""
    x = torch.randn(6, 40, device=DEV)
    w, b = torch.randn(40, device=DEV), torch.randn(40, device=DEV)
    want = torch.nn.functional.layer_norm(x, (40,), w, b)
    torch.testing.assert_close(torch.vmap(lambda t: layer_norm(t, w, b))(x), want)
    _, jvp = torch.func.jvp(lambda t: layer_norm(t, w, b), (x,), (torch.ones_like(x),))
    assert float(jvp.abs().max()) < 1e-4  # a constant added to a row changes nothing
    torch.testing.assert_close(torch.compile(lambda t: layer_norm(t, w, b) * 2)(x), 2 * want)


def test_refusals():
    x, w = torch.randn(4, 32, device=DEV, dtype=BF), torch.ones(32, device=DEV, dtype=BF)
    for call in (lambda: layer_norm(x.double()), lambda: layer_norm(x, w[:31]), lambda: layer_norm(x, w.half()),
                 lambda: layer_norm(x, out_dtype=FP), lambda: add_layer_norm(x, x[:3]), lambda: add_layer_norm(x, x.half()),
                 lambda: layer_norm(torch.zeros(2, 8193, device=DEV)), lambda: layer_norm(torch.zeros(2, 0, device=DEV)),
                 lambda: layer_norm(x, w.cpu()), lambda: layer_norm(torch.zeros((), device=DEV))):
        with pytest.raises(DsaltError):
            call()
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    assert _hip.LAYER_NORM_MAX_DIM == 8192
