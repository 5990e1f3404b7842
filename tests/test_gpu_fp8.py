"""fp8_quantize, fp8_matmul and fp8_linear against float64."""
import pytest
import torch

from dsalt import DsaltError, _hip
from dsalt.kernels import FP8Linear, fp8_linear, fp8_matmul, fp8_quantize
from dsalt.kernels.fp8 import torch_fp8_matmul, torch_fp8_quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def rand(*shape, seed=0, dtype=FP, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return (torch.randn(*shape, device=DEV, generator=g) * std * torch.exp(torch.randn(shape[-1], device=DEV, generator=g))).to(dtype)


def spread(scale, n, k, tile):
    s = scale.double().repeat_interleave(128, 1)[:, :k]
    return s.repeat_interleave(128, 0)[:n] if tile else s


def exact_quantize(x, tile):
    """Scales by comparison with every power of two, elements rounded on e4m3's grid in float64."""
    n, k = x.shape
    rows = 128 if tile else 1
    nb, kb = -(-n // rows), -(-k // 128)
    pad = torch.zeros(nb * rows, kb * 128, dtype=torch.float64, device=DEV)
    pad[:n, :k] = x.double()
    v = pad.view(nb, rows, kb, 128)
    amax = v.abs().amax((1, 3))
    scale = torch.ones_like(amax)
    powers = torch.exp2(torch.arange(-127, 121, dtype=torch.float64, device=DEV))  # exact, as 2.0 ** is not
    at = (448 * powers < amax[..., None]).sum(-1)
    scale = torch.where(amax > 0, powers[at.clamp(max=len(powers) - 1)], 1.0)
    r = v / scale[:, None, :, None]
    step = torch.exp2(torch.frexp(r.abs().clamp(min=2.0 ** -6))[1].double() - 4)
    q = torch.round(r / step) * step
    return q.reshape(pad.shape)[:n, :k], scale


@pytest.mark.parametrize("n,k", [(1, 1), (1, 16), (3, 127), (5, 128), (7, 129), (130, 264), (128, 1024), (257, 1000), (64, 4096)])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("tile", [False, True])
def test_quantize(n, k, dtype, tile):
    x = rand(n, k, dtype=dtype)
    x[0, 0] = 0
    q, s = fp8_quantize(x, tile)
    wq, ws = exact_quantize(x, tile)
    assert q.dtype is E4 and s.dtype is E8 and q.shape == x.shape and s.shape == ws.shape
    assert torch.equal(s.double(), ws) and torch.equal(q.double(), wq)
    q2, s2 = fp8_quantize(x, tile, FP)
    assert s2.dtype is FP and torch.equal(s2.double(), ws) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))
    tq, ts = torch_fp8_quantize(x, tile, E8)
    assert torch.equal(tq.view(torch.uint8), q.view(torch.uint8)) and torch.equal(ts.view(torch.uint8), s.view(torch.uint8))


def test_quantize_edges():
    """Largest values on and beside 448 times a power of two, zeros, tiny values, the types' largest."""
    row = torch.zeros(12, 128, device=DEV)
    tops = [448.0, 448.00003, 447.99997, 0.0, 1e-45, 2.0 ** -126, 448 * 2.0 ** -127, 449 * 2.0 ** -127, 3.4028235e38, 1.0, 256.0, 1.75]
    row[:, 5] = torch.tensor(tops, device=DEV)
    row[:, 7] = -row[:, 5] / 3
    q, s = fp8_quantize(row)
    wq, ws = exact_quantize(row, False)
    assert torch.equal(s.double(), ws) and torch.equal(q.double(), wq)
    ties = (torch.arange(128, device=DEV) / 16 + 16).expand(1, 128).clone()  # halves of e4m3's steps between 16 and 24
    ties[0, 0] = 448.0
    q, _ = fp8_quantize(ties)
    assert torch.equal(q.double(), exact_quantize(ties, False)[0])


def test_quantize_nonfinite():
    x = torch.ones(4, 300, device=DEV)
    x[1, 130], x[2, 299] = float("inf"), float("nan")
    q, s = fp8_quantize(x)
    bad = torch.zeros(4, 3, dtype=torch.bool, device=DEV)
    bad[1, 1] = bad[2, 2] = True
    assert torch.equal(torch.isnan(s.float()), bad)
    assert torch.equal(torch.isnan(q.float()), bad.repeat_interleave(128, 1)[:, :300])
    q, s = fp8_quantize(x[:3], tile=True)
    assert torch.equal(torch.isnan(s.float())[0], torch.tensor([False, True, True], device=DEV))


def test_quantize_shapes_and_strides():
    x = rand(6, 5, 200, dtype=BF)
    q, s = fp8_quantize(x)
    assert q.shape == x.shape and s.shape == (6, 5, 2)
    for y in (x.transpose(0, 1).contiguous().transpose(0, 1), rand(6, 5, 201, dtype=BF)[..., 1:]):
        q, s = fp8_quantize(y)
        wq, ws = exact_quantize(y.reshape(30, 200), False)
        assert torch.equal(q.double().view(30, 200), wq) and torch.equal(s.double().view(30, 2), ws)
    q, s = fp8_quantize(torch.zeros(0, 64, device=DEV))
    assert q.shape == (0, 64) and s.shape == (0, 1)
    q, s = fp8_quantize(rand(70, dtype=FP))
    assert q.shape == (70,) and s.shape == (1,)


def operands(m, n, k, a_f32=False, b_f32=False, seed=0):
    a, sa = fp8_quantize(rand(m, k, seed=seed), scale_dtype=FP if a_f32 else E8)
    b, sb = fp8_quantize(rand(n, k, seed=seed + 1, std=0.02), True, FP if b_f32 else E8)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if a_f32:  # any fp32 values
        sa = sa * (0.5 + torch.rand(sa.shape, device=DEV, generator=g))
    if b_f32:
        sb = sb * (0.5 + torch.rand(sb.shape, device=DEV, generator=g))
    return a, sa, b, sb


def check(out, a, sa, b, sb, bias=None, dtype=BF):
    """The matrix instruction adds the products of eight consecutive k aligned to the largest one's exponent, to
    13 bits below it: each of the other seven loses less than 2^-13 of that product, which the group's largest
    a times its largest b bounds. Beyond a group all is fp32: a sum of k terms in any order is within
    k 2^-24 of the sum of magnitudes; scales and bias add three roundings, and the result's own is half a step."""
    m, k, n = a.shape[0], a.shape[1], b.shape[0]
    x, w = a.double() * spread(sa, m, k, False), b.double() * spread(sb, n, k, True)
    want = x @ w.t()
    size = x.abs() @ w.abs().t()
    cut = 7 * 2.0 ** -13 * (x.abs().view(m, -1, 8).amax(-1) @ w.abs().view(n, -1, 8).amax(-1).t())
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    assert out.dtype is dtype and out.shape == want.shape
    err = (out.double() - want).abs()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + cut + (k + 3) * 2.0 ** -24 * size + (2.0 ** -25 if dtype is HF else 0.0)
    assert bool((err <= tol).all()), float((err / tol).max())


SIZES = [(1, 1, 16), (1, 128, 128), (3, 17, 144), (16, 16, 1024), (17, 200, 272), (32, 1024, 2816), (33, 64, 128), (64, 64, 128),
         (65, 130, 160), (100, 1001, 1360), (128, 128, 256), (200, 72, 4096), (257, 256, 128), (575, 712, 272), (300, 5000, 640),
         (2048, 1000, 384), (4100, 4200, 272)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("a_f32,b_f32", [(False, False), (True, True), (False, True), (True, False)])
def test_matmul(m, n, k, a_f32, b_f32):
    a, sa, b, sb = operands(m, n, k, a_f32, b_f32)
    for dtype in (BF, FP):
        check(fp8_matmul(a, sa, b, sb, out_dtype=dtype), a, sa, b, sb, dtype=dtype)


@pytest.mark.parametrize("m", [1, 20, 40, 600])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("bias_dtype", [None, BF, HF, FP])
def test_outputs_and_bias(m, dtype, bias_dtype):
    for n in (96, 101):
        a, sa, b, sb = operands(m, n, 336, seed=m)
        bias = None if bias_dtype is None else rand(n, dtype=bias_dtype)
        check(fp8_matmul(a, sa, b, sb, bias, dtype), a, sa, b, sb, bias, dtype)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("f32", [False, True])
def test_linear(m, n, k, dtype, f32):
    """The linear layer quantises as fp8_quantize does, also where the product's kernel does it."""
    x = rand(m, k, dtype=dtype, seed=5)
    _, _, b, sb = operands(1, n, k, b_f32=f32)
    q, s = fp8_quantize(x)
    check(fp8_linear(x, b, sb), q, s, b, sb, dtype=dtype)


def test_sums_over_blocks_keep_fp32():
    """2^16 in one block and 2^-6 in every other: blocks are added in fp32, which holds the sum exactly."""
    for m in (16, 64, 600):
        k = 128 * 40
        a, b = torch.zeros(m, k, device=DEV), torch.zeros(256, k, device=DEV)
        a[:, 64::128], b[:, 64::128] = 0.125, 0.125
        a[:, 64], b[:, 64] = 256.0, 256.0
        one = [torch.full((r, 40), 127, device=DEV, dtype=torch.uint8).view(E8) for r in (m, 2)]
        for scales in (one, [t.float() for t in one]):
            y = fp8_matmul(a.to(E4), scales[0], b.to(E4), scales[1], out_dtype=FP)
            assert bool((y == 2.0 ** 16 + 39 * 2.0 ** -6).all())
    for m, n, k in ((16, 64, 16384), (64, 64, 16384), (600, 600, 16384)):
        a, sa, b, sb = operands(m, n, k)
        check(fp8_matmul(a, sa, b, sb, out_dtype=FP), a, sa, b, sb, dtype=FP)


def test_strides():
    """Operands inside wider ones, transposed scales, misaligned rows: the contiguous bits."""
    for m in (9, 150):
        a, sa, b, sb = operands(m, 200, 272)
        want = fp8_matmul(a, sa, b, sb)
        wide = torch.zeros(m, 320, device=DEV, dtype=torch.uint8).view(E4)
        wide[:, 16:288] = a
        odd = torch.zeros(200, 299, device=DEV, dtype=torch.uint8).view(E4)
        odd[:, 5:277] = b
        turned = [t.view(torch.uint8).t().contiguous().t().view(E8) for t in (sa, sb)]
        for A in (a, wide[:, 16:288]):
            for B in (b, odd[:, 5:277]):
                for SA, SB in ((sa, sb), turned):
                    assert torch.equal(fp8_matmul(A, SA, B, SB), want)
        x = rand(m, 272, dtype=BF)
        wx = torch.zeros(m, 301, device=DEV, dtype=BF)
        wx[:, 7:279] = x
        assert torch.equal(fp8_linear(wx[:, 7:279], b, sb), fp8_linear(x, b, sb))


def test_leading_dimensions_and_empty():
    _, _, b, sb = operands(1, 48, 160)
    x = rand(3, 5, 160, dtype=BF)
    assert torch.equal(fp8_linear(x, b, sb), fp8_linear(x.view(15, 160), b, sb).view(3, 5, 48))
    assert fp8_linear(x[:0], b, sb).shape == (0, 5, 48)
    assert torch.equal(fp8_linear(x[0, 0], b, sb), fp8_linear(x.view(15, 160)[:1], b, sb)[0])
    q, s = fp8_quantize(x)
    assert torch.equal(fp8_matmul(q, s, b, sb), fp8_linear(x, b, sb))


@pytest.mark.parametrize("m", [5, 70])
def test_nonfinite_rows_stay_in_their_rows(m):
    _, _, b, sb = operands(1, 80, 272)
    x = rand(m, 272, dtype=BF)
    want = fp8_linear(x, b, sb)
    x[3, 200] = float("nan")
    x[1, 0] = float("inf")
    got = fp8_linear(x, b, sb)
    bad = torch.zeros(m, dtype=torch.bool, device=DEV)
    bad[1] = bad[3] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])


def test_same_bits_again_and_on_streams():
    for m in (8, 100, 3000):
        a, sa, b, sb = operands(m, 1000, 1360)
        want = fp8_matmul(a, sa, b, sb)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [fp8_matmul(a, sa, b, sb) for _ in range(3)]
        side.synchronize()
        assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("m", [4, 100, 900])
def test_captured_and_replayed(m):
    x = rand(m, 1024, dtype=BF)
    _, _, b, sb = operands(1, 600, 1024)
    with torch.no_grad():
        fp8_linear(x, b, sb)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8_linear(x, b, sb)
        for k in range(4):
            x.copy_(rand(m, 1024, dtype=BF, seed=k))
            graph.replay()
            torch.cuda.synchronize()
            kept = y.clone()
            assert torch.equal(kept, fp8_linear(x, b, sb))


def test_offsets_past_32_bits():
    """Rows of the operand and of the result past 4 GiB."""
    m, n, k = (1 << 32) // 4096 + 300, 2048, 4096
    a = torch.zeros(m, k, device=DEV, dtype=torch.uint8).view(E4)
    sa = torch.full((m, 32), 127, device=DEV, dtype=torch.uint8).view(E8)
    ta, tsa, b, sb = operands(300, n, k)
    a[-300:], sa[-300:] = ta, tsa
    out = fp8_matmul(a, sa, b, sb)
    check(out[-300:], ta, tsa, b, sb)
    assert out.numel() * 2 > 1 << 32 and not out[:-300].any()


def test_module():
    for bias in (False, True):
        lin = torch.nn.Linear(272, 200, bias=bias).to(DEV, BF)
        m = FP8Linear.from_linear(lin)
        x = rand(50, 272, dtype=BF)
        with torch.no_grad():
            y = m(x)
            assert torch.equal(y, fp8_linear(x, *fp8_quantize(lin.weight, tile=True), lin.bias))
            assert float((y.float() - lin(x).float()).norm() / lin(x).float().norm()) < 0.06  # two e4m3 roundings of 2^-4 at most
        assert m.half().weight_bits.dtype is torch.uint8 and not list(p for p in m.parameters() if p.requires_grad)
        other = FP8Linear(272, 200, bias, DEV, HF)
        other.load_state_dict(m.state_dict())
        with torch.no_grad():
            assert torch.equal(other(x), m(x))


def test_torch_forms():
    """What tracing and transforms run: the same quantisation, the product in fp32."""
    a, sa, b, sb = operands(20, 200, 272, b_f32=True)
    check(torch_fp8_matmul(a, sa, b, sb, None, FP), a, sa, b, sb, dtype=FP)
    x = rand(6, 272)
    got = torch.vmap(lambda t: fp8_linear(t, b, sb))(x.view(3, 2, 272))
    check(got.view(6, 200), *fp8_quantize(x), b, sb, dtype=FP)
    assert torch.equal(torch.compile(lambda t: fp8_linear(t, b, sb) * 2)(x), 2 * fp8_linear(x, b, sb))


def test_refusals():
    a, sa, b, sb = operands(40, 64, 256)
    x = rand(40, 256, dtype=BF)
    for call in (lambda: fp8_matmul(x, sa, b, sb), lambda: fp8_matmul(a, sa[:39], b, sb), lambda: fp8_matmul(a, sa, b, sb[:, :1]),
                 lambda: fp8_matmul(a[:, :250], sa, b[:, :250], sb), lambda: fp8_matmul(a, sa, b[:, :128], sb[:, :1]),
                 lambda: fp8_matmul(a, sa.to(BF), b, sb), lambda: fp8_matmul(a, sa, b, sb, out_dtype=torch.float64),
                 lambda: fp8_matmul(a, sa, b, sb, torch.zeros(63, device=DEV)), lambda: fp8_linear(x.double(), b, sb),
                 lambda: fp8_linear(x[:, :128], b, sb), lambda: fp8_linear(x, b, sb.cpu()), lambda: fp8_quantize(x.double()),
                 lambda: fp8_quantize(x.view(5, 8, 256), tile=True), lambda: fp8_quantize(x, scale_dtype=HF),
                 lambda: fp8_quantize(x[:, :0])):
        with pytest.raises(DsaltError):
            call()
    with pytest.raises(DsaltError, match="inference"):
        fp8_linear(x.requires_grad_(), b, sb)
    with torch.no_grad():
        fp8_linear(x, b, sb)
    assert _hip.FP8_FEW_ROWS == _hip.lib().dsalt_fp8_few_rows()
