"""fp8_matmul and fp8_linear on every tile and split that sizes choose, each at ragged sizes, with a bias and in every
type of result. A case names the plan that it means to reach."""
import pytest
import torch

from dsalt import _hip
from dsalt.kernels import fp8_linear, fp8_matmul, fp8_quantize
from test_gpu_fp8 import BF, DEV, FP, HF, check, operands, rand

pytestmark = pytest.mark.gpu

# m, n, k, the plan with fp32 scales, the plan with e8m0 ones (rows and columns of a tile, splits of k)
T64, T128, T256 = (64, 128, 1), (128, 128, 1), (256, 256, 1)
LARGE = [
    (2500, 3000, 1040, T128, T128), (2500, 3001, 1040, T128, T128), (2500, 3002, 144, T128, T128), (2100, 3001, 16, T128, T128),
    (3001, 2056, 1040, T128, T128), (3001, 2056, 128, T128, T128), (4100, 3002, 144, T128, T256), (4100, 3008, 528, T128, T256),
    (3001, 3000, 1040, T64, T256), (3001, 3001, 1040, T64, T256), (1999, 5001, 16, T64, T256), (4099, 2056, 128, T64, T256),
    (2049, 4100, 2064, T64, T256), (5000, 5001, 272, T128, T256), (6473, 5000, 528, T128, T128), (300, 5001, 640, T64, T64), (33, 1001, 272, T64, T64)]
SPLIT = [(65, 5001, 4112, 2), (300, 515, 2064, 4), (200, 258, 2064, 6), (100, 1000, 4112, 7), (33, 3001, 8208, 8), (64, 101, 2064, 9)]


def reached(m, n, k, want, e8m0):
    assert _hip.fp8_plan(m, n, k, e8m0) == want


@pytest.mark.parametrize("m,n,k,f32_plan,e8_plan", LARGE)
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("with_bias", [False, True])
def test_large_tiles(m, n, k, f32_plan, e8_plan, f32, dtype, with_bias):
    reached(m, n, k, f32_plan if f32 else e8_plan, not f32)
    a, sa, b, sb = operands(m, n, k, f32, f32)
    bias = rand(n, dtype=dtype) if with_bias else None
    check(fp8_matmul(a, sa, b, sb, bias, dtype), a, sa, b, sb, bias, dtype)


@pytest.mark.parametrize("m,n,k,splits", SPLIT)
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("with_bias", [False, True])
def test_splits(m, n, k, splits, f32, dtype, with_bias):
    reached(m, n, k, (64, 128, splits), not f32)
    a, sa, b, sb = operands(m, n, k, f32, f32)
    bias = rand(n, dtype=dtype) if with_bias else None
    check(fp8_matmul(a, sa, b, sb, bias, dtype), a, sa, b, sb, bias, dtype)


@pytest.mark.parametrize("m", [1, 16, 17, 32])
@pytest.mark.parametrize("n,columns", [(15359, 16), (15360, 32), (15362, 32), (30719, 32), (30720, 64), (30723, 64)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("f32", [False, True])
def test_few_rows(m, n, columns, dtype, f32):
    """Rows in 8 bits and rows that are quantised on the way, with a bias; 1200 columns of k end inside a block."""
    reached(m, n, 1200, (16 if m <= 16 else 32, columns, 1), not f32)
    a, sa, b, sb = operands(m, n, 1200, f32, f32)
    bias = rand(n, dtype=dtype)
    check(fp8_matmul(a, sa, b, sb, bias, dtype), a, sa, b, sb, bias, dtype)
    x = rand(m, 1200, dtype=dtype, seed=5)
    q, s = fp8_quantize(x)
    check(fp8_linear(x, b, sb, bias), q, s, b, sb, bias, dtype)


@pytest.mark.parametrize("m,n,k,f32", [(2500, 3001, 1040, True), (2500, 3001, 1040, False), (3001, 3001, 1040, False), (65, 5001, 4112, True)])
def test_large_calls(m, n, k, f32):
    """Rows of NaN stay in their rows; transposed scales, another stream and a captured graph give the same bits."""
    a, sa, b, sb = operands(m, n, k, f32, f32)
    want = fp8_matmul(a, sa, b, sb)
    turned = [t.t().contiguous().t() for t in (sa, sb)] if f32 else \
        [t.view(torch.uint8).t().contiguous().t().view(t.dtype) for t in (sa, sb)]
    assert torch.equal(fp8_matmul(a, turned[0], b, turned[1]), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [fp8_matmul(a, sa, b, sb) for _ in range(2)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8_matmul(a, sa, b, sb)
    for seed in range(3):
        new, ns, _, _ = operands(m, 1, k, f32, f32, seed=seed)
        a.copy_(new)
        sa.copy_(ns)
        graph.replay()
        torch.cuda.synchronize()
        kept = y.clone()
        assert torch.equal(kept, fp8_matmul(a, sa, b, sb))
    want = fp8_matmul(a, sa, b, sb)
    a.view(torch.uint8)[[3, m - 1], 5] = 0x7f  # NaN
    got = fp8_matmul(a, sa, b, sb)
    bad = torch.zeros(m, dtype=torch.bool, device=DEV)
    bad[3] = bad[m - 1] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])
