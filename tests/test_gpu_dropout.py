"""counter_dropout against numpy's unsigned integer arithmetic: the mask to the bit, values to
their one rounding, and its gradient, seeds, offsets and replays."""
import numpy as np
import pytest
import torch

from dsalt import _hip
from dsalt.kernels import counter_dropout
from philox_reference import keep_mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def want(x, p, seed, offset):
    """One fp32 product of x and the fp32 scale, rounded to the dtype."""
    t = _hip.keep_threshold(p)
    keep = torch.from_numpy(keep_mask(x.numel(), p, seed, offset)).view(x.shape).to(x.device)
    return torch.where(keep, x.float() * np.float32(65536.0 / max(t, 1)).item(), 0.0).to(x.dtype)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n", [1, 3, 7, 8, 9, 63, 64, 2047, 2048, 100003, 5000011])
def test_values(n, dtype):
    print(f"dropout {n} {dtype}", flush=True)
    x = torch.randn(n, device=DEV, generator=torch.Generator(DEV).manual_seed(n)).to(dtype)
    for p, seed, offset in ((0.1, 7, 0), (0.5, -(2 ** 63), 1), (0.97, 2 ** 64 - 1, 2 ** 63 - 1), (0.0, 5, 3), (1.0, 5, 3),
                            (2.0 ** -17, 1, 0), (1 - 2.0 ** -16, 1, 2 ** 32)):
        assert torch.equal(counter_dropout(x, p, seed, offset), want(x, p, seed, offset)), (p, seed, offset)


def test_offsets_past_32_bits():
    """More than 2^32 elements: pieces on both sides of 2^31 and 2^32, and the odd end."""
    n = 2 ** 32 + 2 ** 20 + 5
    print(f"dropout {n}", flush=True)
    y = counter_dropout(torch.ones(n, device=DEV, dtype=BF), 0.25, 11, 3)
    for at, size in ((0, 4096), (2 ** 31 - 2048, 4096), (2 ** 32 - 2048, 4096), (2 ** 32 + 2 ** 20 - 2043, 2048)):
        first = at // 8 * 8
        keep = keep_mask(at + size - first, 0.25, 11, 3, first // 8)[at - first:]
        want = torch.from_numpy(keep).to(DEV).to(BF) * (1 / 0.75)
        assert torch.equal(y[at:at + size], want.to(BF)), at
    assert y[at + size:].numel() == 0


def test_gradient_is_the_same_mask():
    x = torch.randn(33, 77, device=DEV, requires_grad=True)
    dy = torch.randn(33, 77, device=DEV)
    y = counter_dropout(x, 0.3, 11, 4)
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, want(dy, 0.3, 11, 4))
    # a graph of the backward: linear, so the second gradient is the mask again
    up = dy.clone().requires_grad_()
    g, = torch.autograd.grad(counter_dropout(x, 0.3, 11, 4), x, up, create_graph=True)
    assert torch.equal(torch.autograd.grad(g, up, torch.ones_like(g))[0], want(torch.ones_like(dy), 0.3, 11, 4))
    # expanded gradients
    assert torch.equal(torch.autograd.grad(counter_dropout(x, 0.3, 11, 4).sum(), x)[0], want(torch.ones_like(dy), 0.3, 11, 4))


def test_logical_order_and_alignment():
    """The mask belongs to the element's place in the tensor, not to its address."""
    base = torch.randn(64 * 50 + 5, device=DEV).to(BF)
    for view in (base[1:1 + 64 * 50].view(64, 50), base[:64 * 50].view(50, 64).t(), base[:64 * 50].view(64, 50)[:, ::2],
                 base[:50].expand(3, 50), base[:1].view(()), base[:0]):
        got = counter_dropout(view, 0.25, 3)
        assert got.shape == view.shape and got.is_contiguous()
        assert torch.equal(got, want(view.contiguous(), 0.25, 3, 0))


def test_dropped_infinities_are_zero():
    x = torch.full((4096,), float("inf"), device=DEV)
    x[::3] = float("nan")
    y = counter_dropout(x, 0.5, 1)
    keep = torch.from_numpy(keep_mask(4096, 0.5, 1, 0)).to(DEV)
    assert bool((y[~keep] == 0).all()) and not bool(y[keep].isfinite().any())


def test_kept_share_and_scale():
    """The kept share is binomial: within 6 standard deviations of 1 - p (2^-17 more for p's own
    rounding), and different seeds, offsets and halves agree no more than chance."""
    n, p = 1 << 22, 0.1
    one = torch.ones(n, device=DEV)
    a, b, c = (counter_dropout(one, p, s, o) != 0 for s, o in ((1, 0), (2, 0), (1, 1)))
    sd = (p * (1 - p) / n) ** 0.5
    for m in (a, b, c):
        assert abs(float(m.double().mean()) - (1 - p)) <= 6 * sd + 2.0 ** -17
    both = (1 - p) ** 2
    for m, k in ((a, b), (a, c), (a[1:], a[:-1]), (a[8:], a[:-8])):
        assert abs(float((m & k).double().mean()) - both) <= 6 * (2 * both * (1 - both) / n) ** 0.5 + 2.0 ** -15


def test_seed_tensor_streams_and_graph():
    x = torch.randn(3001, device=DEV).to(HF).requires_grad_()
    dy = torch.randn(3001, device=DEV).to(HF)
    seed = torch.tensor([-5], device=DEV)
    assert torch.equal(counter_dropout(x, 0.2, seed, 9), want(x, 0.2, -5, 9))
    y = counter_dropout(x, 0.2, seed, 9)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, x, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = counter_dropout(x, 0.2, seed)
        torch.autograd.grad(y, x, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want(x, 0.2, -4, 0))
    # a leaf of its own: torch cannot capture a backward to a leaf that an eager graph still holds
    x = x.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = counter_dropout(x, 0.2, seed)
        dx, = torch.autograd.grad(y, x, dy)
    for s in (3, 2 ** 62, -1):  # each replay takes the seed that is there
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want(x, 0.2, s, 0)) and torch.equal(dx, want(dy, 0.2, s, 0))
        counter_dropout(x, 0.4, 1)


def test_refusals_on_gpu():
    x = torch.randn(16, device=DEV)
    for seed in (torch.tensor([1]), torch.tensor([1.0], device=DEV), torch.tensor([1, 2], device=DEV)):
        with pytest.raises(_hip.DsaltError):
            counter_dropout(x, 0.1, seed)
    for bad in (x.double(), x.int()):
        with pytest.raises(_hip.DsaltError):
            counter_dropout(bad, 0.1, 1)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            counter_dropout(x, p, 1)
    for seed, offset in ((None, 0), (2 ** 64, 0), (-2 ** 63 - 1, 0), (1, -1), (1, 2 ** 63)):
        with pytest.raises(ValueError):
            counter_dropout(x, 0.1, seed, offset)


def test_scalars_and_no_elements():
    x = torch.full((), 2.0, device=DEV)
    assert torch.equal(counter_dropout(x, 0.5, 3), want(x, 0.5, 3, 0)) and counter_dropout(x, 0.5, 3).shape == ()
    empty = torch.zeros(4, 0, 8, device=DEV, dtype=BF, requires_grad=True)
    y = counter_dropout(empty, 0.5, 3)
    g, = torch.autograd.grad(y, empty, torch.zeros_like(y))
    assert y.shape == g.shape == (4, 0, 8)


def test_numpy_seeds_and_offsets():
    x = torch.randn(100, device=DEV, requires_grad=True)
    for seed, offset in ((np.int64(-7), np.int32(3)), (np.uint64(2 ** 64 - 7), np.int64(3))):
        y = counter_dropout(x, 0.4, seed, offset)
        assert torch.equal(y, want(x, 0.4, -7, 3)) and torch.equal(torch.autograd.grad(y, x, x)[0], y)


class Tagged(torch.Tensor):
    """A tensor subclass with nothing of its own."""


def test_transforms_tracing_and_subclasses():
    """What an autograd function with a HIP kernel does not know runs as torch's ops, with the same bits."""
    x, up = torch.randn(6, 50, device=DEV), torch.randn(6, 50, device=DEV)
    seed = torch.tensor([21], device=DEV)
    for s in (21, seed):
        drop = lambda t: counter_dropout(t, 0.3, s, 4)
        mask, each = want(torch.ones_like(x), 0.3, 21, 4), want(torch.ones(50, device=DEV), 0.3, 21, 4)
        assert torch.equal(torch.func.grad(lambda t: (drop(t) * up).sum())(x), want(up, 0.3, 21, 4))
        assert torch.equal(torch.func.jvp(drop, (x,), (up,))[1], mask * up)
        assert torch.equal(torch.func.vmap(drop)(x), x * each)
        with torch.no_grad():
            assert torch.equal(torch.func.vmap(drop)(x), x * each)
        traced = torch.jit.trace(drop, (x,))
        assert torch.equal(traced(up), up * mask)
        got = drop(x.as_subclass(Tagged))
        assert type(got) is Tagged and torch.equal(got.as_subclass(torch.Tensor), x * mask)
    seeds = torch.arange(6, device=DEV)[:, None]
    got = torch.func.vmap(lambda t, s: counter_dropout(t, 0.3, s, 4))(x, seeds)
    assert torch.equal(got, torch.stack([want(x[i], 0.3, i, 4) for i in range(6)]))


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n", [5, 8, 4099, 5000011])
def test_entry_in_place(n, dtype):
    """The C entry takes out = x."""
    x = torch.randn(n, device=DEV).to(dtype)
    ref = want(x, 0.3, 9, 1)
    _hip._call("dsalt_dropout", _hip._DROPOUT_PACK.pack(n, _hip._SCORE_DTYPES[dtype], _hip.keep_threshold(0.3), x.data_ptr(),
                                                        x.data_ptr(), 9, 1, 0), x.device)
    assert torch.equal(x, ref)
