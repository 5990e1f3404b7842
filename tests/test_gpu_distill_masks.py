"""distill_loss of logits that hold large finite masks or lie far from zero, against float64 autograd."""
import pytest
import torch

from dsalt.kernels import distill_loss
from test_gpu_distill import BF, DEV, FP, HF, compare, inputs

pytestmark = pytest.mark.gpu

# One wave a row, four, slices of few rows, and lone rows of one workgroup and of slices.
SHAPES = [(5, 600), (1, 600), (600, 4500), (5, 9001), (1, 9001), (1, 70001)]
MASKS = [-1e4, -1e6, -1e9, -1e10, -1e20, -1e30, "half", "lowest"]


def mask_value(mask, dtype):
    lowest = torch.finfo(dtype).min
    return {"half": lowest / 2, "lowest": lowest}.get(mask) if isinstance(mask, str) else max(mask, lowest)


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("dtype,tau,lam", [(FP, 1.0, 0.5), (BF, 2.0, 0.5), (FP, 1.5, 0.25), (BF, 0.5, 0.25), (FP, 2.0, 0.0), (HF, 1.0, 1.0)])
def test_masks(rows, V, mask, dtype, tau, lam):
    """A masked prefix, suffix, middle, every other run of 40, all but one token of a row, and a row that the mask
    leaves nothing of (its softmax is 1 / V): the masked logits have no probability and no gradient beside others."""
    low = mask_value(mask, dtype)
    s, z, ids, y = inputs((rows,), V, 4, dtype, holes=False)
    at = torch.arange(V, device=DEV)
    free = {0: at >= V // 3, 1: at < V // 2, 2: (at < V // 4) | (at >= V // 2), 3: at // 40 % 2 == 1, 4: at == V - 2, 5: at < 0}
    first = MASKS.index(mask) if rows == 1 else 0
    for r in range(min(rows, 13)):
        keep = free[(first + r) % 6]
        s[r, ~keep] = low
        if bool(keep.any()):  # tokens that are masked have an infinite loss: none of them is taught
            live = at[keep]
            ids[r], y[r] = live[ids[r] % live.numel()], live[y[r] % live.numel()]
            if r == 1:
                y[r] = -100
    y[13:] = -100
    _, g = compare(s, z, ids, y, tau=tau, lam=lam)
    for r in range(min(rows, 13)):
        keep = free[(first + r) % 6]
        assert not bool(keep.any()) or not g[r, ~keep].any()


@pytest.mark.parametrize("V", [600, 4500, 9001])
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("tau,lam", [(1.0, 0.5), (1.5, 0.5), (2.0, 0.5)])
def test_two_masks(V, dtype, tau, lam):
    """Rows that hold two masks and nothing else: the softmax is uniform over the larger one's places."""
    s, z, ids, y = inputs((4,), V, 4, dtype, holes=False)
    for r, (a, b) in enumerate(((-1e10, -1e30), (-1e30, -1e10), (-1e5, -1e9), (-1e20, float("-inf")))):
        s[r, ::2], s[r, 1::2] = a, b
    odd = torch.tensor([0, 1, 0, 0], device=DEV)  # where the larger mask lies
    ids, y = (t % (V - 1) // 2 * 2 + odd.view(-1, *[1] * (t.dim() - 1)) for t in (ids, y))
    compare(s, z, ids, y, tau=tau, lam=lam)


@pytest.mark.parametrize("rows,V", SHAPES)
@pytest.mark.parametrize("offset", [1e3, -3e4, 4.6e4, -1e5, 1e6])
@pytest.mark.parametrize("tau,lam", [(1.0, 0.5), (1.5, 0.5), (2.0, 0.5)])
def test_offsets(rows, V, offset, tau, lam):
    """Logits far from zero have the loss of their differences, to the precision of logits around it."""
    s, z, ids, y = inputs((rows,), V, 4, FP, holes=False)
    y[12:] = -100
    compare(s + offset, z, ids, y, tau=tau, lam=lam)


def test_infinite_logits_stay_in_their_rows():
    """+inf has no softmax: its row is NaN, beside rows of large masks."""
    s, z, ids, y = inputs((4,), 5000, 4, FP, holes=False)
    s[0, 7], s[2, 100:] = float("inf"), -1e30
    ids[2], y[2] = ids[2] % 100, y[2] % 100
    leaf = s.requires_grad_()
    rows = distill_loss(leaf, z, ids, y, temperature=2.0, label_weight=0.5, reduction="none")
    g, = torch.autograd.grad(rows.sum(), leaf)
    assert bool(torch.isnan(rows[0])) and bool(torch.isfinite(rows[1:]).all()) and bool(torch.isfinite(g[1:]).all())
