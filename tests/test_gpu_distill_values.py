"""distill_loss at the ends of what its operands hold: teachers of the types' lowest and largest values."""
import pytest
import torch

from test_gpu_distill import BF, FP, HF, compare, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [600, 9001])
@pytest.mark.parametrize("t_dtype", [FP, BF, HF])
@pytest.mark.parametrize("tau,lam", [(0.25, 0.5), (0.9, 0.0), (1.0, 0.5), (2.0, 0.5)])
def test_teacher_of_extreme_values(V, t_dtype, tau, lam):
    """Slots of the type's lowest value beside others have no share; where all are alike, each has 1 / K, also where
    the value over the temperature is past fp32's range."""
    s, z, ids, y = inputs((6,), V, 70, t_dtype=t_dtype, holes=False)
    y[1] = 3
    top = torch.finfo(t_dtype).max
    z[0, ::3], z[1], z[2], z[3] = -top, -top, -top / 2, top
    z[4, :35], z[4, 35:] = -top, float("-inf")
    z[5, 1:] = -top
    compare(s, z, ids, y, tau=tau, lam=lam)
