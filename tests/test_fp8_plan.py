"""The plan of an 8-bit product (no GPU): its values and refusals."""
import pytest

import dsalt._hip as hip


def test_plans_hold_their_sizes():
    """Tiles that exist, splits that leave no part of k empty, the workspace that the parts need."""
    for e8m0 in (False, True):
        for m in (1, 16, 17, 32, 33, 64, 300, 2500, 4100, 1 << 20):
            for n in (1, 101, 1024, 15360, 30720, 11008):
                for k in (16, 128, 272, 2064, 16400):
                    rows, columns, splits = hip.fp8_plan(m, n, k, e8m0)
                    if m <= hip.FP8_FEW_ROWS:
                        assert rows == (16 if m <= 16 else 32) and columns in (16, 32, 64) and splits == 1
                        continue
                    assert (rows, columns) in ((64, 128), (128, 128)) or (e8m0 and (rows, columns) == (256, 256))
                    blocks = -(-k // 128)
                    assert 1 <= splits <= min(16, blocks) and -(-blocks // -(-blocks // splits)) == splits
                    assert splits == 1 or rows == 64
                    need = hip.lib().dsalt_fp8_matmul_workspace_size(m, n, k)
                    assert need >= (splits * m * n * 4 if splits > 1 else 0)


@pytest.mark.parametrize("size", [(0, 64, 128), (1 << 25, 64, 128), (64, 0, 128), (64, 1 << 21, 128), (64, 64, 0), (64, 64, 1 << 21)])
def test_sizes_that_no_product_has(size):
    with pytest.raises(hip.DsaltError, match="sizes"):
        hip.fp8_plan(*size, True)
    assert hip.lib().dsalt_fp8_matmul_plan(64, 64, 128, 1, None) == 1
