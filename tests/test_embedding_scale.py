"""Scales that single precision does not have: tables' entry points refuse them, instead of making zeros NaN or numbers zeros."""
import math

import pytest

torch = pytest.importorskip("torch")

WRONG = [math.inf, -math.inf, math.nan, 1e39, -1e300, 1e-39, -1e-300]
RIGHT = [0.0, -0.0, 1.0, -3.4028234663852886e38, 2.0 ** -126]


def test_entry_points():
    from symmetrix_amd import finetune
    L = finetune._lib_functions()
    for scale in WRONG:
        assert L.smx_embedding_forward(0, 0, 5, 8, None, 8, None, scale, None, 8, None) == -1 and "scale" in L.smx_last_error().decode()
        assert L.smx_embedding_backward(0, 10, 0, 8, None, 8, None, None, None, scale, None, None, 0, None) == -1 and "scale" in L.smx_last_error().decode()
    for scale in RIGHT:          # (no rows, no entries: nothing to do)
        assert L.smx_embedding_forward(0, 0, 5, 8, None, 8, None, scale, None, 8, None) == 0
        assert L.smx_embedding_backward(0, 10, 0, 8, None, 8, None, None, None, scale, None, None, 0, None) == 0


@pytest.mark.gpu
def test_scales():
    from symmetrix_amd import finetune
    table = torch.tensor([[0.0, 1.0, -0.5, 2.0 ** -10]], device="cuda")
    index = torch.zeros(3, dtype=torch.int32, device="cuda")
    for scale in RIGHT:
        want = (table.double() * scale).float().expand(3, 4)
        assert torch.equal(finetune.embedding_forward(table, index, scale), want)
        # (three equal rows: their sum is exact, and the product is rounded once)
        dy = table.expand(3, 4)
        assert torch.equal(finetune.embedding_backward(dy, index, 1, scale), (3 * table.double() * scale).float())
    for scale in WRONG:
        with pytest.raises(ValueError):
            finetune.embedding_forward(table, index, scale)
        with pytest.raises(ValueError):
            finetune.embedding_backward(table, index[:1], 1, scale)
