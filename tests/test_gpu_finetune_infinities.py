"""Adapters: infinities are where the definition has them, whatever way a size goes."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_finetune_adapters import NAMES, _close, _data, _reference  # noqa: E402


def _compare(got, want, off, dtype):
    """Infinities and NaN as in 64 bits, everything else as close as always."""
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)].double(), want[torch.isinf(want)])
    zero = torch.zeros_like(want)
    _close(torch.where(finite, got.double(), zero).to(dtype), torch.where(finite, want, zero), torch.where(finite, off, zero), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("rows,d_in,d_out", [(24, 160, 96), (100, 160, 96), (100, 1024, 96), (700, 160, 320), (5000, 160, 1056), (8500, 96, 2080)])
@pytest.mark.parametrize("rank", [1, 8, 12, 40])
def test_positive_factors(rank, rows, d_in, d_out, dtype):
    """With nothing but positive numbers a sum that an infinity is in is infinite, and no product of it is with zero."""
    from symmetrix_amd import finetune
    t = NAMES[dtype]
    data, dy = _data(rows, d_in, d_out, rank, 4, t, "runs")
    for k in ("x", "weight", "A", "B"):
        data[k] = (data[k].abs() + 0.01).to(t)
    dy = (dy.abs() + 0.01).to(t)
    data["index"][rows // 2:rows // 2 + 9] = 2          # (an adapter that occurs, beside others)
    data["index"][rows // 2 + 9] = 1
    inf = float("inf")
    for name, place in (("B", (2, 5, rank - 1)), ("A", (2, 0, 3)), ("x", (rows // 2 + 1, 7)), ("B", (2,))):
        broken = dict(data)
        broken[name] = data[name].clone()
        broken[name][place] = -inf if place == (2,) else inf
        ref = _reference(**broken)["y"]
        assert torch.isinf(ref[0]).any() and not torch.isnan(ref[0]).any()
        _compare(finetune.adapted_linear_forward(**broken), *ref, t)
        if name != "x":
            dx = finetune.adapted_linear_backward(dy, **broken, need=(True, False, False))[0]
            _compare(dx, *_reference(**broken, dy=dy)["dx"], t)
    dy[rows // 2 + 1, 3] = inf
    _compare(finetune.adapted_linear_backward(dy, **data, need=(True, False, False))[0], *_reference(**data, dy=dy)["dx"], t)
