"""Adapters beside a shared projection: products of so many rows and columns that every way of tiling them takes its part, with sums of
many steps, odd numbers of them among these."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_finetune_adapters import NAMES, _close, _data, _reference  # noqa: E402

# Tiles of 256 x 256, 192 of them or more: 306 (28 rows of tiles at once and the rest in small ones), 216 in one launch, 355 (the rest in 351 tiles of
# 128 x 128), 576 with columns that end inside a tile.
SIZES = [(8500, 1056, 2080, 32, 24), (6000, 2080, 2080, 8, 3), (18000, 992, 1056, 16, 40), (8185, 1055, 4607, 64, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("order", ["runs", "own"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(size, order, dtype):
    from symmetrix_amd import finetune
    data, _ = _data(*size, NAMES[dtype], order)
    _close(finetune.adapted_linear_forward(**data), *_reference(**data)["y"], NAMES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gradient(size, dtype):
    from symmetrix_amd import finetune
    rows, d_out, d_in, rank, adapters = size
    data, dy = _data(rows, d_in, d_out, rank, adapters, NAMES[dtype])
    got = dict(zip(("dx", "dA", "dB"), finetune.adapted_linear_backward(dy, **data)))
    for k, (want, off) in _reference(**data, dy=dy).items():
        _close(got[k], want, off, NAMES[dtype])
