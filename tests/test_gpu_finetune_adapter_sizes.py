"""Adapters beside a shared projection at the ends of what the entry points take: very wide results of few rows, many rows of few numbers."""
import itertools

import pytest

torch = pytest.importorskip("torch")

from test_gpu_finetune_adapters import NAMES, _close, _data, _reference  # noqa: E402

HBM = 288e9


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("kind", [0, 1, 2], ids=["float32", "bfloat16", "float16"])
def test_wide_results_have_launches(kind, backward):
    """The sizes of a call's launches are looked at where its workspace is counted: one without blocks is refused there."""
    from symmetrix_amd import finetune
    for rows in (65, 96, 100, 128, 129, 200, 255, 256, 257, 300, 511, 513, 700, 8500):
        for wide in [*range(4096, 1 << 20, 4099), 65536, 70000, 98304, 151936, 1 << 20]:
            d_in, d_out = (wide, 40) if backward else (40, wide)
            finetune._adapted_workspace.__wrapped__((kind, d_in, d_out, 8, 5, rows, d_in, d_in), backward)


@pytest.mark.parametrize("kind", [0, 1, 2], ids=["float32", "bfloat16", "float16"])
def test_every_size_has_launches(kind):
    """No size inside the documented limits that fits the memory is refused."""
    from symmetrix_amd import finetune
    rows_of = [1, 2, 63, 64, 65, 96, 100, 128, 129, 200, 255, 256, 257, 300, 511, 513, 700, 1000, 1537, 4091, 8179, 8500, 70001, 1 << 20, 1 << 24, 1 << 28]
    widths = [1, 31, 32, 96, 1000, 4096, 4097, 32768, 65536, 65537, 65792, 70000, 98304, 131073, 151936, 200000, 1 << 19, (1 << 20) - 1, 1 << 20]
    seen = 0
    for rows, d_in, d_out in itertools.product(rows_of, widths, widths):
        size = 4 if kind == 0 else 2
        if size * (rows * (d_in + d_out) + d_in * d_out) > HBM:
            continue
        for rank, adapters in ((8, 3), (64, 0), (128, 40), (1, 4096)):
            for backward in (0, 1):
                if 4 * rows * rank + size * (rows * (d_in + d_out) * (1 + backward) + d_in * d_out + adapters * rank * (d_in + d_out)) > HBM:
                    continue
                finetune._adapted_workspace.__wrapped__((kind, d_in, d_out, rank, adapters, rows, d_in, d_in), backward)
                seen += 1
    assert seen > 10000


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("rows,wide", [(100, 70000), (100, 151936), (128, 131100), (200, 65792), (300, 70000), (65, 98303)])
def test_few_rows_of_very_wide_results(rows, wide, dtype):
    """More tiles of columns than the chip works on at once, in one row of tiles or two: as results, and as the gradient of x."""
    from symmetrix_amd import finetune
    data, dy = _data(rows, 40, wide, 8, 5, NAMES[dtype], "mixed", seed=rows)
    _close(finetune.adapted_linear_forward(**data), *_reference(**data)["y"], NAMES[dtype])
    data, dy = _data(rows, wide, 40, 8, 5, NAMES[dtype], "mixed", seed=rows)
    dx = finetune.adapted_linear_backward(dy, **data, need=(True, False, False))[0]
    _close(dx, *_reference(**data, dy=dy)["dx"], NAMES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_more_blocks_than_a_launch_takes(dtype):
    """2^26 rows and some: h in two launches.  4 096 adapters of 65 600 numbers: their layout for the gradient in three."""
    from symmetrix_amd import finetune
    rows = (1 << 26) + 77
    data, _ = _data(400, 3, 5, 2, 3, NAMES[dtype], "mixed")
    some = torch.cat([torch.arange(100), torch.arange(rows - 300, rows)]).cuda()
    x, index = torch.zeros(rows, 3, dtype=NAMES[dtype], device="cuda"), torch.ones(rows, dtype=torch.int32, device="cuda")
    x[some], index[some] = data["x"], data["index"]
    y = finetune.adapted_linear_forward(**dict(data, x=x, index=index))
    _close(y[some], *_reference(**data)["y"], NAMES[dtype])
    assert (y[100:rows - 300] == 0).all()
    data, dy = _data(70, 33, 65600, 1, 4096, NAMES[dtype], "own")
    dx = finetune.adapted_linear_backward(dy, **data, need=(True, False, False))[0]
    _close(dx, *_reference(**data, dy=dy)["dx"], NAMES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_as_far_apart_as_a_tile_takes_them(dtype):
    """2^22 numbers from row to row: offsets inside a tile of 256 rows pass 2^31 bytes, of x and of the projection."""
    from symmetrix_amd import finetune
    stride = 1 << 22
    store = torch.empty(255 * stride + 64, dtype=dtype, device="cuda")
    far = store.as_strided((256, 64), (stride, 1))
    data, _ = _data(256, 64, 49152, 8, 3, dtype, "own")
    far.copy_(data["x"])
    _close(finetune.adapted_linear_forward(**dict(data, x=far)), *_reference(**data)["y"], dtype)
    data, _ = _data(49152, 64, 256, 8, 3, dtype)
    far.copy_(data["weight"])
    _close(finetune.adapted_linear_forward(**dict(data, weight=far)), *_reference(**data)["y"], dtype)
