"""Adapters beside a shared projection at the ends of what the entry points take: very wide results of few rows, many rows of few numbers."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_finetune_adapters import NAMES, _close, _data, _reference  # noqa: E402


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("kind", [0, 1, 2], ids=["float32", "bfloat16", "float16"])
def test_wide_results_have_launches(kind, backward):
    """The sizes of a call's launches are looked at where its workspace is counted: one without blocks is refused there."""
    from symmetrix_amd import finetune
    for rows in (65, 96, 100, 128, 129, 200, 255, 256, 257, 300, 511, 513, 700, 8500):
        for wide in [*range(4096, 1 << 20, 4099), 65536, 70000, 98304, 151936, 1 << 20]:
            d_in, d_out = (wide, 40) if backward else (40, wide)
            finetune._adapted_workspace.__wrapped__((kind, d_in, d_out, 8, 5, rows, d_in, d_in), backward)


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
