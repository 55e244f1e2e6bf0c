"""Tensors without a last dimension, or with one of no numbers, are refused as other wrong shapes are."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_finetune_adapters import _data  # noqa: E402


@pytest.mark.gpu
def test_no_rows_to_speak_of():
    from symmetrix_amd import finetune
    one = torch.tensor(1.0, device="cuda")
    data, dy = _data(6, 32, 48, 4, 3, torch.float32)
    flat = torch.zeros(2, 3, 0, device="cuda")
    stats = torch.zeros(2, 3, device="cuda")
    for call in (lambda: finetune.layer_norm_forward(one), lambda: finetune.layer_norm_backward(one, one, one, one), lambda: finetune.layer_norm(one),
                 lambda: finetune.layer_norm_forward(flat), lambda: finetune.layer_norm_backward(flat, flat, stats, stats),
                 lambda: finetune.adapted_linear_forward(**dict(data, x=one)), lambda: finetune.adapted_linear(**dict(data, x=one)),
                 lambda: finetune.adapted_linear_backward(dy, **dict(data, x=one)), lambda: finetune.adapted_linear_forward(**dict(data, x=flat))):
        with pytest.raises(ValueError):
            call()
    # a row by itself is one
    row = dict(data, x=data["x"][0], index=data["index"][0])
    assert torch.equal(finetune.adapted_linear_forward(**row), finetune.adapted_linear_forward(**dict(data, x=data["x"][:1], index=data["index"][:1]))[0])
    y, mean, rstd = finetune.layer_norm_forward(data["x"][0])
    assert y.shape == (32,) and mean.shape == rstd.shape == ()
    assert finetune.layer_norm_backward(y, data["x"][0], mean, rstd)[0].shape == (32,)
