"""A projection that belongs to a module is served as it is."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_finetune_adapters import _data  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_parameters_without_gradients_recorded(mode):
    from symmetrix_amd import finetune
    data, _ = _data(30, 96, 64, 8, 5, torch.float32)
    want = finetune.adapted_linear_forward(**data)
    linear = torch.nn.Linear(96, 64, bias=False, device="cuda")
    linear.weight.data.copy_(data["weight"])
    scale = torch.nn.Parameter(data["scale"].clone())
    with mode():
        got = finetune.adapted_linear(**dict(data, weight=linear.weight, scale=scale))
    assert torch.equal(got, want) and not got.requires_grad
    for k, v in (("weight", linear.weight), ("scale", scale)):
        with pytest.raises(ValueError):
            finetune.adapted_linear(**dict(data, **{k: v}))
