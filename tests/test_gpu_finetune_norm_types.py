"""Layer norm's gradients of weight and bias come in the type that these have."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("kind", ["own", "float32"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_through_differentiation(dtype, kind, weighted):
    """Sums in single precision that are stored with the bias's own bits: up to 500 terms one after the other and in parts, and the rounding
    to the type.  In half precision the features' type could not even hold them: 500 rows of gradients around 1 000."""
    from symmetrix_amd import finetune
    rows, dim = 500, 72
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    dy = (1000 + 100 * torch.randn(rows, dim, generator=g, device="cuda")).to(dtype)
    if kind == "own" and dtype == torch.float16:
        dy = dy / 16
    own = dtype if kind == "own" else torch.float32
    bias = torch.zeros(dim, dtype=own, device="cuda", requires_grad=True)
    weight = torch.ones(dim, dtype=own, device="cuda", requires_grad=True) if weighted else None
    finetune.layer_norm(x, weight, bias).backward(dy)
    unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[own]
    want = dy.double().sum(0)
    assert bias.grad.dtype == own
    assert ((bias.grad.double() - want).abs() <= rows * 2.0 ** -24 * dy.double().abs().sum(0) + unit * (1 + 2.0 ** -8) * want.abs()).all()
    if kind == "float32" and dtype == torch.float16:
        assert (want > 65504).all()
    if weighted:
        assert weight.grad.dtype == own


@pytest.mark.gpu
def test_a_type_that_does_not_fit():
    from symmetrix_amd import finetune
    x = torch.randn(5, 16, device="cuda").bfloat16()
    y, mean, rstd = finetune.layer_norm_forward(x)
    assert finetune.layer_norm_backward(y, x, mean, rstd)[2].dtype == torch.bfloat16
    assert finetune.layer_norm_backward(y, x, mean, rstd, bias_type=torch.float32)[2].dtype == torch.float32
    for weight, kind in ((None, torch.float16), (None, torch.float64), (torch.ones(16, device="cuda"), torch.bfloat16)):
        with pytest.raises(TypeError):
            finetune.layer_norm_backward(y, x, mean, rstd, weight, bias_type=kind)
