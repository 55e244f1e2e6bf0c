"""Clipping and the memory of what is written: gradients given as their own results, orders of dimensions."""
import math

import pytest

torch = pytest.importorskip("torch")


def _turned(*shape, seed=0):
    """Numbers whose dimensions lie in the other order."""
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").t()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_gradients_as_their_own_results(dtype):
    """out=grads is clipping in place, whatever the order of the dimensions is."""
    from symmetrix_amd import finetune
    make = lambda: [_turned(40, 30).to(getattr(torch, dtype)), None, _turned(7, 5, seed=1).contiguous(), _turned(300, 200, seed=2)[:, ::2]]          # noqa: E731
    want, mine, alone = make(), make(), make()[0]
    norm = finetune.clip_grads(want, 3.0)          # (in place)
    true = math.sqrt(math.fsum(float(g.double().square().sum()) for g in make() if g is not None))
    assert abs(float(norm) - true) <= 2.0 ** -23 * true and true > 6.0
    for g, b in zip(want, make()):
        assert g is None or not torch.equal(g, b)
    versions = [g._version for g in mine if g is not None]
    assert torch.equal(finetune.clip_grads(mine, 3.0, out=mine), norm)
    assert all(a is None or torch.equal(a, b) for a, b in zip(mine, want))
    assert all(g._version > v for g, v in zip([g for g in mine if g is not None], versions))
    # one tensor, and some in place beside others that are not
    plain = torch.empty_like(alone, memory_format=torch.contiguous_format)
    norm = finetune.clip_grads([alone], 3.0, out=[plain])
    assert torch.equal(finetune.clip_grads(alone, 3.0, out=alone), norm) and torch.equal(alone, plain)
    mine, out = make(), make()
    out[0], out[3] = mine[0], torch.empty_like(mine[3], memory_format=torch.contiguous_format)
    out[2].zero_()
    finetune.clip_grads(mine, 3.0, out=out)
    assert all(a is None or torch.equal(a, b) for a, b in zip(out, want))
    assert torch.equal(mine[2], make()[2]) and torch.equal(mine[3], make()[3])

