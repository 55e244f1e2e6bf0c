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



def _clip(*tensors):
    """What the C entry point says to (type, gradient, result, numbers); nothing is launched: its workspace is too small."""
    from symmetrix_amd import finetune
    L = finetune._lib_functions()
    pack = b"".join(finetune._GRAD_TENSOR.pack(*t) for t in tensors)
    assert L.smx_clip_grads(pack, len(tensors), 1.0, 4096, 4096, 8, None) == -1
    return L.smx_last_error().decode()


A, B = 1 << 20, 1 << 21


@pytest.mark.parametrize("tensors", [
    [(0, A, A, 10), (0, A, A, 10)],                                    # the same twice
    [(0, A, A, 100), (0, A + 200, A + 200, 100)],                      # ranges that overlap
    [(0, A + 200, A + 200, 100), (1, B, B, 7), (0, A, A, 51)],         # by one number, in any order
    [(1, A, A, 100), (0, A + 196, A + 196, 10)],                       # of other types
    [(0, A, B, 10), (0, B, A, 10)],                                    # one's result is the other's gradient
    [(0, A, A, 10), (0, A, B, 10)],
    [(0, A, B, 1000), (0, B + 3996, B + 8000, 1)],
    [(0, A, A + 4, 10)],                                               # a part of its own gradient
    [(2, A + 2, A, 2)],
], ids=range(9))
def test_results_in_common_memory_are_refused(tensors):
    assert "shares memory" in _clip(*tensors) or "share memory" in _clip(*tensors)


@pytest.mark.parametrize("tensors", [
    [(0, A, A, 50), (0, A + 200, A + 200, 100), (1, A + 600, A + 600, 3)],          # one right behind the other
    [(0, A, B, 50), (0, A + 100, B + 200, 50), (0, A, B + 400, 50)],                # gradients may overlap where they are only read
    [(0, A, A + 40, 10), (0, A - 40, A + 80, 10)],
    [(0, A, A, 0), (0, A, A, 10), (0, A + 8, A + 8, 0)],                            # of no numbers
    [(2, A, A + 4, 2), (2, A + 8, A + 8, 1)],
], ids=range(5))
def test_results_with_memory_of_their_own_are_taken(tensors):
    assert "smx_grad_norm_workspace" in _clip(*tensors)


def test_orders_of_dimensions():
    """Gradients that are clipped in a copy and written back: once each, and no other result in between."""
    from symmetrix_amd import finetune
    t, buf = torch.ones(4, 3).t(), torch.ones(100)
    cols = buf.view(10, 10)[:, :5]
    for grads, out in (([t, t], None), ([t, t.t().t()], None), ([t, torch.ones(2)], [t, t.t()[0][:2]]), ([t, t], [t, t]),
                       ([cols, torch.ones(7)], [cols, buf[3:10]])):
        with pytest.raises(ValueError, match="memory of its own"):
            finetune.clip_grads(grads, 1.0, out=out)
    assert buf.eq(1).all() and t.eq(1).all()


@pytest.mark.gpu
def test_refused_before_anything_is_written():
    from symmetrix_amd import finetune
    buf, other = torch.ones(1000, device="cuda"), torch.full((500,), 2.0, device="cuda")
    a, b = buf[:500], buf[500:]
    for grads, out in (([buf[:600], buf[400:]], None), ([a, b], [b, a]), ([a, other], [a, buf[499:999]]), ([a], [buf[1:501]]), ([a, a], [a, other])):
        with pytest.raises(ValueError):
            finetune.clip_grads(grads, 1.0, out=out)
    assert buf.eq(1).all() and other.eq(2).all()
    # columns of one array, and gradients that share memory where others are written
    cols = [buf.view(20, 50)[:, :30], buf.view(20, 50)[:, 30:]]
    finetune.clip_grads(cols, 0.5 * math.sqrt(1000))
    assert buf.eq(0.5).all()
    out = [torch.empty(600, device="cuda"), torch.empty(600, device="cuda")]
    norm = finetune.clip_grads([buf[:600], buf[400:]], 1.0, out=out)
    assert abs(float(norm) - math.sqrt(300)) <= 2.0 ** -23 * math.sqrt(300) and torch.equal(out[0], out[1]) and buf.eq(0.5).all()


@pytest.mark.gpu
def test_gradients_that_hang_on_a_graph():
    """Recorded gradients (create_graph) and tensors that require gradients are clipped too, in any order of dimensions; nothing is recorded."""
    from symmetrix_amd import finetune
    for turn in (False, True):
        make = lambda: _turned(40, 30) if turn else _turned(40, 30).contiguous()          # noqa: E731
        want = make()
        norm = finetune.clip_grads(want, 3.0)
        leaf = make().requires_grad_()
        x = torch.ones_like(leaf, requires_grad=True)
        recorded, = torch.autograd.grad((x * x * leaf).sum() * 0.5, x, create_graph=True)
        recorded = recorded if recorded.is_contiguous() != turn else recorded.t().contiguous().t()
        assert recorded.requires_grad
        for g in (leaf, recorded):
            version, node = g._version, g.grad_fn
            assert torch.equal(finetune.clip_grads([g], 3.0), norm)
            assert torch.equal(g.detach(), want) and g._version > version and g.requires_grad and g.grad_fn is node
