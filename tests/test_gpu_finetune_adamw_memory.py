"""AdamW works on what its parameters, moments and masters hold when a step is taken: memory that was replaced since the optimizer was made
is used or refused, and memory that was let go is not written."""
import pytest

torch = pytest.importorskip("torch")

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [300, 7, 5000]


def _tensors(dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, generator=g, device="cuda").to(dtype) for n in SIZES]


def _copies(states):
    return [tuple(t.clone() for t in s) for s in states]


def _ahead(bits, dtype=torch.float32, masters=None):
    """An optimizer after two steps."""
    opt = __import__("symmetrix_amd.finetune", fromlist=["AdamW"]).AdamW(_tensors(dtype), state_bits=bits, masters=masters, **HYPER)
    for t in (1, 2):
        opt.step(_tensors(dtype, seed=t))
    return opt


def _same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_assigned_moments_are_the_ones_that_are_used(bits):
    from symmetrix_amd import finetune
    saved = _ahead(bits).states
    opt = finetune.AdamW(_tensors(seed=5), state_bits=bits, step=2, **HYPER)
    first = opt.states
    untouched = _copies(first)
    opt.states = _copies(saved)
    ref = finetune.AdamW(_tensors(seed=5), state_bits=bits, states=_copies(saved), step=2, **HYPER)
    for t in (3, 4):
        opt.step(_tensors(seed=t))
        ref.step(_tensors(seed=t))
    assert _same(opt.params, ref.params)
    assert all(_same(s, r) for s, r in zip(opt.states, ref.states))
    assert all(_same(s, r) for s, r in zip(first, untouched))          # those of before are nobody's any more
    # one by one they cannot be replaced unnoticed, and what does not fit is refused and changes nothing
    with pytest.raises(TypeError):
        opt.states[0] = ref.states[0]
    kept = opt.states
    for wrong in (ref.states[:2], [s[:1] for s in ref.states], [tuple(t[:3] for t in s) for s in ref.states],
                  [tuple(t.cpu() for t in s) for s in ref.states], [tuple(t.half() for t in s) for s in ref.states]):
        with pytest.raises(ValueError):
            opt.states = wrong
        assert opt.states is kept


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_moment_with_other_memory(bits):
    """Given other numbers through .data, in step; given fewer, refused."""
    from symmetrix_amd import finetune
    opt = _ahead(bits)
    saved = _copies(opt.states)
    ref = finetune.AdamW([p.clone() for p in opt.params], state_bits=bits, states=_copies(saved), step=2, **HYPER)
    for t in opt.states[2]:
        t.data = t.data.clone()
    opt.step(_tensors(seed=3))
    ref.step(_tensors(seed=3))
    assert _same(opt.params, ref.params) and all(_same(s, r) for s, r in zip(opt.states, ref.states))
    before = [p.clone() for p in opt.params]
    opt.states[2][0].data = opt.states[2][0].data[:100].clone()
    with pytest.raises(ValueError):
        opt.step(_tensors(seed=4))
    assert _same(opt.params, before) and opt.step_count == 3


@pytest.mark.gpu
def test_assigned_masters_are_the_ones_that_are_used():
    from symmetrix_amd import finetune
    opt = _ahead(32, torch.bfloat16, masters=True)
    first = opt.masters
    untouched = [m.clone() for m in first]
    opt.masters = [m + 1 for m in first]
    ref = finetune.AdamW([p.clone() for p in opt.params], masters=[m + 1 for m in first], states=_copies(opt.states), step=2, **HYPER)
    opt.step(_tensors(torch.bfloat16, seed=3))
    ref.step(_tensors(torch.bfloat16, seed=3))
    assert _same(opt.masters, ref.masters) and _same(opt.params, ref.params) and _same(first, untouched)
    opt.masters[0].data = opt.masters[0].data.clone()
    opt.step(_tensors(torch.bfloat16, seed=4))
    ref.step(_tensors(torch.bfloat16, seed=4))
    assert _same(opt.masters, ref.masters) and _same(opt.params, ref.params)
    for wrong in (list(opt.masters)[:2], [m.half() for m in opt.masters], [m[:3] for m in opt.masters], [m.cpu() for m in opt.masters]):
        with pytest.raises(ValueError):
            opt.masters = wrong


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_with_other_memory(bits):
    from symmetrix_amd import finetune
    opt = _ahead(bits)
    ref = finetune.AdamW([p.clone() for p in opt.params], state_bits=bits, states=_copies(opt.states), step=2, **HYPER)
    opt.params[0].data = opt.params[0].data.clone()          # as moving a model there and back does
    opt.step(_tensors(seed=3))
    ref.step(_tensors(seed=3))
    assert _same(opt.params, ref.params)
    good = opt.params[2].data
    before = [p.clone() for p in opt.params]
    for kind, other in ((ValueError, good[:100].clone()), (ValueError, good.cpu()), (TypeError, good.half()), (ValueError, torch.zeros(2 * 5000, device="cuda")[::2]),
                        (ValueError, good.view(50, 100))):
        opt.params[2].data = other
        for grads in (_tensors(seed=4), [None, None, torch.zeros_like(other)]):
            with pytest.raises((kind, ValueError) if other.device.type == "cpu" else kind):
                opt.step(grads)
    opt.params[2].data = good
    assert _same(opt.params, before) and opt.step_count == 3


@pytest.mark.gpu
def test_the_kind_of_moments_stays():
    opt = _ahead(8)
    with pytest.raises(AttributeError):
        opt.state_bits = 32
    assert opt.state_bits == 8


@pytest.mark.gpu
def test_memory_named_twice_is_refused():
    """A step goes over all tensors at once."""
    from symmetrix_amd import finetune
    p = _tensors()
    zeros = lambda: [(torch.zeros_like(t), torch.zeros_like(t)) for t in p]          # noqa: E731
    shared, both = zeros(), zeros()
    shared[1] = (shared[1][0], shared[1][0])
    both[1] = (both[0][0][:7], both[1][1])
    half = [t.half() for t in p]
    for call in (lambda: finetune.AdamW([p[0], p[1], p[0]]), lambda: finetune.AdamW([p[0], p[0][:10]]), lambda: finetune.AdamW(p, states=shared),
                 lambda: finetune.AdamW(p, states=both), lambda: finetune.AdamW([half[1], half[1].clone()], masters=[p[1], p[1]])):
        with pytest.raises(ValueError, match="memory of its own"):
            call()
    empty = torch.zeros(0, device="cuda")
    finetune.AdamW([p[0], empty, empty]).step([p[1].new_ones(300), empty, empty])
