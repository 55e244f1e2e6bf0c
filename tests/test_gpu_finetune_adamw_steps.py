"""A parameter's steps are those that it had a gradient in: its corrections by 1 - beta^t, and the places where its codes are rounded, go by them."""
import pytest

torch = pytest.importorskip("torch")

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [300, 7, 5000, 256]


def _tensors(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, generator=g, device="cuda") for n in SIZES]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_come_and_go(bits):
    from symmetrix_amd import finetune
    opt = finetune.AdamW(_tensors(), state_bits=bits, **HYPER)
    alone = [finetune.AdamW([p], state_bits=bits, **HYPER) for p in _tensors()]
    having = [{0, 2}, {0}, {0, 1, 2}, set(), {1, 2, 3}, {0, 1, 2, 3}, {3}]
    for t, have in enumerate(having):
        grads = _tensors(seed=t + 1)
        opt.step([g if i in have else None for i, g in enumerate(grads)])
        for i in have:
            alone[i].step([grads[i]])
        assert all(torch.equal(p, a.params[0]) for p, a in zip(opt.params, alone))
        assert all(torch.equal(s, r) for state, a in zip(opt.states, alone) for s, r in zip(state, a.states[0]))
    assert opt.steps == tuple(sum(i in have for have in having) for i in range(4)) and opt.step_count == len(having)
    # and go on from there
    again = finetune.AdamW([p.clone() for p in opt.params], state_bits=bits, states=[tuple(s.clone() for s in state) for state in opt.states], step=opt.steps, **HYPER)
    assert again.steps == opt.steps
    grads = _tensors(seed=99)
    opt.step(grads)
    again.step(grads)
    assert all(torch.equal(p, q) for p, q in zip(opt.params, again.params))


@pytest.mark.gpu
def test_the_first_step_of_a_late_parameter():
    """Its moments are a tenth and a hundredth of the first gradient and its square, corrected by as much: it moves by lr, to the roundings of
    about ten operations."""
    from symmetrix_amd import finetune
    opt = finetune.AdamW([torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")], lr=1e-2, betas=(0.9, 0.99), weight_decay=0.0)
    for _ in range(20):
        opt.step([torch.ones(100, device="cuda"), None])
    opt.step([None, torch.full((100,), -2.0, device="cuda")])
    assert ((opt.params[1].double() - 1e-2).abs() <= 1e-2 * 16 * 2.0 ** -24 + 1e-9).all()


@pytest.mark.gpu
def test_refused_steps():
    from symmetrix_amd import finetune
    for step in (-1, [0, 0, 0], [0, 0, 0, -1], [0] * 5):
        with pytest.raises(ValueError):
            finetune.AdamW(_tensors(), step=step)
