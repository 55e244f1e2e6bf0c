"""AdamW over many tensors against its formula in 64 bits, and moments in 8 bits against the same operations in numpy, bit for bit."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [1, 2, 3, 255, 256, 257, 0, 4095, 4096, 4097, 40001]


def _tensors(sizes, dtype, seed=0, scale=0.05):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dtype) for n in sizes]


def _formula(p, g, m, v, t, lr, betas, eps, weight_decay):
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    change = lr / (1 - betas[0] ** t) * m / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    return (1 - lr * weight_decay) * p - change, m, v, change


def _np(t):
    return t.detach().double().cpu().numpy().reshape(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("grad_type", ["own", "float32"])
@pytest.mark.parametrize("dtype", list(UNIT))
def test_moments_in_32_bits(dtype, grad_type, masters):
    """Three steps, each against the formula from what the step before left.  Roundings in single precision: m three, v four,
    the change about ten beyond what m and sqrt(v) carry; then p's own two, and the one to its type."""
    from symmetrix_amd import finetune
    if masters and dtype == torch.float32:
        pytest.skip("masters are for 16 bits")
    params = _tensors(SIZES, dtype)
    opt = finetune.AdamW(params, masters=True if masters else None, **HYPER)
    u = 2.0 ** -24
    for t in range(1, 4):
        grads = _tensors(SIZES, torch.float32 if grad_type == "float32" else dtype, seed=t, scale=0.01)
        before = [(_np(opt.masters[i] if masters else p), _np(opt.states[i][0]), _np(opt.states[i][1])) for i, p in enumerate(params)]
        opt.step(grads)
        for i, p in enumerate(params):
            g = _np(grads[i])
            want, m, v, change = _formula(before[i][0], g, before[i][1], before[i][2], t, **HYPER)
            slack_m = 4 * u * (np.abs(before[i][1]) + np.abs(g))
            assert (np.abs(_np(opt.states[i][0]) - m) <= slack_m).all()
            assert (np.abs(_np(opt.states[i][1]) - v) <= 5 * u * v + 1e-45).all()
            # (the largest |m| a change can be off by, over the smallest root below it)
            ratio = HYPER["lr"] / (1 - HYPER["betas"][0] ** t) / (np.sqrt(v / (1 - HYPER["betas"][1] ** t)) + HYPER["eps"])
            slack = 16 * u * np.abs(change) + slack_m * ratio + 3 * u * np.abs(before[i][0])
            if masters:
                assert (np.abs(_np(opt.masters[i]) - want) <= slack).all()
                assert torch.equal(opt.masters[i].to(dtype), p)
            else:
                assert (np.abs(_np(p) - want) <= slack + UNIT[dtype] * (1 + 2.0 ** -8) * np.abs(want) + 2.0 ** -25).all()


def _f(x):
    return np.float32(x)


def _codes_step(p, g, cm, sm, cv, sv, t, lr, betas, eps, weight_decay):
    """The step with moments in 8 bits in numpy's single precision, one rounding an operation."""
    n = len(p)
    wide = lambda s: np.repeat(s, 256)[:n]          # noqa: E731
    q = cm.astype(np.float32) * _f(_f(1) / _f(127))
    m = q * np.abs(q) * wide(sm)
    r = cv.astype(np.float32) * _f(_f(1) / _f(255))
    r = r * r
    v = r * r * wide(sv)
    m = m * _f(betas[0]) + g * _f(1 - betas[0])
    v = v * _f(betas[1]) + g * _f(1 - betas[1]) * g
    p = p * _f(1 - lr * weight_decay) - m * _f(lr / (1 - betas[0] ** t)) / (np.sqrt(v) * _f(1 / math.sqrt(1 - betas[1] ** t)) + _f(eps))
    blocks = -(-n // 256)
    pad = lambda a: np.concatenate([a, np.zeros(blocks * 256 - n, dtype=np.float32)]).reshape(blocks, 256)          # noqa: E731
    sm, sv = np.abs(pad(m)).max(1), pad(v).max(1)
    over = lambda a, s: a / wide(np.where(s > 0, s, _f(1)))          # noqa: E731
    inside = np.arange(n, dtype=np.uint64)
    turn = lambda k: (((inside * 0x9E3779B1 + (2 * t + k) * 0x85EBCA6B) % (1 << 32)) >> 8).astype(np.float32) * _f(2.0 ** -24)          # noqa: E731
    qm = np.minimum(np.floor(np.sqrt(over(np.abs(m), sm)) * _f(127) + turn(0)), _f(127))
    qv = np.minimum(np.floor(np.sqrt(np.sqrt(over(v, sv))) * _f(255) + turn(1)), _f(255))
    cm = np.where(m < 0, -qm, qm).astype(np.int8)
    cv = np.where(v > 0, np.maximum(qv, _f(1)), _f(0)).astype(np.uint8)
    return p, cm, sm, cv, sv


@pytest.mark.gpu
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("dtype", list(UNIT))
def test_moments_in_8_bits(dtype, masters):
    """Codes, scales and parameters are the formulas', bit for bit."""
    from symmetrix_amd import finetune
    if masters and dtype == torch.float32:
        pytest.skip("masters are for 16 bits")
    params = _tensors(SIZES, dtype)
    opt = finetune.AdamW(params, masters=True if masters else None, state_bits=8, **HYPER)
    for t in range(1, 5):
        grads = _tensors(SIZES, dtype, seed=t, scale=0.01)
        if t == 2:
            grads = [torch.zeros_like(g) for g in grads]
        before = [((opt.masters[i] if masters else p).float().cpu().numpy().copy(), [s.cpu().numpy().copy() for s in opt.states[i]]) for i, p in enumerate(params)]
        opt.step(grads)
        for i, p in enumerate(params):
            if not SIZES[i]:
                continue
            want = _codes_step(before[i][0], grads[i].float().cpu().numpy(), *before[i][1], t, **HYPER)
            have = opt.masters[i] if masters else p
            assert torch.equal(have.cpu(), torch.from_numpy(want[0]).to(have.dtype))
            for s, w in zip(opt.states[i], want[1:]):
                assert np.array_equal(s.cpu().numpy(), w)
            m, v = finetune.moment_values(*opt.states[i])
            q, r = want[1].astype(np.float32) * _f(_f(1) / _f(127)), want[3].astype(np.float32) * _f(_f(1) / _f(255))
            r = r * r
            wide = lambda s: np.repeat(s, 256)[:SIZES[i]]          # noqa: E731
            assert np.array_equal(m.cpu().numpy(), q * np.abs(q) * wide(want[2])) and np.array_equal(v.cpu().numpy(), r * r * wide(want[4]))


@pytest.mark.gpu
def test_moments_in_8_bits_follow_those_in_32():
    """A moment decays though a step moves it by much less than a code: with gradients that fall to a tenth after 200 steps, the root of the
    second moment (beta2 = 0.99) follows to within a code's width at its place, two codes of 255 around a value that carries
    half of the scale or more, averaged over the numbers of a tensor."""
    from symmetrix_amd import finetune
    n = 4096
    runs = []
    for bits in (32, 8):
        p = [torch.zeros(n, device="cuda")]
        opt = finetune.AdamW(p, lr=1e-4, betas=(0.9, 0.99), weight_decay=0.0, state_bits=bits)
        for t in range(500):
            g = torch.Generator(device="cuda").manual_seed(t)
            opt.step([torch.randn(n, generator=g, device="cuda") * (1.0 if t < 200 else 0.1)])
        v = opt.states[0][1] if bits == 32 else finetune.moment_values(*opt.states[0])[1]
        runs.append(torch.sqrt(v.double()).mean().item())
    assert abs(runs[1] / runs[0] - 1) < 2 * 2 / 255


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_unaligned_ones(bits):
    """More tensors than a launch takes, and tensors that start at any number of one array."""
    from symmetrix_amd import finetune
    sizes = [1 + (37 * i) % 700 for i in range(150)]
    flat = torch.randn(sum(sizes) + 1, device="cuda")
    views, at = [], 1
    for n in sizes:
        views.append(flat[at:at + n])
        at += n
    alone = [v.clone() for v in views]
    opt, ref = (finetune.AdamW(p, state_bits=bits, **HYPER) for p in (views, alone))
    for t in range(2):
        grads = _tensors(sizes, torch.float32, seed=t)
        opt.step(grads)
        for i in range(len(sizes)):          # one at a time
            one = finetune.AdamW([alone[i]], state_bits=bits, states=[ref.states[i]], step=t, **HYPER)
            one.step([grads[i]])
    assert all(torch.equal(p, q) for p, q in zip(views, alone))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_number_that_is_not_finite(bits):
    """With 32 bits it keeps to its own place, with 8 to its own 256; other tensors and blocks never see it."""
    from symmetrix_amd import finetune
    for value in (float("nan"), float("inf")):
        runs = []
        for bad in (False, True):
            p = _tensors([1000, 300], torch.float32)
            opt = finetune.AdamW(p, state_bits=bits, **HYPER)
            for t in range(2):
                g = _tensors([1000, 300], torch.float32, seed=t)
                if bad:
                    g[0][300] = value
                opt.step(g)
            runs.append(p)
        (a, b), (c, d) = runs
        assert torch.equal(b, d) and torch.isnan(c[300])
        other = torch.ones(1000, dtype=torch.bool)
        if bits == 8:
            other[256:512] = False
        else:
            other[300] = False
        assert torch.equal(a[other.cuda()], c[other.cuda()])


@pytest.mark.gpu
def test_parameters_without_gradients_and_own_gradients():
    from symmetrix_amd import finetune
    p = [torch.nn.Parameter(t) for t in _tensors([10, 20, 30], torch.float32)]
    before = [t.detach().clone() for t in p]
    opt = finetune.AdamW(p, **HYPER)
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(p, before)) and opt.step_count == 1
    p[1].grad = torch.ones(20, device="cuda")
    opt.step()
    assert torch.equal(p[0], before[0]) and not torch.equal(p[1], before[1]) and torch.equal(p[2], before[2])
    # a product that saved the old value notices
    x = (p[1] * p[1]).sum()
    opt.step()
    with pytest.raises(RuntimeError):
        x.backward()


@pytest.mark.gpu
def test_beyond_32_bits():
    """A tensor of more than 2^31 numbers: its last ones are updated as those of a short one."""
    from symmetrix_amd import finetune
    n = (1 << 31) + 300
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(300, device="cuda").to(torch.bfloat16)
    p[-300:] = tail
    g[-300:] = tail * 0.5
    short, = (tail.clone(),)
    opt = finetune.AdamW([p], state_bits=8, **HYPER)
    ref = finetune.AdamW([short], state_bits=8, **HYPER)
    opt.step([g])
    ref.step([(tail * 0.5).to(torch.bfloat16)])
    assert torch.equal(p[-300:], short) and (p[:1000] == 0).all()
    # (2^31 is a multiple of 256, and of what the rounding's place repeats after only by chance: scales are the same, codes may not be)
    assert torch.equal(opt.states[0][1][-2:], ref.states[0][1])


@pytest.mark.gpu
def test_in_a_graph():
    from symmetrix_amd import finetune
    p, q = _tensors([5000], torch.float32), _tensors([5000], torch.float32)
    opt, ref = finetune.AdamW(p, **HYPER), finetune.AdamW(q, **HYPER)
    g = torch.zeros(5000, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([g])
    for k in range(3):
        g.copy_(torch.randn(5000, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        ref.step_count = 0          # (a graph keeps the number of the step it was captured with)
        ref.step([g])
        assert torch.equal(p[0], q[0])


@pytest.mark.gpu
def test_refusals():
    from symmetrix_amd import finetune
    p = _tensors([8, 300], torch.float32)
    g = _tensors([8, 300], torch.float32)
    make = finetune.AdamW
    bad = [
        (ValueError, lambda: make([t.cpu() for t in p])),
        (TypeError, lambda: make([t.double() for t in p])),
        (TypeError, lambda: make([p[0], p[1].half()])),
        (ValueError, lambda: make([torch.zeros(4, 4, device="cuda").t()[1:, 1:]])),
        (ValueError, lambda: make(p, state_bits=16)),
        (ValueError, lambda: make(p, betas=(1.0, 0.9))),
        (ValueError, lambda: make(p, lr=-1.0)),
        (ValueError, lambda: make(p, masters=True)),
        (ValueError, lambda: make([t.half() for t in p], masters=p[:1])),
        (ValueError, lambda: make(p, states=[(p[0], p[0])])),
        (ValueError, lambda: make(p, states=[(t.half(), t.half()) for t in p])),
        (ValueError, lambda: make(p, state_bits=8, states=[(t, t) for t in p])),
        (ValueError, lambda: make(p, step=-1)),
        (ValueError, lambda: make(p).step(g[:1])),
        (ValueError, lambda: make(p).step([g[0], g[1][:299]])),
        (ValueError, lambda: make(p).step([g[0], g[1].cpu()])),
        (TypeError, lambda: make(p).step([g[0], g[1].half()])),
        (TypeError, lambda: make(p).step([t.half() for t in g])),
        (TypeError, lambda: finetune.moment_values(p[0], p[0], p[0], p[0])),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_c_entry_refuses_without_touching_a_device():
    import ctypes as C
    from symmetrix_amd import finetune
    L = finetune._lib_functions()
    one = (finetune._AdamwTensor * 1)(finetune._AdamwTensor(1, 1, 0, 1, 1, 0, 0, 4))          # (never read)
    call = lambda pt=0, gt=0, bits=32, t=one, n=1, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, step=1: L.smx_adamw_step(          # noqa: E731
        pt, gt, bits, C.addressof(t) if t is not None else 0, n, lr, b1, b2, eps, wd, step, 0)
    assert call(pt=5) == -1 and call(gt=1) == -1 and call(bits=16) == -1 and call(t=None) == -1 and call(n=-1) == -1
    assert call(step=0) == -1 and call(b1=1.0) == -1 and call(lr=float("inf")) == -1 and call(eps=float("nan")) == -1
    assert call(bits=8) == -1 and b"scales" in L.smx_last_error()
    assert call(n=0) == 0
    one[0].master = 1
    assert call() == -1 and b"masters" in L.smx_last_error()
    one[0].numel = 0
    assert call() == 0
    assert L.smx_moment_values(-1, 0, 0, 0, 0, 0, 0, 0) == -1 and L.smx_moment_values(0, 0, 0, 0, 0, 0, 0, 0) == 0


@pytest.mark.gpu
def test_values_of_more_codes_than_a_launch_takes():
    from symmetrix_amd import finetune
    n = (1 << 30) + 600
    cm, cv = torch.zeros(n, dtype=torch.int8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    cm[-600:] = torch.randint(-127, 128, (600,), device="cuda").to(torch.int8)
    cv[-600:] = torch.randint(0, 256, (600,), device="cuda").to(torch.uint8)
    sm, sv = torch.rand((n + 255) // 256, device="cuda") + 0.5, torch.rand((n + 255) // 256, device="cuda") + 0.5
    m, v = finetune.moment_values(cm, sm, cv, sv)
    m0, v0 = finetune.moment_values(cm[-600:].clone(), sm[-3:].clone(), cv[-600:].clone(), sv[-3:].clone())
    assert torch.equal(m[-600:], m0) and torch.equal(v[-600:], v0)
