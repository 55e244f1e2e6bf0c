"""The norm of many tensors' gradients, clipping, and AdamW's steps by clipped gradients."""
import math

import pytest

torch = pytest.importorskip("torch")

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _grads(sizes, dtypes, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _norm(grads):
    """In 64 bits, whatever the size of the squares."""
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def _is_norm(got, want):
    """Sums in double precision, rounded once."""
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got.double()) - want) <= 2.0 ** -24 * (1 + 2.0 ** -10) * want + 2.0 ** -149


SIZES = [[1], [0, 1, 0], [5, 3], [255, 256, 257], [4095], [4096], [4097, 1, 12289], [1] * 300, [7, 100_003, 64, 999] * 30, [8_500_001], [2_000_000, 3] * 3]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES) + ["all"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_norm_and_clip(sizes, dtype):
    from symmetrix_amd import finetune
    dtypes = [NAMES[dtype]] if dtype != "all" else list(NAMES.values())
    grads = _grads(sizes, dtypes)
    want = _norm(grads)
    _is_norm(finetune.grad_norm(grads), want)
    assert torch.equal(finetune.grad_norm(grads), finetune.grad_norm(grads))
    for max_norm in (0.0, 0.3 * want, 2.0 * want, math.inf):
        out = [torch.full_like(g, 7.0) for g in grads]
        _is_norm(finetune.clip_grads(grads, max_norm, out=out), want)
        mine = [g.clone() for g in grads]
        _is_norm(finetune.clip_grads(mine, max_norm), want)
        factor = min(1.0, max_norm / want) if want else 1.0
        for g, o, m in zip(grads, out, mine):
            assert torch.equal(o, m)
            # the factor is rounded once, and the product
            assert ((o.double() - factor * g.double()).abs() <= (UNIT[g.dtype] + 2.0 ** -24) * 1.01 * (factor * g.double()).abs() + SMALLEST[g.dtype] / 2).all()
            assert factor < 1 or torch.equal(o, g)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-44, 1e25, 1e35])
def test_squares_neither_overflow_nor_vanish(scale):
    from symmetrix_amd import finetune
    grads = _grads([1000, 77], [torch.float32], scale)
    _is_norm(finetune.grad_norm(grads), _norm(grads))


@pytest.mark.gpu
def test_norms_that_are_not_finite_clip_nothing():
    from symmetrix_amd import finetune
    for value in (math.inf, -math.inf, math.nan):
        grads = _grads([5000, 33], [torch.float32, torch.bfloat16])
        grads[0][4999] = value
        before = [g.clone() for g in grads]
        norm = finetune.clip_grads(grads, 1.0)
        assert not norm.isfinite() and norm.isnan() == math.isnan(value)
        assert all(torch.equal(a.nan_to_num(3.0), b.nan_to_num(3.0)) for a, b in zip(grads, before))


@pytest.mark.gpu
def test_tensors_of_any_kind():
    """Starts at any alignment, other orders of dimensions, gradients that are not there, none at all, another stream."""
    from symmetrix_amd import finetune
    flat = torch.randn(10_001, device="cuda").bfloat16()
    views = [flat[1:100], flat[101:102], flat[103:9000], flat[9001:]]
    want = _norm(views)
    before = flat.clone()
    _is_norm(finetune.clip_grads(views, 0.5 * want), want)
    kept = torch.ones_like(flat, dtype=torch.bool)
    for a, b in ((1, 100), (101, 102), (103, 9000), (9001, 10_001)):
        kept[a:b] = False
    assert torch.equal(flat[kept], before[kept]) and torch.equal(flat[1:100], (before[1:100].float() * (0.5 * want / want)).bfloat16())
    turned = torch.randn(40, 30, device="cuda").t()
    version, old = turned._version, turned.clone()
    _is_norm(finetune.clip_grads([None, turned], 1.0), _norm([old]))
    assert turned._version > version and torch.allclose(turned, old / _norm([old]), rtol=1e-6, atol=0)
    assert float(finetune.grad_norm([])) == 0 and float(finetune.grad_norm([None])) == 0 and float(finetune.clip_grads([None, torch.zeros(0, device="cuda")], 1.0)) == 0
    _is_norm(finetune.grad_norm(turned), 1.0 * _norm([turned]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = finetune.grad_norm(views)
    side.synchronize()
    assert torch.equal(there, finetune.grad_norm(views))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", list(NAMES))
def test_adamw_by_clipped_gradients(dtype, bits):
    """The step is bit for bit the one of gradients multiplied by the factor in single precision."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    sizes = [1000, 1, 777, 5000]
    params = _grads(sizes, [dtype], 0.1)
    a, b = [p.clone() for p in params], [p.clone() for p in params]
    one, two = finetune.AdamW(a, lr=1e-2, state_bits=bits), finetune.AdamW(b, lr=1e-2, state_bits=bits)
    for k, max_norm in enumerate((0.5, 1e6, 3.0)):
        grads = _grads(sizes, [dtype], 0.3, seed=k)
        if k == 2:
            grads[2] = None
        there = [g for g in grads if g is not None]
        norm = one.step(grads, max_norm=max_norm)
        _is_norm(norm, _norm(there))
        factor = torch.tensor(min(1.0, max_norm / _norm(there)), dtype=torch.float32, device="cuda")
        clipped = [None if g is None else g.float() * factor for g in grads]
        assert two.step(clipped) is None
        for p, q in zip(a, b):
            assert torch.equal(p, q)
        for s, t in zip(one.states, two.states):
            assert all(torch.equal(u, v) for u, v in zip(s, t))
    assert float(one.step([None] * 4, max_norm=1.0)) == 0 and one.steps == (4 - 1, 4 - 1, 2, 4 - 1)
    with pytest.raises(ValueError):
        one.step(clipped, max_norm=-1.0)


@pytest.mark.gpu
def test_captured():
    from symmetrix_amd import finetune
    grads, out = _grads([3000, 50_001], [torch.float32, torch.float16]), None
    out = [torch.zeros_like(g) for g in grads]
    run = lambda: (finetune.grad_norm(grads), finetune.clip_grads(grads, 1.0, out=out))          # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = run()
    for _ in range(4):
        for g in grads:
            g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for a, b in zip(norms, run()):
            assert torch.equal(a, b)
        assert all(torch.equal(a, b) for a, b in zip(got, out))


@pytest.mark.gpu
def test_refusals():
    from symmetrix_amd import finetune
    g = torch.ones(10, device="cuda")
    for call in (lambda: finetune.grad_norm([g.double()]), lambda: finetune.grad_norm([g.int()]), lambda: finetune.clip_grads([g], 1.0, out=[g.half()])):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: finetune.grad_norm([g.cpu()]), lambda: finetune.clip_grads([g], -1.0), lambda: finetune.clip_grads([g], math.nan),
                 lambda: finetune.clip_grads([g, g], 1.0), lambda: finetune.clip_grads([g], 1.0, out=[g[:5]]), lambda: finetune.clip_grads([g], 1.0, out=[]),
                 lambda: finetune.clip_grads([g], 1.0, out=[None]), lambda: finetune.clip_grads([g, g + 1], 1.0, out=[g, g])):
        with pytest.raises(ValueError):
            call()
    assert g.eq(1).all()


@pytest.mark.gpu
def test_a_tensor_of_more_than_four_gigabytes():
    from symmetrix_amd import finetune
    n = 2_200_000_011
    big, small = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16), torch.full((3,), 2.0, device="cuda")
    big[-1] = 64.0
    want = math.sqrt(0.25 * (n - 1) + 64.0 ** 2 + 12.0)
    _is_norm(finetune.grad_norm([big, small]), want)
    _is_norm(finetune.clip_grads([big, small], want / 4), want)
    # a quarter, but for the factor's rounding, which 8 bits do not show
    assert float(big[-1]) == 16.0 and bool((big[:-1] == 0.125).all()) and ((small - 0.5).abs() <= 0.5 * 2.0 ** -23).all()


def test_a_broadcast_gradient_is_not_clipped_in_place():
    from symmetrix_amd import finetune
    with pytest.raises(ValueError, match="memory of their own"):
        finetune.clip_grads([torch.ones(3), torch.ones(()).expand(4, 5)], 1.0)


@pytest.mark.gpu
def test_broadcast_gradients():
    """As sums have them: one number in memory for all."""
    from symmetrix_amd import finetune
    p, q = torch.zeros(40, 3, device="cuda", requires_grad=True), torch.ones(7, device="cuda", requires_grad=True)
    grads = list(torch.autograd.grad(p.sum() + (q * q).sum(), [p, q]))
    assert grads[0].stride() == (0, 0)
    want = math.sqrt(120 + 28)
    _is_norm(finetune.grad_norm(grads), want)
    with pytest.raises(ValueError):
        finetune.clip_grads(grads, 1.0)
    assert grads[1].eq(2).all()
    out = [torch.empty(40, 3, device="cuda"), torch.empty(7, device="cuda")]
    _is_norm(finetune.clip_grads(grads, 1.0, out=out), want)
    assert ((out[0].double() - 1 / want).abs() <= 2.0 ** -23).all() and ((out[1].double() - 2 / want).abs() <= 2.0 ** -22).all()
    a = finetune.AdamW([p], lr=0.1, weight_decay=0.0)
    _is_norm(a.step([grads[0]], max_norm=1.0), math.sqrt(120))
    assert ((p + 0.1).abs() <= 1e-6).all()
