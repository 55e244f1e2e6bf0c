"""A shared projection with a low-rank adapter per row and its gradient against the definition in 64 bits: types, widths, ranks,
orders of rows, rows without an adapter, adapters without a row, strides, infinities and NaN, refusals."""
import pytest

torch = pytest.importorskip("torch")

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(UNIT)
NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24


def _index(rows, n, order, seed=0):
    """runs: requests of some rows each, one in eight without an adapter; mixed: any order; own: neighbours differ; one: a single adapter"""
    g = torch.Generator().manual_seed(seed)
    if order == "one":
        return torch.full((rows,), max(n - 1, 0), dtype=torch.int32, device="cuda")
    if order == "own":
        return (torch.arange(rows) % max(n, 1)).to(torch.int32).cuda()
    if order == "none":
        return torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    index = torch.randint(-1 if order == "mixed" else 0, n, (rows,), generator=g, dtype=torch.int32)
    if order == "runs":
        length = max(1, rows // (2 * n))
        index = index[torch.arange(rows) // length]
        index[torch.rand(rows // length + 1, generator=g)[torch.arange(rows) // length] < 0.125] = -1
    return index.cuda()


def _data(rows, d_in, d_out, rank, n, dtype, order="runs", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    return dict(x=r(rows, d_in).to(dtype), weight=(r(d_out, d_in) * d_in ** -0.5).to(dtype), A=(r(n, rank, d_in) * d_in ** -0.5).to(dtype),
                B=(r(n, d_out, rank) * rank ** -0.5).to(dtype), scale=torch.rand(n, generator=g, device="cuda") + 0.5,
                index=_index(rows, n, order, seed)), r(rows, d_out).to(dtype)


def _reference(x, weight, A, B, scale, index, dy=None):
    """Results in 64 bits, and of each the sum of its terms' sizes with what the terms carry of earlier roundings."""
    x, weight, A, B, index = x.double(), weight.double(), A.double(), B.double(), index.long()
    n, rank, d_in = A.shape
    d_out = weight.shape[0]
    ones = torch.ones(n, dtype=torch.float64, device=x.device) if scale is None else scale.double()
    lam = 8.0          # of a sum's error bound lam sqrt(terms) u sum |terms|, which random roundings stay below
    steps = lambda k: lam * (k ** 0.5 + 2) * U          # noqa: E731
    if dy is None:
        y = x @ weight.t()
        off = (x.abs() @ weight.abs().t()) * steps(d_in)
        for a in range(n):
            at = (index == a).nonzero()[:, 0]
            if not len(at):
                continue
            h = ones[a] * (x[at] @ A[a].t())
            size = ones[a] * (x[at].abs() @ A[a].abs().t())
            y[at] += h @ B[a].t()
            off[at] += (size * steps(d_in)) @ B[a].abs().t() + (h.abs() @ B[a].abs().t()) * steps(rank + 1)
        return {"y": (y, off)}
    dy = dy.double()
    dx, off = dy @ weight, (dy.abs() @ weight.abs()) * steps(d_out)
    dA, dB = torch.zeros_like(A), torch.zeros_like(B)
    off_a, off_b = torch.zeros_like(A), torch.zeros_like(B)
    for a in range(n):
        at = (index == a).nonzero()[:, 0]
        if not len(at):
            continue
        g, h = ones[a] * (dy[at] @ B[a]), ones[a] * (x[at] @ A[a].t())
        g_off, h_off = steps(d_out) * ones[a] * (dy[at].abs() @ B[a].abs()), steps(d_in) * ones[a] * (x[at].abs() @ A[a].abs().t())
        dx[at] += g @ A[a]
        off[at] += g_off @ A[a].abs() + (g.abs() @ A[a].abs()) * steps(rank + 1)
        dA[a], dB[a] = g.t().contiguous() @ x[at], dy[at].t().contiguous() @ h
        k = steps(len(at))
        off_a[a] = (g_off + k * g.abs()).t().contiguous() @ x[at].abs()
        off_b[a] = dy[at].abs().t().contiguous() @ (h_off + k * h.abs())
    return {"dx": (dx, off), "dA": (dA, off_a), "dB": (dB, off_b)}


def _close(got, want, off, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    # what a factor brought to two parts of a 16-bit type may lose of a product: 2^-16 of it, in off's terms
    more = 0 if dtype == torch.float32 else 2.0 ** -16 / (8 * 2 * U)
    assert ((got.double() - want).abs() <= off * (1 + more) + UNIT[dtype] * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25).all()


def _check(data, dy=None, backward=True):
    from symmetrix_amd import finetune
    dtype = data["x"].dtype
    y = finetune.adapted_linear_forward(**data)
    _close(y, *_reference(**data)["y"], dtype)
    if backward:
        got = dict(zip(("dx", "dA", "dB"), finetune.adapted_linear_backward(dy, **data)))
        for k, (want, off) in _reference(**data, dy=dy).items():
            _close(got[k], want, off, dtype)


SHAPES = [  # rows, d_in, d_out, rank, adapters
    (1, 32, 32, 1, 1), (1, 96, 128, 4, 3), (2, 64, 48, 8, 5), (7, 33, 65, 3, 2), (15, 128, 96, 16, 4), (16, 256, 512, 8, 16), (17, 200, 136, 24, 7),
    (24, 192, 128, 4, 3), (31, 1, 1, 1, 1), (33, 1, 70, 2, 3), (33, 70, 1, 2, 3), (63, 129, 257, 5, 6), (64, 512, 512, 32, 9), (65, 96, 96, 64, 4), (100, 320, 64, 128, 3),
    (127, 256, 256, 16, 64), (128, 257, 255, 17, 11), (129, 1024, 512, 16, 12), (255, 96, 192, 12, 100), (256, 2048, 1000, 16, 8), (257, 640, 640, 48, 5),
    (500, 128, 128, 8, 300), (1000, 192, 288, 8, 12), (1023, 500, 300, 7, 17), (2049, 256, 512, 8, 12), (4097, 96, 128, 16, 33),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(shape, dtype):
    for order in ("runs", "mixed"):
        data, dy = _data(*shape, NAMES[dtype], order, seed=sum(shape))
        _check(data, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("order", ["own", "one", "none"])
def test_orders(order, dtype):
    for shape in ((16, 512, 256, 16, 16), (300, 160, 224, 8, 40), (2000, 96, 96, 4, 3)):
        data, dy = _data(*shape, NAMES[dtype], order)
        _check(data, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_larger(dtype):
    data, dy = _data(20011, 256, 512, 8, 12, NAMES[dtype])
    _check(data, dy)
    data, dy = _data(1531, 2080, 1184, 32, 24, NAMES[dtype])
    _check(data, dy)
    data, dy = _data(70001, 64, 32, 4, 4096, NAMES[dtype], "mixed")
    from symmetrix_amd import finetune
    y = finetune.adapted_linear_forward(**data)
    keep = torch.arange(0, 70001, 97, device="cuda")
    few = dict(data, x=data["x"][keep], index=data["index"][keep])
    _close(y[keep], *_reference(**few)["y"], NAMES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_rows_of_one_token(dtype):
    """One row, and a few with an adapter each, through wide projections."""
    for rows in (1, 2, 5, 16, 17, 32, 48, 64, 128):
        data, dy = _data(rows, 2048, 1536, 16, 64, NAMES[dtype], "own")
        _check(data, dy, backward=rows in (1, 17))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_no_rows_no_adapters(dtype):
    from symmetrix_amd import finetune
    data, dy = _data(0, 64, 32, 4, 3, NAMES[dtype], "one")
    assert finetune.adapted_linear_forward(**data).shape == (0, 32)
    dx, dA, dB = finetune.adapted_linear_backward(dy, **data)
    assert dx.shape == (0, 64) and (dA == 0).all() and (dB == 0).all()
    data, dy = _data(40, 64, 32, 4, 0, NAMES[dtype], "none")
    _check(data, dy)
    # one adapter without a row, before, between and behind others
    data, dy = _data(90, 64, 96, 4, 7, NAMES[dtype])
    data["index"] = torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda").repeat_interleave(30)
    _check(data, dy)
    assert all((finetune.adapted_linear_backward(dy, **data)[k][::2] == 0).all() for k in (1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("shape", [(20, 256, 128, 8, 4), (200, 96, 64, 8, 4), (700, 256, 320, 16, 6)], ids=str)
def test_an_index_out_of_range(shape, dtype):
    """Its row is NaN and has no part in anything else."""
    from symmetrix_amd import finetune
    data, dy = _data(*shape, NAMES[dtype])
    clean = dict(data, index=data["index"].clone())
    bad = torch.tensor([0, 7, shape[0] - 1], device="cuda")
    for value, i in zip((-2, shape[4], 2 ** 31 - 1), bad.tolist()):
        data["index"][i] = value
        clean["index"][i] = -1
    y, z = finetune.adapted_linear_forward(**data), finetune.adapted_linear_forward(**clean)
    good = torch.ones(shape[0], dtype=torch.bool, device="cuda")
    good[bad] = False
    assert torch.isnan(y[bad]).all() and torch.equal(y[good], z[good])
    got, want = finetune.adapted_linear_backward(dy, **data), finetune.adapted_linear_backward(dy, **clean)
    assert torch.isnan(got[0][bad]).all() and torch.equal(got[0][good], want[0][good])
    for k, (ref, off) in enumerate(list(_reference(**clean, dy=dy).values())[1:], 1):
        _close(got[k], ref, off, NAMES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("order", ["runs", "own"])
@pytest.mark.parametrize("rows", [16, 50, 400])
def test_an_adapter_that_is_not_finite_keeps_to_its_rows(rows, order, dtype):
    from symmetrix_amd import finetune
    data, dy = _data(rows, 160, 96, 8, 5, NAMES[dtype], order)
    y, grads = finetune.adapted_linear_forward(**data), finetune.adapted_linear_backward(dy, **data)
    mine = data["index"] == 2
    for name, value in (("A", float("nan")), ("B", float("inf")), ("scale", float("nan"))):
        broken = dict(data)
        broken[name] = data[name].clone()
        broken[name][2] = value
        z, changed = finetune.adapted_linear_forward(**broken), finetune.adapted_linear_backward(dy, **broken)
        assert torch.equal(z[~mine], y[~mine]) and not torch.isfinite(z[mine]).any()
        assert torch.equal(changed[0][~mine], grads[0][~mine])
        others = torch.tensor([0, 1, 3, 4], device="cuda")
        assert torch.equal(changed[1][others], grads[1][others]) and torch.equal(changed[2][others], grads[2][others])
    # a row that is not finite: other rows, and other adapters' gradients, never see it
    i = int(mine.nonzero()[0]) if mine.any() else 0
    broken = dict(data, x=data["x"].clone())
    broken["x"][i] = float("nan")
    z, changed = finetune.adapted_linear_forward(**broken), finetune.adapted_linear_backward(dy, **broken)
    rest = torch.arange(rows, device="cuda") != i
    assert torch.equal(z[rest], y[rest]) and torch.isnan(z[i]).all() and torch.equal(changed[0], grads[0])
    a = int(data["index"][i])
    others = torch.tensor([k for k in range(5) if k != a], device="cuda")
    assert torch.equal(changed[1][others], grads[1][others]) and torch.equal(changed[2][others], grads[2][others])


@pytest.mark.gpu
def test_the_range_of_single_precision():
    """Infinities where the definition has them, numbers near both ends of the range, sums that overflow."""
    from symmetrix_amd import finetune
    for rows in (5, 40, 300):
        data, _ = _data(rows, 96, 64, 4, 2, torch.float32, "one")
        for factor in (2.0 ** 100, 2.0 ** -100, 2.0 ** 110, 2.0 ** -120):
            big = dict(data, x=data["x"] * factor)
            want, off = _reference(**big)["y"]
            assert ((finetune.adapted_linear_forward(**big).double() - want).abs() <= off + 2.0 ** -24 * want.abs() + 96 * 2.0 ** -148).all()
        huge = dict(data, x=data["x"].clone())
        huge["x"][3, 5] = float("inf")
        y = finetune.adapted_linear_forward(**huge)
        expect = torch.matmul(huge["x"].double(), huge["weight"].double().t())
        assert torch.isfinite(y[[0, 1, 2, 4]]).all() and not torch.isfinite(y[3]).any() and not torch.isfinite(expect[3]).any()
        plain = dict(huge, index=torch.full_like(huge["index"], -1))
        assert torch.equal(finetune.adapted_linear_forward(**plain)[3], expect[3].float())
        huge["x"][3, 5] = 3e38
        huge["weight"] = data["weight"].clone()
        huge["weight"][7] = 100.0
        assert torch.isinf(finetune.adapted_linear_forward(**huge)[3, 7])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_strides_and_alignment(dtype):
    """Rows of wider arrays at odd offsets, more dimensions than two, a weight that is a part of a larger one, copies where needed."""
    from symmetrix_amd import finetune
    t = NAMES[dtype]
    for rows in (13, 300):
        data, dy = _data(rows, 96, 64, 8, 5, t)
        wide = torch.randn(rows, 303, device="cuda").to(t)
        big = (torch.randn(64, 211, device="cuda") * 0.1).to(t)
        _check(dict(data, x=wide[:, 1:97], weight=big[:, 3:99]), wide[:, 130:194])
        _check(dict(data, x=wide[:, 100:196], weight=big[:, 99:195]), wide[:, 1:65])
        odd = torch.randn(5 * 8 * 96 + 1, device="cuda").to(t)
        _check(dict(data, A=odd[1:].view(5, 8, 96), B=odd[1:1 + 5 * 64 * 8].view(5, 64, 8)), dy)
        _check(dict(data, x=torch.randn(96, rows, device="cuda").to(t).t(), scale=None), dy)
        _check(dict(data, x=torch.randn(1, 96, device="cuda").to(t).expand(rows, 96)), dy)
    data, dy = _data(24, 96, 64, 8, 5, t)
    y = finetune.adapted_linear_forward(**dict(data, x=data["x"].view(2, 3, 4, 96), index=data["index"].view(2, 3, 4)))
    assert y.shape == (2, 3, 4, 64) and torch.equal(y.view(24, 64), finetune.adapted_linear_forward(**data))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    stride = (1 << 30) + 8
    store = torch.empty(3 * stride + 96, dtype=torch.bfloat16, device="cuda")
    data, dy = _data(4, 96, 64, 8, 3, torch.bfloat16, "own")
    x = store.as_strided((4, 96), (stride, 1))
    x.copy_(data["x"])
    _check(dict(data, x=x), dy)
    # enough rows for the ways of larger calls
    stride = (1 << 24) + 8
    store = torch.empty(299 * stride + 96, dtype=torch.bfloat16, device="cuda")
    data, dy = _data(300, 96, 64, 8, 3, torch.bfloat16, "mixed")
    x = store.as_strided((300, 96), (stride, 1))
    x.copy_(data["x"])
    _check(dict(data, x=x), dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_the_same_bits_every_time(dtype):
    from symmetrix_amd import finetune
    data, dy = _data(6007, 192, 160, 8, 12, NAMES[dtype], "mixed")
    first = (finetune.adapted_linear_forward(**data),) + finetune.adapted_linear_backward(dy, **data)
    for _ in range(3):
        again = (finetune.adapted_linear_forward(**data),) + finetune.adapted_linear_backward(dy, **data)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.gpu
def test_single_gradients_are_those_of_all():
    from symmetrix_amd import finetune
    data, dy = _data(900, 128, 96, 8, 6, torch.float32)
    every = finetune.adapted_linear_backward(dy, **data)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        got = finetune.adapted_linear_backward(dy, **data, need=need)
        for g, e, wanted in zip(got, every, need):
            assert (g is None) != wanted and (g is None or torch.equal(g, e))


@pytest.mark.gpu
def test_automatic_differentiation_and_differences():
    """The output is linear in x, in A and in B, so that differences have no error of their own: what is left is the forward's."""
    from symmetrix_amd import finetune
    data, c = _data(300, 96, 64, 8, 5, torch.float32, "mixed")
    leaves = {k: data[k].requires_grad_() for k in ("x", "A", "B")}
    (finetune.adapted_linear(**data) * c).sum().backward()
    fixed = {k: v.detach() for k, v in data.items()}
    _, off = _reference(**fixed)["y"]
    for k, leaf in leaves.items():
        d = torch.randn_like(leaf)
        value = lambda side: (finetune.adapted_linear_forward(**dict(fixed, **{k: fixed[k] + side * d})).double() * c.double()).sum().item()          # noqa: E731
        want = (value(1) - value(-1)) / 2
        got = (leaf.grad.double() * d.double()).sum().item()
        # (a sum of values that are each off by less than `off`; moved inputs are about twice as large)
        assert abs(got - want) <= 8 * (off * c.double().abs()).sum().item()
    data["weight"] = data["weight"].detach().requires_grad_()
    with pytest.raises(ValueError):
        finetune.adapted_linear(**data)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    from symmetrix_amd import finetune
    for shape in ((16, 256, 128, 8, 16), (1500, 128, 96, 8, 12)):
        data, dy = _data(*shape, torch.float32)
        side = torch.cuda.Stream()
        want = finetune.adapted_linear_forward(**data)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = finetune.adapted_linear_forward(**data)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = finetune.adapted_linear_forward(**data)
            grads = finetune.adapted_linear_backward(dy, **data)
        for k in range(4):
            data["x"].copy_(torch.randn_like(data["x"]))
            data["index"].copy_(_index(shape[0], shape[4], "mixed", seed=k))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, finetune.adapted_linear_forward(**data))
            assert all(torch.equal(p, q) for p, q in zip(grads, finetune.adapted_linear_backward(dy, **data)))


@pytest.mark.gpu
def test_refusals():
    from symmetrix_amd import finetune
    data, dy = _data(6, 32, 48, 4, 3, torch.float32)
    call = lambda **k: finetune.adapted_linear_forward(**dict(data, **k))          # noqa: E731
    bad = [
        (ValueError, lambda: call(x=data["x"].cpu())),
        (ValueError, lambda: call(index=data["index"].cpu())),
        (ValueError, lambda: call(x=data["x"][:, :31])),
        (ValueError, lambda: call(weight=data["weight"][0])),
        (ValueError, lambda: call(A=data["A"][0])),
        (ValueError, lambda: call(A=data["A"][:2])),
        (ValueError, lambda: call(B=data["B"][:, :47])),
        (ValueError, lambda: call(scale=data["scale"][:2])),
        (ValueError, lambda: call(index=data["index"][:5])),
        (ValueError, lambda: call(A=torch.zeros(1, 129, 32, device="cuda"), B=torch.zeros(1, 48, 129, device="cuda"), scale=None)),
        (ValueError, lambda: call(A=torch.zeros(4097, 1, 32, device="cuda"), B=torch.zeros(4097, 48, 1, device="cuda"), scale=None)),
        (TypeError, lambda: call(x=data["x"].double())),
        (TypeError, lambda: call(x=data["x"].half())),
        (TypeError, lambda: call(index=data["index"].long())),
        (TypeError, lambda: call(scale=data["scale"].double())),
        (ValueError, lambda: finetune.adapted_linear_backward(dy[:5], **data)),
        (ValueError, lambda: finetune.adapted_linear_backward(dy[:, :47], **data)),
        (TypeError, lambda: finetune.adapted_linear_backward(dy.half(), **data)),
    ]
    for kind, f in bad:
        with pytest.raises(kind):
            f()


def test_c_entry_refuses_without_touching_a_device():
    import ctypes as C
    from symmetrix_amd import finetune
    L = finetune._lib_functions()
    good = dict(type=0, d_in=32, d_out=32, rank=4, num_adapters=2, rows=10, x=1, x_stride=32, weight=1, weight_stride=32, A=1, B=1, scale=0, index=1)
    size = C.c_long()
    describe = lambda **k: C.byref(finetune._Adapted(**dict(good, **k)))          # noqa: E731
    assert L.smx_adapted_linear_workspace(describe(), 1, C.byref(size)) == 0 and size.value > 0
    for wrong in (dict(type=3), dict(d_in=0), dict(d_out=0), dict(rank=0), dict(rank=129), dict(num_adapters=-1), dict(num_adapters=4097), dict(rows=-1),
                  dict(x=0), dict(x_stride=31), dict(weight=0), dict(weight_stride=31), dict(A=0), dict(B=0), dict(index=0)):
        assert L.smx_adapted_linear_workspace(describe(**wrong), 0, C.byref(size)) == -1, wrong
        assert L.smx_adapted_linear_forward(describe(**wrong), 1, 32, 1, 1 << 40, 0) == -1, wrong
        assert L.smx_adapted_linear_backward(describe(**wrong), 1, 32, 1, 32, 1, 1, 1, 1 << 40, 0) == -1, wrong
    assert L.smx_adapted_linear_forward(0, 1, 32, 1, 1 << 40, 0) == -1
    assert L.smx_adapted_linear_forward(describe(), 0, 32, 1, 1 << 40, 0) == -1
    assert L.smx_adapted_linear_forward(describe(), 1, 31, 1, 1 << 40, 0) == -1
    assert L.smx_adapted_linear_forward(describe(), 1, 32, 1, 0, 0) == -1 and b"workspace" in L.smx_last_error()
    assert L.smx_adapted_linear_backward(describe(), 1, 31, 1, 32, 1, 1, 1, 1 << 40, 0) == -1
    assert L.smx_adapted_linear_forward(describe(rows=0), 1, 32, 0, 0, 0) == 0
