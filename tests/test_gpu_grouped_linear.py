"""A product with a matrix of the row's own group and its gradient against the definition in 64 bits: types, widths, orders of rows, groups
of any size and empty ones, rows without a group, strides, infinities and NaN, refusals."""
import pytest

torch = pytest.importorskip("torch")

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24


def _index(rows, n, order, seed=0):
    """mixed: any order, some without a group; runs: sorted; few: most groups empty; own: neighbours differ; one: a single group; none"""
    g = torch.Generator().manual_seed(seed)
    if order == "one":
        index = torch.full((rows,), n - 1)
    elif order == "none":
        index = torch.full((rows,), -1)
    elif order == "own":
        index = torch.arange(rows) % n
    elif order == "few":
        index = torch.randint(0, n, (3,), generator=g)[torch.randint(0, 3, (rows,), generator=g)]
    else:
        index = torch.randint(-1, n, (rows,), generator=g)
        if order == "runs":
            index = index.sort().values
    return index.to(torch.int32).cuda()


def _data(rows, d_in, d_out, n, dtype, order="mixed", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    return dict(x=r(rows, d_in).to(dtype), weight=(r(n, d_out, d_in) * d_in ** -0.5).to(dtype), bias=r(n, d_out).to(dtype), index=_index(rows, n, order, seed)), \
        r(rows, d_out).to(dtype)


def _steps(k):
    """Of the sizes of k terms, what a sum in single precision may be off by: 8 (sqrt(k) + 2) u, which random roundings stay below."""
    return 8 * (k ** 0.5 + 2) * U


def _reference(x, weight, bias, index, dy=None):
    """Results in 64 bits, and bounds of what sums in single precision are off by."""
    x, weight, index = x.double(), weight.double(), index.long()
    n, d_out, d_in = weight.shape
    rows = x.shape[0]
    zero = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)          # noqa: E731
    if dy is None:
        y, off = zero(rows, d_out), zero(rows, d_out)
    else:
        dy = dy.double()
        dx, dw, db = zero(rows, d_in), zero(n, d_out, d_in), zero(n, d_out)
        off_x, off_w, off_b = zero(rows, d_in), zero(n, d_out, d_in), zero(n, d_out)
    for g in range(n):
        at = (index == g).nonzero()[:, 0]
        if not len(at):
            continue
        w = weight[g]
        if dy is None:
            b = 0.0 if bias is None else bias[g].double()
            y[at] = x[at] @ w.t() + b
            off[at] = (x[at].abs() @ w.abs().t() + (0.0 if bias is None else b.abs())) * _steps(d_in + 1)
        else:
            d = dy[at]
            dx[at], off_x[at] = d @ w, (d.abs() @ w.abs()) * _steps(d_out)
            dw[g], off_w[g] = d.t() @ x[at], (d.abs().t() @ x[at].abs()) * _steps(len(at))
            db[g], off_b[g] = d.sum(0), d.abs().sum(0) * _steps(len(at))
    if dy is None:
        return {"y": (y, off)}
    return {"dx": (dx, off_x), "dweight": (dw, off_w), "dbias": (db, off_b)}


def _close(got, want, off, dtype, what=""):
    assert got.dtype == dtype and got.shape == want.shape
    bad = ~((got.double() - want).abs() <= off + UNIT[dtype] * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist())


def _check(data, dy, backward=True):
    from symmetrix_amd import finetune
    dtype = data["x"].dtype
    _close(finetune.grouped_linear_forward(**data), *_reference(**data)["y"], dtype, "y")
    if backward:
        got = dict(zip(("dx", "dweight", "dbias"), finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"])))
        for k, (want, off) in _reference(**data, dy=dy).items():
            _close(got[k], want, off, dtype, k)


SHAPES = [  # rows, d_in, d_out, groups
    (1, 1, 1, 1), (1, 32, 32, 1), (1, 96, 128, 3), (2, 64, 48, 5), (7, 33, 65, 2), (15, 128, 96, 4), (16, 256, 512, 16), (17, 200, 136, 7), (24, 192, 128, 3),
    (33, 1, 70, 3), (33, 70, 1, 3), (40, 40, 24, 40), (63, 129, 257, 6), (64, 512, 512, 9), (65, 96, 96, 4), (66, 264, 72, 30), (100, 320, 64, 3), (127, 256, 256, 64),
    (128, 257, 255, 11), (129, 1024, 512, 12), (255, 96, 192, 100), (256, 2048, 1000, 8), (257, 640, 640, 5), (500, 128, 128, 300), (513, 136, 120, 2),
    (1000, 192, 288, 12), (1023, 500, 300, 17), (2049, 256, 512, 12), (4097, 96, 128, 33), (2000, 72, 520, 1), (3001, 130, 66, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(shape, dtype):
    for order in ("mixed", "runs", "few"):
        _check(*_data(*shape, NAMES[dtype], order, seed=sum(shape)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("order", ["own", "one", "none"])
def test_orders(order, dtype):
    for shape in ((16, 512, 256, 16), (64, 160, 96, 16), (300, 160, 224, 40), (2000, 96, 96, 3)):
        _check(*_data(*shape, NAMES[dtype], order))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_larger(dtype):
    for shape, order in (((20_011, 256, 512, 12), "mixed"), ((1531, 2080, 1184, 24), "runs"), ((6000, 1024, 768, 3), "mixed"), ((9001, 96, 64, 500), "mixed")):
        _check(*_data(*shape, NAMES[dtype], order))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_most_groups(dtype):
    _check(*_data(5000, 32, 16, 4096, NAMES[dtype], "mixed"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_single_tokens(dtype):
    """One row, and a few with a group each, through wide layers."""
    for rows in (1, 2, 5, 16, 17, 48, 64, 80):
        _check(*_data(rows, 2048, 520, 64, NAMES[dtype], "mixed", seed=rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_strides(dtype):
    """Rows of wider arrays at any alignment, matrices apart, one matrix for all groups; results are those of contiguous ones."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    for rows, d_in, d_out in ((40, 64, 48), (700, 96, 80), (1500, 320, 256)):
        x, w = torch.randn(rows, 2 * d_in + 3, device="cuda").to(dtype), torch.randn(8, d_out + 1, 2 * d_in + 1, device="cuda").to(dtype)
        dy, index = torch.randn(rows, d_out + 5, device="cuda").to(dtype), _index(rows, 4, "mixed")
        for a in (0, 1, 8):
            xs, ws, ds = x[:, a:a + d_in], w[::2, 1:, a:a + d_in], dy[:, a % 5:a % 5 + d_out]
            data = dict(x=xs, weight=ws, bias=None, index=index)
            _check(data, ds)
        data = dict(x=x[:, :d_in], weight=w[:1, 1:, :d_in].expand(4, -1, -1), bias=None, index=index)
        _check(data, dy[:, :d_out])
    many = finetune.grouped_linear_forward(x[:600, :d_in].reshape(3, 4, 50, d_in), w[:4, 1:, :d_in], None, index[:600].view(3, 4, 50))
    assert many.shape == (3, 4, 50, d_out)
    assert torch.equal(many.view(600, d_out), finetune.grouped_linear_forward(x[:600, :d_in], w[:4, 1:, :d_in], None, index[:600]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_rows_do_not_depend_on_where_they_are(dtype):
    """The rows' results do not change with the groups given beforehand, nor with other streams."""
    from symmetrix_amd import finetune
    for shape in ((48, 256, 128, 8), (900, 128, 160, 6)):
        data, dy = _data(*shape, NAMES[dtype])
        groups = finetune.group_rows(data["index"], shape[3])
        sorted_first = dict(data, index=groups)
        assert torch.equal(finetune.grouped_linear_forward(**data), finetune.grouped_linear_forward(**sorted_first))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = finetune.grouped_linear_backward(dy, data["x"], data["weight"], groups)
        side.synchronize()
        for a, b in zip(there, finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"])):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("rows", [20, 90, 1200])
def test_infinities_and_bad_indices_stay_with_their_rows(rows, dtype):
    from symmetrix_amd import finetune
    for d_in, d_out in ((96, 80), (101, 63), (192, 256)):
        data, dy = _data(rows, d_in, d_out, 5, NAMES[dtype], "mixed", seed=rows)
        clean = finetune.grouped_linear_forward(**data)
        clean_back = finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"])
        x, weight, index, back = data["x"].clone(), data["weight"].clone(), data["index"].clone(), dy.clone()
        index[0], index[1], index[2], index[3] = 1, 5, -1, -7
        weight[2] = float("nan")          # of another group
        x[1:4], back[1:4] = float("inf"), float("nan")          # rows without a group: no part in anything
        x[0, 3] = float("inf")
        y = finetune.grouped_linear_forward(x, weight, data["bias"], index)
        assert y[1].isnan().all() and y[3].isnan().all() and not y[2].any()
        want = x[0].double()[None, 3:4] * weight[1][:, 3].double()
        assert torch.equal(y[0].double(), want) or not y[0].isfinite().any()
        rest = (index != 2) & (torch.arange(rows, device="cuda") > 3)
        assert torch.equal(y[rest], clean[rest]) or (y[rest] - clean[rest]).abs().max() <= 2 * UNIT[NAMES[dtype]] * clean[rest].abs().max()
        assert y[(index == 2)].isnan().all()
        dx, dw, db = finetune.grouped_linear_backward(back, x, weight, index)
        assert dx[1].isnan().all() and dx[3].isnan().all() and not dx[2].any()
        for g in (0, 3, 4):          # (groups whose rows are as they were)
            if not (data["index"][:4] == g).any():
                assert dw[g].isfinite().all() and db[g].isfinite().all()
                assert (dw[g].double() - clean_back[1][g].double()).abs().max() <= 1e-2 * clean_back[1][g].double().abs().max()
        assert dw[1][:, 3].isfinite().sum() == 0 and dw[1][:, :3].isfinite().all() and dw[1][:, 4:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [30, 400])
def test_large_and_small_numbers(rows):
    """Numbers over the whole range of single precision keep their precision."""
    from symmetrix_amd import finetune
    for size in (2.0 ** -100, 2.0 ** -60, 2.0 ** 60, 2.0 ** 110):
        data, dy = _data(rows, 96, 64, 3, torch.float32)
        data["x"] *= size
        data["weight"] *= 2.0 ** -20
        data["bias"] = None
        y = finetune.grouped_linear_forward(**data)
        want, off = _reference(**data)["y"]
        assert ((y.double() - want).abs() <= off + U * want.abs() + 2.0 ** -149).all()
        dx, dw, db = finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"])
        for k, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
            want, off = _reference(**data, dy=dy)[k]
            assert ((got.double() - want).abs() <= off + U * want.abs() + 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_empty_calls(dtype):
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    index = torch.zeros(0, dtype=torch.int32, device="cuda")
    x, w, b = torch.zeros(0, 24, device="cuda", dtype=dtype), torch.ones(3, 16, 24, device="cuda", dtype=dtype), torch.ones(3, 16, device="cuda", dtype=dtype)
    assert finetune.grouped_linear_forward(x, w, b, index).shape == (0, 16)
    dx, dw, db = finetune.grouped_linear_backward(x.new_zeros(0, 16), x, w, index)
    assert dx.shape == (0, 24) and not dw.any() and not db.any()
    for rows in (5, 100):
        none = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
        x = torch.ones(rows, 24, device="cuda", dtype=dtype)
        assert not finetune.grouped_linear_forward(x, w[:0], b[:0], none).any()
        dx, dw, db = finetune.grouped_linear_backward(x.new_ones(rows, 16), x, w[:0], none)
        assert not dx.any() and dw.shape == (0, 16, 24) and db.shape == (0, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_parts_that_are_asked_for(dtype):
    from symmetrix_amd import finetune
    data, dy = _data(700, 96, 64, 5, NAMES[dtype])
    every = finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"])
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, False, False)):
        for k, got, want, asked in zip(range(3), finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"], need), every, need):
            if not asked:
                assert got is None
            elif k == 2 and not need[1]:          # (alone, and beside the weights' gradient: sums in another order)
                _close(got, *_reference(**data, dy=dy)["dbias"], NAMES[dtype])
            else:
                assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 500])
def test_differentiated(rows):
    from symmetrix_amd import finetune
    data, c = _data(rows, 40, 24, 4, torch.float32)
    leaves = [data[k].requires_grad_() for k in ("x", "weight", "bias")]
    (finetune.grouped_linear(**data) * c).sum().backward()
    with torch.no_grad():
        for a, b in zip((t.grad for t in leaves), finetune.grouped_linear_backward(c, data["x"], data["weight"], data["index"])):
            assert torch.equal(a, b)
        # against differences: the sum is linear in each of the three
        for k, t in zip(("x", "weight", "bias"), leaves):
            e = torch.randn_like(t)
            f = lambda v: (finetune.grouped_linear(**dict(data, **{k: v})).double() * c).sum()          # noqa: E731
            change = float(f(t + e) - f(t - e)) / 2
            size = sum(float((u.grad.double().abs() * u.abs()).sum()) for u in leaves) + float((t.grad.double().abs() * e.abs()).sum()) + float(c.abs().sum())
            assert abs(change - float((t.grad.double() * e).sum())) <= 64 * _steps(40) * size
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(finetune.grouped_linear(**data).square().sum(), data["x"], create_graph=True)[0].sum(), data["weight"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("rows", [30, 1000])
def test_captured(rows, dtype):
    from symmetrix_amd import finetune
    data, dy = _data(rows, 128, 96, 6, NAMES[dtype])
    run = lambda: (finetune.grouped_linear_forward(**data), *finetune.grouped_linear_backward(dy, data["x"], data["weight"], data["index"]))          # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        data["index"].copy_(_index(rows, 6, ("mixed", "one", "few", "none")[k], seed=k))
        data["x"].normal_()
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals():
    from symmetrix_amd import finetune
    data, dy = _data(10, 16, 8, 3, torch.float32)
    forward = lambda **k: finetune.grouped_linear_forward(**dict(data, **k))          # noqa: E731
    for wrong in (dict(x=data["x"].double()), dict(weight=data["weight"].half()), dict(bias=data["bias"].half()), dict(index=data["index"].long())):
        with pytest.raises(TypeError):
            forward(**wrong)
    for wrong in (dict(x=data["x"][:, :9]), dict(weight=data["weight"][0]), dict(bias=data["bias"][:2]), dict(index=data["index"][:9]), dict(x=data["x"].cpu()),
                  dict(index=finetune.group_rows(data["index"], 4)), dict(weight=data["weight"].new_zeros(finetune.MAX_GROUPS + 1, 8, 16), bias=None),
                  dict(index=torch.zeros(20, dtype=torch.int32, device="cuda")[::2])):
        with pytest.raises(ValueError):
            forward(**wrong)
    with pytest.raises(ValueError):
        finetune.grouped_linear_backward(dy[:, :5], data["x"], data["weight"], data["index"])
    with pytest.raises(TypeError):
        finetune.grouped_linear_backward(dy.half(), data["x"], data["weight"], data["index"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_apart_by_more_than_four_gigabytes(dtype):
    """Offsets of rows and matrices that 32 bits do not hold, in tiles of every size."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    rows, d_in, d_out, n = 80_011, 64, 72, 3
    store = torch.empty(rows * 40_000, device="cuda", dtype=dtype)          # 6.4 or 12.8 GB, of which little is touched
    x, dy = store.view(rows, 40_000)[:, :d_in], store.view(rows, 40_000)[:, 8_000:8_000 + d_out]
    g = torch.Generator(device="cuda").manual_seed(1)
    x.normal_(generator=g)
    dy.normal_(generator=g)
    each = store.numel() // (n + 1) // 8 * 8
    weight = store[16_000:].as_strided((n, d_out, d_in), (each, 40_000, 1))          # (among the rows)
    weight.normal_(generator=g).mul_(d_in ** -0.5)
    assert rows * 40_000 * store.element_size() > 1 << 32 and each * n * store.element_size() > 1 << 32
    data = dict(x=x, weight=weight, bias=None, index=_index(rows, n, "mixed"))
    _check(data, dy)
    some = slice(rows - 50, rows)
    _check(dict(data, x=x[some], index=data["index"][some]), dy[some])
    far = dict(data, x=x[some].contiguous(), index=data["index"][some])
    assert torch.equal(finetune.grouped_linear_forward(**far), finetune.grouped_linear_forward(**dict(data, x=x[some], index=far["index"])))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_many_groups_of_several_tiles(dtype):
    """More groups than a wavefront has lanes, of no rows, of one, and of several tiles and pieces."""
    for rows, d_in, d_out, n, order in ((9000, 64, 40, 63, "few"), (9000, 64, 40, 62, "few"), (20_000, 72, 64, 700, "few"), (4000, 33, 20, 2049, "one"), (30_000, 64, 64, 65, "mixed")):
        _check(*_data(rows, d_in, d_out, n, NAMES[dtype], order))


@pytest.mark.gpu
def test_every_sum_not_finite():
    """A row of infinities and NaN makes its own results what the formula says, whatever else shares its tile."""
    from symmetrix_amd import finetune
    for rows in (50, 300, 3000):
        data, _ = _data(rows, 40, 24, 3, torch.float32, seed=rows)
        data["index"].clamp_(min=0)
        data["x"][::7] = float("inf")
        data["x"][3::7] = float("nan")
        data["weight"].abs_()
        data["weight"][2].neg_()
        y = finetune.grouped_linear_forward(**data)
        high, low = torch.full((24,), float("inf"), device="cuda"), torch.full((24,), float("-inf"), device="cuda")
        for i in range(0, rows, 7):
            assert torch.equal(y[i], low if int(data["index"][i]) == 2 else high)
        assert y[3::7].isnan().all()
        others = torch.ones(rows, dtype=torch.bool, device="cuda")
        others[::7] = others[3::7] = False
        want, off = _reference(**{**data, "x": torch.where(others[:, None], data["x"], 0.0)})["y"]
        _close(y[others], want[others], off[others], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_long_groups_in_few_tiles(dtype):
    """Sums over many rows with eight steps under way, whose rows' numbers come from memory while others' tiles do."""
    from symmetrix_amd import finetune
    for rows, d_in, d_out, n in ((2000, 96, 96, 3), (1500, 64, 64, 2), (900, 64, 136, 1), (5000, 128, 64, 4), (3000, 32, 200, 3), (8000, 64, 64, 9)):
        data, dy = _data(rows, d_in, d_out, n, NAMES[dtype], "own", seed=rows)
        _check(data, dy)
        args = dy, data["x"], data["weight"], data["index"], (False, True, True)
        first = finetune.grouped_linear_backward(*args)
        for _ in range(20):
            again = finetune.grouped_linear_backward(*args)
            assert torch.equal(again[1], first[1]) and torch.equal(again[2], first[2])
