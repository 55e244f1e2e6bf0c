"""Rows sorted by group, rows of a table by index and the table's gradient, against the definitions: sizes around the blocks of the sort,
indices without a group and out of range, types, widths, strides, refusals."""
import pytest

torch = pytest.importorskip("torch")

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NAMES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24


def _index(rows, n, kind="mixed", seed=0):
    """mixed: some without a group; bad: some out of range too; skewed: most in a few; runs: neighbours alike; one; none"""
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        index = torch.full((rows,), max(n - 1, -1))
    elif kind == "none":
        index = torch.full((rows,), -1)
    elif kind == "skewed":
        index = (torch.rand(rows, generator=g, dtype=torch.float64) ** 4 * n).long().clamp(max=n - 1)
    else:
        index = torch.randint(-1, n, (rows,), generator=g)
        if kind == "runs":
            index = index.sort().values
        if kind == "bad" and rows:
            wrong = torch.tensor([n, n + 1, -2, 2 ** 31 - 1, -2 ** 31])
            at = torch.rand(rows, generator=g) < 0.2
            index[at] = wrong[torch.randint(0, 5, (rows,), generator=g)][at]
    return index.to(torch.int32).cuda()


def _expected_order(index, n):
    key = torch.where((index >= 0) & (index < n), index, torch.where(index == -1, n, n + 1)).long()
    order = torch.argsort(key, stable=True)
    return order, torch.searchsorted(key[order], torch.arange(n + 2, device=index.device))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 1, 2, 10, 126, 127, 254, 255, 1022, 1023, 5000, 100_000, 1_100_000])
@pytest.mark.parametrize("rows", [0, 1, 63, 64, 65, 1023, 1025, 2047, 2048, 2049, 2561, 5000, 70_001])
def test_rows_are_sorted(rows, n):
    from symmetrix_amd import finetune
    for kind in ("mixed", "bad", "skewed", "runs", "one", "none"):
        if n == 0 and kind == "skewed":
            continue
        index = _index(rows, n, kind, seed=rows + n)
        groups = finetune.group_rows(index, n)
        order, offsets = _expected_order(index, n)
        assert torch.equal(groups.order.long(), order), kind
        assert torch.equal(groups.offsets.long(), offsets), kind


@pytest.mark.gpu
def test_many_rows_are_sorted():
    from symmetrix_amd import finetune
    for n in (7, 40_000):
        index = _index(1_500_011, n, "bad", seed=n)
        groups = finetune.group_rows(index, n)
        order, offsets = _expected_order(index, n)
        assert torch.equal(groups.order.long(), order) and torch.equal(groups.offsets.long(), offsets)


# rows, entries, dim
SHAPES = [(1, 1, 1), (1, 5, 17), (2, 3, 64), (5, 2, 33), (24, 10, 192), (31, 100, 256), (63, 7, 1), (64, 4, 255), (65, 40, 257), (100, 1000, 8), (255, 89, 128),
          (257, 3, 512), (1000, 1, 96), (1023, 17, 1000), (2049, 89, 256), (2050, 5000, 40), (4097, 300, 24), (5000, 2, 264), (20_011, 89, 256), (3001, 70_001, 20)]


def _close(got, want, off, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    assert ((got.double() - want).abs() <= off + UNIT[dtype] * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -25).all()


def _sums(dy, index, n):
    """Sums of rows by entry in 64 bits, and bounds of what sums in single precision of as many terms are off by: 8 (sqrt(terms) + 2) u of the
    terms' sizes, which random roundings stay below."""
    has = (index >= 0) & (index < n)
    at, rows = index[has].long(), dy[has].double()
    zero = torch.zeros(n, dy.shape[-1], dtype=torch.float64, device=dy.device)
    count = torch.bincount(at, minlength=n).double()[:, None]
    return zero.index_add(0, at, rows), zero.index_add(0, at, rows.abs()) * 8 * (count.sqrt() + 2) * U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_table_and_gradient(shape, dtype):
    from symmetrix_amd import finetune
    rows, n, dim = shape
    dtype = NAMES[dtype]
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    table, dy = (torch.randn(k, dim, generator=g, device="cuda").to(dtype) for k in (n, rows))
    for kind, scale in (("mixed", 1.0), ("skewed", 0.37109375), ("bad", -16.0), ("one", 1.0), ("none", 1.0)):
        index = _index(rows, n, kind, seed=rows)
        y = finetune.embedding_forward(table, index, scale)
        has = (index >= 0) & (index < n)
        want = torch.zeros(rows, dim, dtype=torch.float64, device="cuda")
        want[has] = scale * table[index[has].long()].double()
        assert y[~has & (index != -1)].isnan().all()
        y = torch.where((~has & (index != -1))[:, None], torch.zeros_like(y), y)
        _close(y, want, 0.0, dtype)
        dtable = finetune.embedding_backward(dy, index, n, scale)
        want, off = _sums(dy, index, n)
        _close(dtable, scale * want, abs(scale) * off, dtype)
        again = finetune.embedding_backward(dy, finetune.group_rows(index, n), n, scale)
        assert torch.equal(again, dtable)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_large_table(dtype):
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    g = torch.Generator(device="cuda").manual_seed(1)
    for rows, n, dim in ((3001, 200_003, 100), (16_381, 32_000, 512), (50_000, 3, 260)):
        dy = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
        index = _index(rows, n, "skewed", seed=rows)
        want, off = _sums(dy, index, n)
        _close(finetune.embedding_backward(dy, index, n, 2.0), 2 * want, 2 * off, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_strides_and_shapes(dtype):
    """Rows of wider arrays, odd distances and starts, no rows, indices of several dimensions, another stream."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    wide = torch.randn(90, 301, device="cuda").to(dtype)
    index = _index(70, 90, "mixed")
    for a, b in ((0, 64), (1, 65), (3, 300), (7, 8)):
        table = wide[:, a:b]
        assert torch.equal(finetune.embedding_forward(table, index, 3.0), finetune.embedding_forward(table.contiguous(), index, 3.0))
        dy = wide[:70, a:b]
        assert torch.equal(finetune.embedding_backward(dy, index, 90, 3.0), finetune.embedding_backward(dy.contiguous(), index, 90, 3.0))
    some = index[:60].view(3, 4, 5)
    y = finetune.embedding_forward(wide, some)
    assert y.shape == (3, 4, 5, 301) and torch.equal(y.view(60, 301), finetune.embedding_forward(wide, index[:60]))
    assert torch.equal(finetune.embedding_backward(y, some, 90), finetune.embedding_backward(y.view(60, 301), index[:60], 90))
    none = index[:0]
    assert finetune.embedding_forward(wide, none).shape == (0, 301)
    assert not finetune.embedding_backward(wide[:0], none, 90).any()
    assert finetune.embedding_backward(wide[:70], index, 0).shape == (0, 301)
    assert finetune.embedding_forward(wide[:0], torch.full((4,), -1, dtype=torch.int32, device="cuda")).eq(0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = finetune.embedding_backward(wide[:70], index, 90)
    side.synchronize()
    assert torch.equal(there, finetune.embedding_backward(wide[:70], index, 90))


@pytest.mark.gpu
def test_infinities_stay_with_their_entries():
    from symmetrix_amd import finetune
    table = torch.ones(5, 40, device="cuda")
    table[2], table[3, 7] = float("inf"), float("nan")
    index = torch.tensor([0, 2, 3, 4, -1, 2], dtype=torch.int32, device="cuda")
    y = finetune.embedding_forward(table, index, 2.0)
    assert y[[1, 5]].isinf().all() and y[2, 7].isnan() and int(y.isnan().sum()) == 1 and not y[4].any() and y[[0, 3]].eq(2).all()
    dy = torch.ones(6, 40, device="cuda")
    dy[1], dy[4] = float("inf"), float("nan")          # (a row without an entry has no part in any)
    d = finetune.embedding_backward(dy, index, 5, 1.0)
    assert d[2].isinf().all() and d[[0, 3, 4]].eq(1).all() and not d[1].any()


@pytest.mark.gpu
def test_differentiated():
    from symmetrix_amd import finetune
    index = _index(50, 9, "mixed")
    table = torch.randn(9, 33, device="cuda", requires_grad=True)
    c = torch.randn(50, 33, device="cuda")
    (finetune.embedding(table, index, 0.5) * c).sum().backward()
    assert torch.equal(table.grad, finetune.embedding_backward(c, index, 9, 0.5))
    # against differences, which are exact but for roundings: the sum is linear in the table
    e = torch.randn(9, 33, device="cuda")
    f = lambda t: (finetune.embedding(t, finetune.group_rows(index, 9), 0.5).double() * c).sum()          # noqa: E731
    with torch.no_grad():
        change = float(f(table + e) - f(table - e)) / 2
    size = float((table.grad.double().abs() * (table.detach().abs() + e.abs())).sum()) + float(c.abs().double().sum())
    assert abs(change - float((table.grad.double() * e).sum())) <= 4 * 60 * U * size
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(finetune.embedding(table, index).square().sum(), table, create_graph=True)[0].sum(), table)


@pytest.mark.gpu
def test_captured():
    from symmetrix_amd import finetune
    index, dy = _index(3000, 200, "mixed"), torch.randn(3000, 64, device="cuda")
    table = torch.randn(200, 64, device="cuda")
    run = lambda: (finetune.embedding_forward(table, index, 2.0), finetune.embedding_backward(dy, index, 200, 2.0))          # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = run()
    for k in range(4):
        index.copy_(_index(3000, 200, "bad", seed=k))
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert torch.equal(y.nan_to_num(7.0), want[0].nan_to_num(7.0)) and torch.equal(d, want[1])


@pytest.mark.gpu
def test_refusals():
    from symmetrix_amd import finetune
    table, index = torch.zeros(5, 8, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    groups = finetune.group_rows(index, 5)
    with pytest.raises(TypeError):
        finetune.embedding_forward(table, index.long())
    with pytest.raises(TypeError):
        finetune.embedding_forward(table.double(), index)
    with pytest.raises(TypeError):
        finetune.group_rows(index.float(), 5)
    for call in (lambda: finetune.embedding_forward(table.cpu(), index), lambda: finetune.embedding_forward(table[0], index),
                 lambda: finetune.embedding_forward(table, index, float("nan")), lambda: finetune.embedding_forward(table, torch.zeros(12, dtype=torch.int32, device="cuda")[::2]),
                 lambda: finetune.embedding_backward(torch.zeros(5, 8, device="cuda"), index, 5), lambda: finetune.embedding_backward(torch.zeros(6, 8, device="cuda"), index, -1),
                 lambda: finetune.embedding_backward(torch.zeros(6, 8, device="cuda"), groups, 6), lambda: finetune.group_rows(index, -1),
                 lambda: finetune.group_rows(index, finetune.MAX_ENTRIES + 1), lambda: finetune.group_rows(index.cpu(), 5)):
        with pytest.raises(ValueError):
            call()
    index.add_(1)          # the rows are sorted by what the index held before
    with pytest.raises(ValueError):
        finetune.embedding_forward(table, groups)


@pytest.mark.gpu
def test_tables_and_results_of_more_than_four_gigabytes():
    """Numbers that are powers of two tell a row, and sums of a few of them are exact."""
    from symmetrix_amd import finetune
    entries, dim, rows = 70_001, 40_008, 70_003
    table = torch.empty(entries, dim, device="cuda", dtype=torch.bfloat16)
    marks = 2.0 ** (torch.arange(entries, device="cuda") % 15).to(torch.bfloat16)
    table.copy_(marks[:, None].expand(-1, dim))
    index = torch.tensor([entries - 1, 0, -1, entries - 2, 53_688, 53_689], dtype=torch.int32, device="cuda")
    y = finetune.embedding_forward(table, index)
    want = torch.where(index >= 0, marks[index.long().clamp(min=0)], 0.0)
    assert torch.equal(y, want[:, None].expand(-1, dim).to(torch.bfloat16))
    del y
    index = (torch.arange(rows, device="cuda") * 7 % 5).to(torch.int32)
    y = finetune.embedding_forward(table, index)
    assert y.numel() * 2 > 1 << 32 and torch.equal(y, marks[index.long()][:, None].expand(-1, dim))
    del table
    # the gradient: 70 003 rows of which each adds its mark to one of 30 000 entries, two or three an entry
    index = (torch.arange(rows, device="cuda") % 30_000).to(torch.int32)
    got = finetune.embedding_backward(y, index, 30_000)
    each = torch.zeros(30_000, device="cuda", dtype=torch.float64).index_add_(0, index.long(), y[:, 0].double())
    assert torch.equal(got, each.to(torch.bfloat16)[:, None].expand(-1, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
def test_few_of_many_entries(dtype):
    """More entries than rows: zeros beside the sort, at every alignment of the table's gradient, and one entry with half of the rows."""
    from symmetrix_amd import _lib, finetune
    import ctypes as C
    dtype = NAMES[dtype]
    for rows, n, dim in ((129, 5000, 7), (1500, 1500, 33), (4096, 9001, 64), (4097, 4100, 129), (9000, 40_000, 24), (5000, 70_000, 520)):
        g = torch.Generator(device="cuda").manual_seed(rows)
        dy = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
        index = _index(rows, n, "bad", seed=n)
        index[::2] = n - 3
        want, off = _sums(dy, index, n)
        got = finetune.embedding_backward(dy, index, n)
        _close(got, want, off, dtype)
        assert torch.equal(got, finetune.embedding_backward(dy, finetune.group_rows(index, n), n))
        # the C call into the middle of an array: what is beside it stays
        size, kind = C.c_long(), list(NAMES.values()).index(dtype)          # (as SMX_TYPE_* are numbered)
        lib = finetune._lib_functions()
        _lib.check(lib.smx_embedding_backward_workspace(kind, rows, n, dim, C.byref(size)))
        work = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        for shift in (1, 3, 8):
            room = torch.full((n * dim + 16,), 7.0, device="cuda", dtype=dtype)
            out = room[shift:shift + n * dim]
            _lib.check(lib.smx_embedding_backward(kind, rows, n, dim, dy.data_ptr(), dim, index.data_ptr(), 0, 0, 1.0, out.data_ptr(), work.data_ptr(), size.value,
                                                  torch.cuda.current_stream().cuda_stream))
            assert torch.equal(out.view(n, dim), got) and (room[:shift] == 7).all() and (room[shift + n * dim:] == 7).all()
