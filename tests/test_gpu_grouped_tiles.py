"""Products by group in the tiles that large calls take, every way of cutting the last round of them; infinities in every type and way; offsets
of more than 32 bits in large tiles."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_grouped_linear import NAMES, _close, _reference  # noqa: E402

CUS = 256


def _tile(rows, groups, cols):
    """The tile of y and dx in 16 bits, of rows at multiples of 16 bytes, as the host takes it (256, 128, or smaller)."""
    used = min(rows, groups)
    for tile in (256, 128):
        across = -(-cols // tile)
        if (rows // tile + used // 2) * across >= 192 and 4 * cols >= 3 * across * tile and (2 if tile == 128 else 1) * rows >= used * tile:
            return tile
    return 64


def _index(counts, none, bad, order, seed=0):
    """Rows of groups of the given sizes, without a group and out of range."""
    n = len(counts)
    wrong = torch.tensor([n, -2, 2 ** 31 - 1])[torch.arange(bad) % 3]
    index = torch.cat([torch.repeat_interleave(torch.arange(n), torch.tensor(counts)), torch.full((none,), -1), wrong])
    if order == "mixed":
        index = index[torch.randperm(len(index), generator=torch.Generator().manual_seed(seed))]
    return index.to(torch.int32).cuda()


# sizes of the groups, rows without one and out of range; tiles of the last round, in row tiles of 256 and 8 columns of tiles
CASES = [
    ([2048, 2047, 1848, 2148], 0, 0, 8),                    # cut in four; the last tile has 100 rows, half of its parts none
    ([2048, 2047, 1848, 2276], 0, 0, 8),                    # 228 rows in it
    ([1793, 2048, 1500, 2000], 300, 5, 8),                  # rows without a group and out of range in cut tiles
    ([2560, 2561, 2050, 2005], 0, 0, 48),                   # cut in four, two bands
    ([2816, 2561, 2561, 2761], 0, 0, 96),                   # cut in two
    ([2816, 2570, 2561, 2760], 130, 0, 104),                # and with rows without a group
    ([1536, 1536, 1536, 1536], 0, 0, 192),                  # one round, not cut
    ([2048, 2048, 2048, 2048], 0, 0, 0),                    # whole rounds
    ([500] * 30 + [60] * 34 + [2560], 0, 0, 64),            # more groups than a wavefront has lanes for, in four
    ([500] * 30 + [60] * 34 + [3500], 0, 0, 96),            # and in two
    ([500] * 30 + [0] * 20 + [60] * 33 + [3584], 1000, 3, 128),         # groups without rows among them
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("terms", [72, 328])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_largest_tiles(case, terms, dtype):
    """Tiles of 256 x 256 for y and dx, the last column of them not full, steps that are not whole."""
    from symmetrix_amd import finetune
    counts, none, bad, last = CASES[case]
    dtype, wide, n = NAMES[dtype], 2040, len(counts)
    index = _index(counts, none, bad, "runs" if case % 3 == 1 else "mixed", case)
    rows = len(index)
    tiles = sum(-(-c // 256) for c in [*counts, none, bad]) * -(-wide // 256)
    assert _tile(rows, n, wide) == 256 and tiles % CUS == last
    g = torch.Generator(device="cuda").manual_seed(case)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)          # noqa: E731
    out = (index < -1) | (index >= n)
    x, w, b = r(rows, terms), (r(n, wide, terms).float() * terms ** -0.5).to(dtype), r(n, wide)
    y = finetune.grouped_linear_forward(x, w, b, index)
    assert y[out].isnan().all() and not y[index == -1].any()
    y[out] = 0
    _close(y, *_reference(x, w, b, index)["y"], dtype, "y")
    x, w, dy = r(rows, wide), (r(n, terms, wide).float() * terms ** -0.5).to(dtype), r(rows, terms)
    dx, dw, db = finetune.grouped_linear_backward(dy, x, w, index)
    assert dx[out].isnan().all() and not dx[index == -1].any()
    dx[out] = 0
    for name, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
        _close(got, *_reference(x, w, None, index, dy)[name], dtype, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("wide,tile", [(1536, 256), (384, 128)])
def test_large_tiles_of_rows_and_matrices_far_apart(wide, tile, dtype):
    """Rows within and beyond what 32 bits reach (beyond it by way of registers), matrices 4 GB apart and more."""
    dtype, terms, n, apart = NAMES[dtype], 64, 3, 1 << 18
    from symmetrix_amd import finetune
    # (8 191 rows that begin 512 KB apart end just below 4 GB, 8 193 above)
    store = torch.empty(8193 * apart, device="cuda", dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(wide)
    each = (1 << 31) + 8 * 1237
    far = torch.empty(each * (n - 1) + wide * terms, device="cuda", dtype=dtype)
    for rows in (8191, 8193):
        assert _tile(rows, n, wide) == tile and (rows * apart * 2 < 1 << 32) == (rows == 8191)
        lines = store[:rows * apart].view(rows, apart)
        index = torch.randint(-1, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
        for d_in, d_out in ((terms, wide), (wide, terms)):
            w = far.as_strided((n, d_out, d_in), (each, d_in, 1))
            w.copy_(torch.randn(n, d_out, d_in, generator=g, device="cuda") * d_in ** -0.5)
            x, dy = lines[:, :d_in], lines[:, apart - d_out:]
            x.copy_(torch.randn(rows, d_in, generator=g, device="cuda"))
            dy.copy_(torch.randn(rows, d_out, generator=g, device="cuda"))
            if d_out == wide:
                _close(finetune.grouped_linear_forward(x, w, None, index), *_reference(x, w, None, index)["y"], dtype, "y")
            else:
                dx, dw, db = finetune.grouped_linear_backward(dy, x, w, index)
                for name, got in (("dx", dx), ("dweight", dw), ("dbias", db)):
                    _close(got, *_reference(x, w, None, index, dy)[name], dtype, name)


def _signed(inf_or_nan, by):
    """What an infinite number times numbers is, and a finite sum beside it changes nothing of."""
    return inf_or_nan * by.sign()          # (0 times infinity: NaN)


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0, 1.0, -1.0), b.nan_to_num(0.0, 1.0, -1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("rows,d_in,d_out", [(20, 96, 80), (20, 101, 63), (60, 264, 40), (400, 96, 80), (400, 101, 63), (1200, 192, 256), (1200, 130, 257), (9000, 64, 1536)])
def test_an_infinity_goes_where_the_formula_takes_it(rows, d_in, d_out, dtype):
    """One number of x or dy: signs of infinities, NaN only where it meets a zero, the rest as without it."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows + d_in)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)          # noqa: E731
    index = torch.randint(-1, 4, (rows,), generator=g, device="cuda", dtype=torch.int32)
    x, w, b, dy = r(rows, d_in), r(4, d_out, d_in), r(4, d_out), r(rows, d_out)
    for at, column in ((0, 3), (rows - 1, d_in - 1), (rows // 2, d_in // 2)):
        for value in (float("inf"), float("-inf")):
            index[at] = 2
            w[2, ::5, column], dy[at, 1::7] = 0, 0
            clean, clean_dx, clean_dw, clean_db = finetune.grouped_linear_forward(x, w, b, index), *finetune.grouped_linear_backward(dy, x, w, index)
            hot = x.clone()
            hot[at, column] = value
            y = finetune.grouped_linear_forward(hot, w, b, index)
            assert _same(y[at], _signed(value, w[2, :, column]))
            others = torch.arange(rows, device="cuda") != at
            assert torch.equal(y[others], clean[others])
            dx, dw, db = finetune.grouped_linear_backward(dy, hot, w, index)
            assert torch.equal(dx, clean_dx) and torch.equal(db, clean_db)
            assert _same(dw[2, :, column], _signed(value, dy[at]))
            kept = torch.ones_like(dw, dtype=torch.bool)
            kept[2, :, column] = False
            assert torch.equal(dw[kept], clean_dw[kept])
            # and of dy: a row of dx, a row of its group's dW, a number of db
            out = column % d_out
            w[2, out, ::3], x[at, 1::4] = 0, 0
            clean_dx, clean_dw, clean_db = finetune.grouped_linear_backward(dy, x, w, index)
            hot = dy.clone()
            hot[at, out] = value
            dx, dw, db = finetune.grouped_linear_backward(hot, x, w, index)
            assert _same(dx[at], _signed(value, w[2, out])) and torch.equal(dx[others], clean_dx[others])
            assert _same(dw[2, out], _signed(value, x[at])) and db[2, out] == value
            kept = torch.ones_like(dw, dtype=torch.bool)
            kept[2, out] = False
            assert torch.equal(dw[kept], clean_dw[kept])
            kept = torch.ones_like(db, dtype=torch.bool)
            kept[2, out] = False
            assert torch.equal(db[kept], clean_db[kept])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("d_in,d_out", [(40, 24), (41, 23), (64, 1536)])
def test_rows_of_infinities_and_nan(d_in, d_out, dtype):
    """Whole rows of them make their own results what the formula says, whatever else shares their tiles."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    for rows in (50, 300, 9000):
        g = torch.Generator(device="cuda").manual_seed(rows)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)          # noqa: E731
        index = torch.randint(0, 3, (rows,), generator=g, device="cuda", dtype=torch.int32)
        x, w, b = r(rows, d_in), r(3, d_out, d_in).abs() + 2.0 ** -10, r(3, d_out)
        w[2].neg_()
        clean = finetune.grouped_linear_forward(x, w, b, index)
        hot = x.clone()
        hot[::7], hot[3::7] = float("inf"), float("nan")
        y = finetune.grouped_linear_forward(hot, w, b, index)
        want = torch.where(index[::7] == 2, float("-inf"), float("inf"))[:, None].expand(-1, d_out).to(dtype)
        assert torch.equal(y[::7], want) and y[3::7].isnan().all()
        others = torch.ones(rows, dtype=torch.bool, device="cuda")
        others[::7] = others[3::7] = False
        assert torch.equal(y[others], clean[others])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(NAMES))
@pytest.mark.parametrize("rows,d_in,d_out", [(20, 96, 80), (20, 101, 63), (400, 96, 80), (400, 101, 63), (8200, 64, 1536), (8200, 1536, 64)])
def test_subnormal_numbers(rows, d_in, d_out, dtype):
    """Numbers below the normal ones of their type times large ones: whole multiples of one small number, fewer than 2^24 of it in any sum, so that
    sums in single precision are exact and results are rounded once."""
    from symmetrix_amd import finetune
    dtype = NAMES[dtype]
    least, large = {torch.float32: (2.0 ** -149, 2.0 ** 100), torch.bfloat16: (2.0 ** -133, 2.0 ** 100), torch.float16: (2.0 ** -24, 2.0 ** 8)}[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows + d_in)
    whole = lambda high, *s: torch.randint(-high, high + 1, s, generator=g, device="cuda").double()          # noqa: E731
    index = torch.randint(0, 3, (rows,), generator=g, device="cuda", dtype=torch.int32)
    x, dy, w = whole(3, rows, d_in), whole(2, rows, d_out), whole(1, 3, d_out, d_in)
    assert (3 * 2 * rows) < 1 << 24
    small, big = (lambda t: (t * least).to(dtype)), (lambda t: (t * large).to(dtype))
    assert torch.equal(small(x).double(), x * least) and torch.equal(big(dy).double(), dy * large)
    unit = least * large
    y = finetune.grouped_linear_forward(small(x), big(w), None, index)
    dx, _, _ = finetune.grouped_linear_backward(small(dy), small(x), big(w), index)
    _, dw, db = finetune.grouped_linear_backward(big(dy), small(x), big(w), index)
    for k in range(3):
        at = (index == k).nonzero()[:, 0]
        assert torch.equal(y[at], (x[at] @ w[k].t() * unit).to(dtype))
        assert torch.equal(dx[at], (dy[at] @ w[k] * unit).to(dtype))
        assert torch.equal(dw[k], (dy[at].t() @ x[at] * unit).to(dtype))
        assert torch.equal(db[k], (dy[at].sum(0) * large).to(dtype))
    _, _, db = finetune.grouped_linear_backward(small(dy), small(x), big(w), index)
    table = finetune.embedding_backward(small(dy), index, 3)
    for k in range(3):
        want = (dy[index == k].sum(0) * least).to(dtype)
        assert torch.equal(db[k], want) and torch.equal(table[k], want)
