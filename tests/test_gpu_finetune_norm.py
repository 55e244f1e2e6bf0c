"""Layer norm and its gradient against the definition in 64 bits: every way a row is shared, odd widths, strides, alignments,
statistics, refusals, streams and graphs."""
import pytest

torch = pytest.importorskip("torch")

# unit roundoff of the types
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(UNIT)
# Roundings on the way of a sum: at most 32 numbers a thread one after the other (64 in rows beyond 8192), eight in the tree over
# lanes, three over wavefronts; and about ten operations around it.  Single precision bounds of the forms below are this many times
# 2^-24 of the largest term.
STEPS = 64


def _reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    var = (x - mean[..., None]).square().mean(-1)
    rstd = 1 / torch.sqrt(var + eps)
    hat = (x - mean[..., None]) * rstd[..., None]
    y = hat if w is None else hat * w.double()
    return (y if b is None else y + b.double()), mean, rstd, hat


def _data(rows, dim, dtype, seed=0, offset=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    return (r(rows, dim) * 1.5 + offset).to(dtype), (r(dim) * 0.2 + 1).to(dtype), (r(dim) * 0.1).to(dtype), r(rows, dim).to(dtype)


def _check_forward(x, w, b, eps=1e-5):
    from symmetrix_amd import finetune
    y, mean, rstd = finetune.layer_norm_forward(x, w, b, eps)
    want, m, r, hat = _reference(x, w, b, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == x.shape[:-1]
    if not x.numel():
        return
    size = x.double().abs().amax(-1)
    u = 2.0 ** -24
    # mean: a sum's roundings; rstd relative: those of the variance, whose terms are positive, and of a mean that is off
    mean_off = STEPS * u * size
    assert ((mean.double() - m).abs() <= mean_off).all()
    rstd_off = STEPS * u + 0.5 * (mean_off * r).square()
    assert ((rstd.double() / r - 1).abs() <= rstd_off).all()
    big = 1.0 if w is None else w.double().abs()
    off = (hat.abs() * (rstd_off + 4 * u)[..., None] + (mean_off * r)[..., None]) * big
    off = off + (want.abs() + (0 if b is None else b.double().abs())) * (UNIT[x.dtype] * (1 + 2.0 ** -8) + u) + 2.0 ** -25
    assert ((y.double() - want).abs() <= off).all()


def _check_backward(x, w, dy, eps=1e-5, need=(True, True, True)):
    from symmetrix_amd import finetune
    dim = x.shape[-1]
    _, mean, rstd, _ = _reference(x, w, None, eps)
    mean, rstd = mean.float(), rstd.float()
    dx, dw, db = finetune.layer_norm_backward(dy, x, mean, rstd, w, need)
    assert [t is not None for t in (dx, dw, db)] == list(need)
    hat = (x.double() - mean.double()[..., None]) * rstd.double()[..., None]
    g = dy.double() * (1.0 if w is None else w.double())
    u = 2.0 ** -24
    if dx is not None and x.numel():
        s0, s1 = g.mean(-1, keepdim=True), (g * hat).mean(-1, keepdim=True)
        want = rstd.double()[..., None] * (g - s0 - hat * s1)
        terms = rstd.double()[..., None] * (g.abs() + g.abs().mean(-1, keepdim=True) + hat.abs() * (g * hat).abs().mean(-1, keepdim=True))
        # (x - mean, exact to a rounding of the larger of the two)
        near = rstd.double()[..., None] * 2 * u * (x.double().abs() + mean.double().abs()[..., None])
        off = STEPS * u * terms + near * rstd.double()[..., None] * (s1.abs() + (g.abs() * hat.abs()).amax(-1, keepdim=True) + g.abs().amax(-1, keepdim=True) * hat.abs())
        off = off + want.abs() * UNIT[x.dtype] * (1 + 2.0 ** -8) + 2.0 ** -25
        assert ((dx.double() - want).abs() <= off).all()
    for got, each in ((dw, dy.double() * hat), (db, dy.double())):
        if got is None:
            continue
        each = each.reshape(-1, dim)
        want = each.sum(0)
        # a thread's rows one after the other, then the parts of up to 1024 blocks, 16 at a time
        depth = max(x.numel() // dim // 256, 1) + 64 + 32
        slack = (depth + 4) * u * each.abs().sum(0) + 4 * u * (dy.double().abs() * (rstd.double() * (x.double().abs().amax(-1) + mean.double().abs()))[..., None]).reshape(-1, dim).sum(0)
        assert ((got.double() - want).abs() <= slack + want.abs() * UNIT[got.dtype] * (1 + 2.0 ** -8) + 2.0 ** -25).all()


# every way a row is shared among threads, and widths around its ends
WIDTHS = [1, 2, 7, 8, 31, 33, 64, 65, 127, 192, 256, 257, 500, 512, 1000, 1023, 1024, 1025, 2048, 2049, 4096, 4099, 8192, 8193, 20000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_forward(dim, dtype):
    for rows in (1, 5, 130):
        x, w, b, _ = _data(rows, dim, dtype, seed=dim + rows)
        _check_forward(x, w, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_gradient(dim, dtype):
    for rows in (1, 5, 130):
        x, w, _, dy = _data(rows, dim, dtype, seed=dim + rows)
        _check_backward(x, w, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows(dtype):
    x, w, b, dy = _data(20011, 96, dtype)
    _check_forward(x, w, b)
    _check_backward(x, w, dy)
    x, w, b, dy = _data(5003, 2056, dtype)
    _check_forward(x, w, b)
    _check_backward(x, w, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_without_weights_and_with_single_precision_ones(dtype):
    x, w, b, dy = _data(67, 200, dtype)
    _check_forward(x, None, None)
    _check_forward(x, w, None)
    _check_forward(x, None, b)
    _check_forward(x, w.float(), b.float())
    _check_backward(x, None, dy)
    _check_backward(x, w.float(), dy)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        _check_backward(x, w, dy, need=need)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [33, 96, 1000, 9000])
def test_rows_of_wider_arrays(dim, dtype):
    """Columns of a wider array, at an odd offset: rows are neither contiguous nor aligned to more than a number."""
    wide = torch.randn(40, 3 * dim + 5, device="cuda").to(dtype)
    _, w, b, _ = _data(1, dim, dtype)
    x, dy = wide[:, 1:1 + dim], wide[:, dim + 3:2 * dim + 3]
    _check_forward(x, w, b)
    _check_backward(x, w, dy)
    # rows counted backwards in two dimensions, every second row, a column's stride
    _check_forward(wide[::2, :dim], w, b)
    _check_forward(torch.randn(dim, 6, device="cuda").to(dtype).t(), w, b)
    _check_forward(torch.randn(3, 4, dim, device="cuda").to(dtype), w, b)


@pytest.mark.gpu
def test_offset_larger_than_the_spread():
    """The variance is that of centered values: a mean a thousand times the spread costs the digits of x itself and no more."""
    x, w, b, _ = _data(64, 512, torch.float32, offset=1500.0)
    _check_forward(x, w, b)


@pytest.mark.gpu
def test_constant_rows_and_no_rows():
    from symmetrix_amd import finetune
    x = torch.full((3, 96), 2.5, device="cuda")
    y, mean, rstd = finetune.layer_norm_forward(x, None, None, 1e-5)
    assert (y == 0).all() and (mean == 2.5).all() and ((rstd * 1e-5 ** 0.5 - 1).abs() < 1e-6).all()
    x = torch.empty(0, 96, device="cuda")
    y, mean, rstd = finetune.layer_norm_forward(x)
    assert y.shape == (0, 96) and mean.shape == rstd.shape == (0,)
    dx, dw, db = finetune.layer_norm_backward(x, x, mean, rstd, torch.ones(96, device="cuda"))
    assert dx.shape == (0, 96) and (dw == 0).all() and (db == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 700, 3000, 9001])
def test_a_row_that_is_not_finite_keeps_to_itself(dim):
    from symmetrix_amd import finetune
    x, w, b, _ = _data(9, dim, torch.float32)
    clean, mean, rstd = finetune.layer_norm_forward(x, w, b)
    x[4, 3], x[6, dim - 1] = float("nan"), float("inf")
    y, mean, rstd = finetune.layer_norm_forward(x, w, b)
    good = torch.tensor([i for i in range(9) if i not in (4, 6)], device="cuda")
    assert torch.equal(y[good], clean[good])
    assert torch.isnan(y[4]).all() and torch.isnan(y[6]).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    from symmetrix_amd import finetune
    dim, stride = 100, (1 << 31) + 7
    store = torch.empty(2 * stride + dim, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((3, dim), (stride, 1))
    x.copy_(torch.randn(3, dim, device="cuda"))
    _, w, b, dy = _data(3, dim, torch.bfloat16)
    _check_forward(x, w, b)
    _check_backward(x, w, dy)


@pytest.mark.gpu
def test_the_same_bits_every_time():
    from symmetrix_amd import finetune
    x, w, b, dy = _data(9001, 320, torch.float32)
    _, mean, rstd = finetune.layer_norm_forward(x, w, b)
    first = finetune.layer_norm_backward(dy, x, mean, rstd, w)
    for _ in range(3):
        again = finetune.layer_norm_backward(dy, x, mean, rstd, w)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.gpu
def test_automatic_differentiation_and_differences():
    """The derivative along a direction, from values on both sides of a point: the error of second order in h is below h^2 (the third
    derivative of a normalised number along a unit-size direction is of the order of one), values carry STEPS roundings."""
    from symmetrix_amd import finetune
    x, w, b, c = _data(8, 48, torch.float32)
    dirs = [torch.randn_like(t) for t in (x, w, b)]
    x.requires_grad_(); w.requires_grad_(); b.requires_grad_()
    (finetune.layer_norm(x, w, b) * c).sum().backward()
    h = 2.0 ** -7
    for k, t in enumerate((x, w, b)):
        at = [x.detach(), w.detach(), b.detach()]

        def value(side):
            moved = list(at)
            moved[k] = at[k] + side * h * dirs[k]
            return (finetune.layer_norm_forward(*moved)[0].double() * c.double()).sum().item()

        want = (value(1) - value(-1)) / (2 * h)
        got = (t.grad.double() * dirs[k].double()).sum().item()
        scale = c.abs().double().sum().item()
        assert abs(got - want) <= scale * (h * h + STEPS * 2.0 ** -24 / h)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    from symmetrix_amd import finetune
    x, w, b, dy = _data(700, 256, torch.float32)
    want, mean, rstd = finetune.layer_norm_forward(x, w, b)
    grads = finetune.layer_norm_backward(dy, x, mean, rstd, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = finetune.layer_norm_forward(x, w, b)[0]
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, m, r = finetune.layer_norm_forward(x, w, b)
        out = finetune.layer_norm_backward(dy, x, m, r, w)
    for k in range(3):
        x.copy_(torch.randn(700, 256, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want, mean, rstd = finetune.layer_norm_forward(x, w, b)
        assert torch.equal(y, want)
        assert all(torch.equal(p, q) for p, q in zip(out, finetune.layer_norm_backward(dy, x, mean, rstd, w)))


@pytest.mark.gpu
def test_refusals():
    from symmetrix_amd import finetune
    x, w, b, dy = _data(4, 32, torch.float32)
    _, mean, rstd = finetune.layer_norm_forward(x, w, b)
    bad = [
        (ValueError, lambda: finetune.layer_norm_forward(x.cpu(), w.cpu(), b.cpu())),
        (ValueError, lambda: finetune.layer_norm_forward(x, w.cpu(), b)),
        (ValueError, lambda: finetune.layer_norm_forward(x, w[:31], b)),
        (ValueError, lambda: finetune.layer_norm_forward(x, w, b[::2].repeat(2)[::2])),
        (ValueError, lambda: finetune.layer_norm_forward(x, w, b, -1.0)),
        (ValueError, lambda: finetune.layer_norm_forward(x, w, b, float("nan"))),
        (TypeError, lambda: finetune.layer_norm_forward(x.double(), w, b)),
        (TypeError, lambda: finetune.layer_norm_forward(x, w.half(), b.half())),
        (ValueError, lambda: finetune.layer_norm_forward(x.half(), w.half(), b)),
        (ValueError, lambda: finetune.layer_norm_forward(x[:, :0], None, None)),
        (ValueError, lambda: finetune.layer_norm_backward(dy[:3], x, mean, rstd, w)),
        (ValueError, lambda: finetune.layer_norm_backward(dy.half(), x, mean, rstd, w)),
        (ValueError, lambda: finetune.layer_norm_backward(dy, x, mean[:3], rstd, w)),
        (ValueError, lambda: finetune.layer_norm_backward(dy, x, mean.double(), rstd, w)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_c_entry_refuses_without_touching_a_device():
    """Wrong arguments end in a code and a message before a device is looked for."""
    import ctypes as C
    from symmetrix_amd import _lib, finetune
    L = finetune._lib_functions()
    one = 1          # (never read: the calls are refused)
    assert L.smx_layer_norm_forward(7, 0, 1, 8, one, 8, 0, 0, 1e-5, one, 8, 0, 0, 0) == -1
    assert L.smx_layer_norm_forward(1, 2, 1, 8, one, 8, 0, 0, 1e-5, one, 8, 0, 0, 0) == -1
    assert L.smx_layer_norm_forward(0, 0, -1, 8, one, 8, 0, 0, 1e-5, one, 8, 0, 0, 0) == -1
    assert L.smx_layer_norm_forward(0, 0, 1, 0, one, 8, 0, 0, 1e-5, one, 8, 0, 0, 0) == -1
    assert L.smx_layer_norm_forward(0, 0, 1, 8, one, 7, 0, 0, 1e-5, one, 8, 0, 0, 0) == -1
    assert b"strides" in L.smx_last_error()
    assert L.smx_layer_norm_forward(0, 0, 1, 8, 0, 8, 0, 0, 1e-5, one, 8, 0, 0, 0) == -1
    assert L.smx_layer_norm_forward(0, 0, 0, 8, 0, 8, 0, 0, 1e-5, 0, 8, 0, 0, 0) == 0          # no rows: nothing to do
    size = C.c_long()
    assert L.smx_layer_norm_backward_workspace(1000, 64, C.byref(size)) == 0 and size.value > 0
    assert L.smx_layer_norm_backward(0, 0, 1000, 64, one, 64, one, 64, one, one, 0, one, 64, one, one, one, size.value - 1, 0) == -1
    assert b"workspace" in L.smx_last_error()
    with pytest.raises(ValueError):
        _lib.check(-1)


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes():
    """Short rows share a block by 32: 2^22 blocks take 2^27 of them, the rest is another launch."""
    from symmetrix_amd import finetune
    rows, dim = (1 << 27) + 77, 2
    x = torch.zeros(rows, dim, device="cuda")
    some = torch.randn(200, dim, device="cuda")
    x[-200:] = some
    w, b = torch.randn(dim, device="cuda"), torch.randn(dim, device="cuda")
    y, mean, rstd = finetune.layer_norm_forward(x, w, b)
    y0, mean0, rstd0 = finetune.layer_norm_forward(some, w, b)
    assert torch.equal(y[-200:], y0) and torch.equal(mean[-200:], mean0) and torch.equal(rstd[-200:], rstd0)
    assert torch.equal(y[:1000], b.expand(1000, dim)) and (mean[:1000] == 0).all()
