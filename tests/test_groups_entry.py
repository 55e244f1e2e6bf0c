"""What the C entry points of tables, products by group and norms of gradients refuse, before any device is looked for."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def L():
    from symmetrix_amd import finetune
    return finetune._lib_functions()


def _why(L):
    return L.smx_last_error().decode()


def test_workspaces_and_sizes(L):
    n = C.c_long()
    assert L.smx_group_rows_workspace(100_000, 5000, C.byref(n)) == 0 and n.value >= 2 * 4 * 100_000
    assert L.smx_embedding_backward_workspace(0, 1000, 50, 64, C.byref(n)) == 0 and n.value > 0
    for bad in ((-1, 5), (2 ** 28 + 1, 5), (10, -1), (10, 2 ** 24 + 1)):
        assert L.smx_group_rows_workspace(*bad, C.byref(n)) == -1 and _why(L)
    for bad in ((3, 10, 5, 8), (0, -1, 5, 8), (0, 10, -1, 8), (0, 10, 5, 0), (0, 10, 5, 2 ** 20 + 1)):
        assert L.smx_embedding_backward_workspace(*bad, C.byref(n)) == -1 and _why(L)
    assert L.smx_group_rows_workspace(10, 5, None) == -1


def test_pointers_and_strides(L):
    some = 4096
    assert L.smx_group_rows(10, 5, None, some, some, some, 1 << 20, None) == -1 and "null" in _why(L)
    assert L.smx_group_rows(10, 5, some, some, some, some + 4, 1 << 20, None) == -1 and "256" in _why(L)
    assert L.smx_group_rows(5000, 5, some, some, some, some, 8, None) == -1 and "smx_group_rows_workspace" in _why(L)
    assert L.smx_embedding_forward(0, 10, 5, 8, None, 8, some, 1.0, some, 8, None) == -1 and "null" in _why(L)
    assert L.smx_embedding_forward(0, 10, 5, 8, some, 7, some, 1.0, some, 8, None) == -1 and "stride" in _why(L)
    assert L.smx_embedding_forward(0, 10, 5, 8, some, 8, some, 1.0, some, 7, None) == -1 and "stride" in _why(L)
    assert L.smx_embedding_forward(0, 0, 5, 8, None, 8, None, 1.0, None, 8, None) == 0          # (no rows: nothing to do)
    assert L.smx_embedding_backward(0, 10, 5, 8, some, 8, some, some, None, 1.0, some, some, 1 << 20, None) == -1 and "both or neither" in _why(L)
    assert L.smx_embedding_backward(0, 10, 5, 8, some, 8, some, None, None, 1.0, None, some, 1 << 20, None) == -1 and "null" in _why(L)


def test_grouped(L):
    from symmetrix_amd import finetune
    good = dict(kind=0, d_in=8, d_out=4, n=3, rows=10, x=4096, x_stride=8, weight=4096, weight_stride=8, each=32, bias=0, index=4096, order=0, offsets=0)
    pack = lambda **k: finetune._GROUPED.pack(*dict(good, **k).values())          # noqa: E731
    n = C.c_long()
    assert L.smx_grouped_linear_workspace(pack(), 0, C.byref(n)) == 0 and L.smx_grouped_linear_workspace(pack(), 1, C.byref(n)) == 0
    for bad in (dict(kind=3), dict(d_in=0), dict(d_out=2 ** 20 + 1), dict(n=-1), dict(n=4097), dict(rows=-1), dict(rows=2 ** 28 + 1), dict(x=0), dict(x_stride=7),
                dict(weight=0), dict(weight_stride=7), dict(each=-1), dict(index=0), dict(order=4096)):
        assert L.smx_grouped_linear_workspace(pack(**bad), 0, C.byref(n)) == -1, bad
        assert _why(L).startswith("smx_grouped_linear_workspace: ")
    assert L.smx_grouped_linear_workspace(None, 0, C.byref(n)) == -1
    assert L.smx_grouped_linear_forward(pack(rows=0), None, 4, None, 0, None) == 0
    assert L.smx_grouped_linear_forward(pack(), None, 4, 4096, 1 << 20, None) == -1 and "null" in _why(L)
    assert L.smx_grouped_linear_forward(pack(), 4096, 3, 4096, 1 << 20, None) == -1 and "stride" in _why(L)
    assert L.smx_grouped_linear_backward(pack(), None, 4, 4096, 8, None, None, 4096, 1 << 20, None) == -1
    assert L.smx_grouped_linear_backward(pack(), 4096, 4, 4096, 7, None, None, 4096, 1 << 20, None) == -1
    assert L.smx_grouped_linear_backward(pack(), 4096, 4, None, 8, None, None, None, 0, None) == 0          # (nothing asked for)


def test_norms(L):
    from symmetrix_amd import finetune
    n = C.c_long()
    pack = lambda *t: b"".join(finetune._GRAD_TENSOR.pack(*x) for x in t)          # noqa: E731
    assert L.smx_grad_norm_workspace(pack((0, 4096, 4096, 10 ** 8), (1, 4096, 4096, 5)), 2, C.byref(n)) == 0 and 0 < n.value <= 8 * 2304
    assert L.smx_grad_norm_workspace(None, 0, C.byref(n)) == 0
    for bad in ((3, 4096, 4096, 10), (0, 4096, 4096, -1), (0, 4096, 4096, 2 ** 36)):
        assert L.smx_grad_norm_workspace(pack(bad), 1, C.byref(n)) == -1 and _why(L)
    assert L.smx_grad_norm_workspace(None, 1, C.byref(n)) == -1
    good = pack((0, 4096, 4096, 10))
    assert L.smx_grad_norm(pack((0, 0, 0, 10)), 1, 1.0, 4096, 4096, 4096, 4096, None) == -1 and "null" in _why(L)
    assert L.smx_clip_grads(pack((0, 4096, 0, 10)), 1, 1.0, 4096, 4096, 4096, None) == -1 and "out" in _why(L)
    assert L.smx_clip_grads(good, 1, -1.0, 4096, 4096, 4096, None) == -1 and "max_norm" in _why(L)
    assert L.smx_clip_grads(good, 1, float("nan"), 4096, 4096, 4096, None) == -1
    assert L.smx_grad_norm(good, 1, 1.0, 4096, 4096, 4096, 4, None) == -1 and "smx_grad_norm_workspace" in _why(L)
