"""Operators for heads that are fine-tuned on the engine's descriptors and served beside it: layer norm, a shared projection
with a low-rank adapter per row (systems, datasets or users, each with its own), rows of a table by element, dataset or token,
products with a matrix of the row's own group, the norm of gradients, and AdamW over many tensors.

Tensors are torch's, on the GPU, in float32, bfloat16 or float16; work goes to torch's current stream of their device.  The
forward and backward calls are plain functions; layer_norm and adapted_linear are the same for torch's automatic
differentiation.  Wrong arguments raise ValueError (TypeError for element types) before anything is launched."""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct

import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOMENT_BLOCK = 256          # moments in 8 bits: numbers to a scale
MAX_RANK = 128
MAX_ADAPTERS = 4096
MAX_GROUPS = 4096
MAX_ENTRIES = 1 << 24
_NORM_PARTS = 1024          # SMX_GRAD_NORM_PARTS


class _Adapted(C.Structure):
    """smx_adapted_linear"""
    _fields_ = [("type", C.c_int), ("d_in", C.c_int), ("d_out", C.c_int), ("rank", C.c_int), ("num_adapters", C.c_int), ("rows", C.c_long),
                ("x", C.c_void_p), ("x_stride", C.c_long), ("weight", C.c_void_p), ("weight_stride", C.c_long), ("A", C.c_void_p),
                ("B", C.c_void_p), ("scale", C.c_void_p), ("index", C.c_void_p)]


class _AdamwTensor(C.Structure):
    """smx_adamw_tensor"""
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("master", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("scale_avg", C.c_void_p), ("scale_avg_sq", C.c_void_p), ("numel", C.c_long)]


class _Grouped(C.Structure):
    """smx_grouped_linear"""
    _fields_ = [("type", C.c_int), ("d_in", C.c_int), ("d_out", C.c_int), ("num_groups", C.c_int), ("rows", C.c_long), ("x", C.c_void_p), ("x_stride", C.c_long),
                ("weight", C.c_void_p), ("weight_stride", C.c_long), ("weight_each", C.c_long), ("bias", C.c_void_p), ("index", C.c_void_p), ("order", C.c_void_p),
                ("offsets", C.c_void_p)]


class _GradTensor(C.Structure):
    """smx_grad_tensor"""
    _fields_ = [("type", C.c_int), ("grad", C.c_void_p), ("out", C.c_void_p), ("numel", C.c_long)]


# the same as packed bytes, which are made in a fraction of the time
_ADAPTED = struct.Struct("@5iqPqPqPPPP")
_ADAMW_TENSOR = struct.Struct("@7Pq")
_ADAMW_FIRST = struct.Struct("@2P")          # param and grad
_GROUPED = struct.Struct("@4iqPqPqqPPPP")
_GRAD_TENSOR = struct.Struct("@iPPq")
assert _ADAPTED.size == C.sizeof(_Adapted) and _ADAMW_TENSOR.size == C.sizeof(_AdamwTensor)
assert _GROUPED.size == C.sizeof(_Grouped) and _GRAD_TENSOR.size == C.sizeof(_GradTensor)


_functions = None


def _lib_functions():
    global _functions
    if _functions is None:
        L = _lib.lib()
        p, i, n, d = C.c_void_p, C.c_int, C.c_long, C.c_double
        for name, args in (
                ("smx_layer_norm_forward", [i, i, n, n, p, n, p, p, d, p, n, p, p, p]),
                ("smx_layer_norm_backward_workspace", [n, n, p]),
                ("smx_layer_norm_backward", [i, i, n, n, p, n, p, n, p, p, p, p, n, p, p, p, n, p]),
                ("smx_adapted_linear_workspace", [p, i, p]),
                ("smx_adapted_linear_forward", [p, p, n, p, n, p]),
                ("smx_adapted_linear_backward", [p, p, n, p, n, p, p, p, n, p]),
                ("smx_adamw_step", [i, i, i, p, i, d, d, d, d, d, n, p]),
                ("smx_adamw_step_scaled", [i, i, i, p, i, d, d, d, d, d, n, p, p]),
                ("smx_moment_values", [n, p, p, p, p, p, p, p]),
                ("smx_group_rows_workspace", [n, i, p]),
                ("smx_group_rows", [n, i, p, p, p, p, n, p]),
                ("smx_embedding_forward", [i, n, i, i, p, n, p, d, p, n, p]),
                ("smx_embedding_backward_workspace", [i, n, i, i, p]),
                ("smx_embedding_backward", [i, n, i, i, p, n, p, p, p, d, p, p, n, p]),
                ("smx_grouped_linear_workspace", [p, i, p]),
                ("smx_grouped_linear_forward", [p, p, n, p, n, p]),
                ("smx_grouped_linear_backward", [p, p, n, p, n, p, p, p, n, p]),
                ("smx_grad_norm_workspace", [p, i, p]),
                ("smx_grad_norm", [p, i, d, p, p, p, n, p]),
                ("smx_clip_grads", [p, i, d, p, p, n, p])):
            getattr(L, name).argtypes = args
        _functions = L
    return _functions


def _type(t, what):
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{what}: float32, bfloat16 or float16, not {t.dtype}") from None


def _need(holds, what):
    if not holds:
        raise ValueError(what)


def _rows(t, dim, what):
    """t[..., dim] as rows, and the stride from one to the next (a copy where the rows have none)."""
    if t.shape[-1] != dim:
        raise ValueError(f"{what}: rows of {dim} numbers expected, not {t.shape[-1]}")
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    rows = t.shape[0]
    if rows > 1:
        stride = t.stride(0)
        if stride < dim or (dim > 1 and t.stride(1) != 1):
            t, stride = t.contiguous(), dim
    else:
        stride = dim
        if dim > 1 and t.stride(1) != 1:
            t = t.contiguous()
    return t, rows, stride


def _on(t, *others):
    """The ordinal of the tensors' device, which has to be one GPU."""
    device = t.get_device()
    if device < 0:
        raise ValueError("tensors on the GPU expected: there is no CPU path")
    for o in others:
        if o is not None and o.get_device() != device:
            raise ValueError(f"tensors on one device expected: {t.device} and {o.device}")
    return device


def _call(device, entry, *args):
    """Calls an entry point with the device's current stream as its last argument, and the device as the current one."""
    if torch.cuda.current_device() == device:
        code = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            code = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    if code:
        _lib.check(code)


# ---- layer norm

def _affine(x, dim, weight, bias):
    kind = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    if kind != x.dtype and kind != torch.float32:
        raise TypeError(f"weight and bias: {x.dtype} or float32, not {kind}")
    for t in (weight, bias):
        if t is not None:
            _need(t.shape == (dim,) and t.is_contiguous(), f"weight and bias: {dim} contiguous numbers expected")
            _need(t.dtype == kind, "weight and bias: one type expected")
    return kind


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5):
    """y = (x - mean) rstd weight + bias over the last dimension of x; returns y, mean and rstd (float32, a number a row)."""
    kind = _type(x, "x")
    _need(x.dim() >= 1 and x.shape[-1] >= 1, "x: rows of at least one number expected")
    dim = x.shape[-1]
    weights = _affine(x, dim, weight, bias)
    device = _on(x, weight, bias)
    rows_of, rows, stride = _rows(x, dim, "x")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean, rstd = x.new_empty((2,) + x.shape[:-1], dtype=torch.float32).unbind(0)
    _call(device, _lib_functions().smx_layer_norm_forward, kind, _TYPES[weights], rows, dim, rows_of.data_ptr(), stride,
          0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(), eps, y.data_ptr(), dim, mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


@functools.lru_cache(maxsize=1024)
def _norm_workspace(rows, dim):
    size = C.c_long()
    _lib.check(_lib_functions().smx_layer_norm_backward_workspace(rows, dim, C.byref(size)))
    return size.value


def layer_norm_backward(dy, x, mean, rstd, weight=None, need=(True, True, True), bias_type=None):
    """Gradients of x, weight and bias (None where `need` says so); the latter two in weight's type, or without a weight in
    bias_type (None: the type of x)."""
    kind = _type(x, "x")
    _need(x.dim() >= 1 and x.shape[-1] >= 1, "x: rows of at least one number expected")
    dim = x.shape[-1]
    _need(dy.shape == x.shape and dy.dtype == x.dtype, "dy: shape and type of x expected")
    _need(mean.dtype == rstd.dtype == torch.float32 and mean.shape == rstd.shape == x.shape[:-1] and mean.is_contiguous() and rstd.is_contiguous(),
          "mean and rstd: float32, a number a row expected")
    weights = _affine(x, dim, weight, None)
    if bias_type is not None:
        if bias_type not in (x.dtype, torch.float32) or (weight is not None and bias_type != weights):
            raise TypeError(f"bias_type: {x.dtype} or float32, and weight's type, not {bias_type}")
        weights = bias_type
    device = _on(x, dy, mean, rstd, weight)
    x_rows, rows, x_stride = _rows(x, dim, "x")
    dy_rows, _, dy_stride = _rows(dy, dim, "dy")
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    dw = db = work = None
    if need[1] or need[2]:
        dw, db = x.new_empty((2, dim), dtype=weights).unbind(0)
        dw, db = dw if need[1] else None, db if need[2] else None
        work = x.new_empty((_norm_workspace(rows, dim),), dtype=torch.uint8)
    _call(device, _lib_functions().smx_layer_norm_backward, kind, _TYPES[weights], rows, dim, dy_rows.data_ptr(), dy_stride, x_rows.data_ptr(), x_stride,
          mean.data_ptr(), rstd.data_ptr(), 0 if weight is None else weight.data_ptr(), 0 if dx is None else dx.data_ptr(), dim,
          0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(), 0 if work is None else work.data_ptr(), 0 if work is None else work.numel())
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_type = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, ctx.needs_input_grad[:3], ctx.bias_type)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension, differentiable once."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ---- a shared projection with a low-rank adapter per row

def _describe(x, weight, A, B, scale, index):
    kind = _type(x, "x")
    _need(x.dim() >= 1, "x: rows of d_in numbers expected")
    _need(weight.dim() == 2, "weight: [d_out, d_in] expected")
    d_out, d_in = weight.shape
    _need(d_in >= 1 and d_out >= 1, "weight: at least one row and column expected")
    _need(A.dim() == 3 and B.dim() == 3, "A: [adapters, rank, d_in] and B: [adapters, d_out, rank] expected")
    n, rank = A.shape[0], A.shape[1]
    _need(A.shape[2] == d_in and B.shape == (n, d_out, rank), "A: [adapters, rank, d_in] and B: [adapters, d_out, rank] expected")
    if not (weight.dtype == A.dtype == B.dtype == x.dtype):
        raise TypeError("x, weight, A and B: one type expected")
    _need(1 <= rank <= MAX_RANK and n <= MAX_ADAPTERS, f"rank: 1 to {MAX_RANK}, adapters: up to {MAX_ADAPTERS}")
    rows_of, rows, stride = _rows(x, d_in, "x")
    weight, _, weight_stride = _rows(weight, d_in, "weight")
    A, B = A.contiguous(), B.contiguous()
    if index.dtype != torch.int32:
        raise TypeError(f"index: int32 expected, not {index.dtype}")
    _need(index.shape == x.shape[:-1] and index.is_contiguous(), "index: a contiguous number a row expected")
    if scale is not None:
        if scale.dtype != torch.float32:
            raise TypeError(f"scale: float32 expected, not {scale.dtype}")
        _need(scale.shape == (n,) and scale.is_contiguous(), "scale: a contiguous number an adapter expected")
    p = _ADAPTED.pack(kind, d_in, d_out, rank, n, rows, rows_of.data_ptr(), stride, weight.data_ptr(), weight_stride, A.data_ptr(), B.data_ptr(),
                      0 if scale is None else scale.data_ptr(), index.data_ptr())
    # (the copies live until the call is made)
    return p, (kind, d_in, d_out, rank, n, rows, stride, weight_stride), (rows_of, weight, A, B)


@functools.lru_cache(maxsize=1024)
def _adapted_workspace(sizes, backward):
    """Bytes of a call's workspace, which depends on sizes alone."""
    kind, d_in, d_out, rank, n, rows, stride, weight_stride = sizes
    size, some = C.c_long(), 256
    _lib.check(_lib_functions().smx_adapted_linear_workspace(
        _ADAPTED.pack(kind, d_in, d_out, rank, n, rows, some, stride, some, weight_stride, some, some, 0, some), backward, C.byref(size)))
    return size.value


def adapted_linear_forward(x, weight, A, B, scale, index):
    """y = weight x + scale[a] B[a] (A[a] x) for every row of x, a = index of the row (int32; -1: no adapter).

    x[..., d_in], weight[d_out, d_in], A[adapters, rank, d_in] and B[adapters, d_out, rank] are of one type, scale[adapters] is
    float32 (None: ones).  Rows may come in any order.  A row whose index is out of range is NaN."""
    device = _on(x, weight, A, B, scale, index)
    p, sizes, keep = _describe(x, weight, A, B, scale, index)
    y = x.new_empty(x.shape[:-1] + (sizes[2],))
    work = x.new_empty((_adapted_workspace(sizes, 0),), dtype=torch.uint8)
    _call(device, _lib_functions().smx_adapted_linear_forward, p, y.data_ptr(), sizes[2], work.data_ptr(), work.numel())
    return y


def adapted_linear_backward(dy, x, weight, A, B, scale, index, need=(True, True, True)):
    """Gradients of x, A and B (None where `need` says so); weight and scale are fixed."""
    device = _on(x, dy, weight, A, B, scale, index)
    p, sizes, keep = _describe(x, weight, A, B, scale, index)
    d_in, d_out = sizes[1:3]
    _need(dy.shape == x.shape[:-1] + (d_out,), "dy: a row of d_out numbers for every row of x expected")
    if dy.dtype != x.dtype:
        raise TypeError("dy: the type of x expected")
    dy_rows, _, dy_stride = _rows(dy, d_out, "dy")
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    dA = torch.empty_like(A, memory_format=torch.contiguous_format) if need[1] else None
    dB = torch.empty_like(B, memory_format=torch.contiguous_format) if need[2] else None
    work = x.new_empty((_adapted_workspace(sizes, 1),), dtype=torch.uint8)
    _call(device, _lib_functions().smx_adapted_linear_backward, p, dy_rows.data_ptr(), dy_stride, 0 if dx is None else dx.data_ptr(), d_in,
          0 if dA is None else dA.data_ptr(), 0 if dB is None else dB.data_ptr(), work.data_ptr(), work.numel())
    return dx, dA, dB


class _AdaptedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, A, B, scale, index):
        ctx.save_for_backward(x, weight, A, B, scale, index)
        return adapted_linear_forward(x, weight, A, B, scale, index)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, A, B, scale, index = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        dx, dA, dB = adapted_linear_backward(dy, x, weight, A, B, scale, index, (wanted[0], wanted[2], wanted[3]))
        return dx, None, dA, dB, None, None


def adapted_linear(x, weight, A, B, scale, index):
    """adapted_linear_forward, differentiable once with respect to x, A and B; weight and scale have to be fixed (where gradients are
    not recorded, as in serving, they may be parameters of a module)."""
    _need(not torch.is_grad_enabled() or not (weight.requires_grad or (scale is not None and scale.requires_grad)),
          "weight and scale are fixed: they cannot require gradients")
    return _AdaptedLinear.apply(x, weight, A, B, scale, index)


# ---- rows by group

class RowGroups:
    """Rows sorted by group, for calls that share one index: what group_rows returns, to be given in the index's place, and refused once the
    index, order or offsets have been written to.  (A captured graph cannot refuse: one that uses RowGroups from outside of it needs the index
    as it was; one that is to follow the index has group_rows in it.)

    order: the rows (int32), those of group 0 first, then 1 and so on, then rows without a group (-1), then those whose index is out of range.
    offsets: where in it each group begins, where the rows without one do, and where those out of range do [num_groups + 2]."""

    def __init__(self, index, num_groups, order, offsets):
        if order.dtype != torch.int32 or offsets.dtype != torch.int32 or order.numel() != index.numel() or offsets.numel() != num_groups + 2 \
                or not (order.is_contiguous() and offsets.is_contiguous() and order.get_device() == offsets.get_device() == index.get_device()):
            raise ValueError("order and offsets as group_rows returns them expected")
        if index.is_inference() or order.is_inference() or offsets.is_inference():
            raise ValueError("tensors that count their versions expected, not of inference mode")
        self.index, self.num_groups, self.order, self.offsets = index, num_groups, order, offsets
        self._versions = index._version, order._version, offsets._version

    def of(self, num_groups):
        _need(num_groups == self.num_groups, f"rows by {num_groups} groups expected, not by {self.num_groups}")
        _need((self.index._version, self.order._version, self.offsets._version) == self._versions, "the index, order or offsets have been written to since the rows were sorted")
        return self


@functools.lru_cache(maxsize=1024)
def _group_rows_workspace(rows, num_groups):
    size = C.c_long()
    _lib.check(_lib_functions().smx_group_rows_workspace(rows, num_groups, C.byref(size)))
    return size.value


def _index(index, shape=None):
    """The tensor of an index (int32, one number a row) or of RowGroups."""
    groups = None
    if isinstance(index, RowGroups):
        index, groups = index.index, index
    if index.dtype != torch.int32:
        raise TypeError(f"index: int32 expected, not {index.dtype}")
    _need((shape is None or index.shape == shape) and index.is_contiguous(), "index: a contiguous number a row expected")
    return index, groups


def group_rows(index, num_groups):
    """The rows of an index (int32; -1: no group) sorted by group, in their own order inside each.

    An index of torch's inference mode, which counts no writes, is copied: calls by its RowGroups go by what it held."""
    if torch.is_inference_mode_enabled():
        with torch.inference_mode(False):          # (so that order and offsets count theirs)
            return group_rows(index, num_groups)
    index, _ = _index(index)
    _need(0 <= num_groups <= MAX_ENTRIES, f"num_groups: 0 to {MAX_ENTRIES}")
    device, rows = _on(index), index.numel()
    if index.is_inference():
        index = index.clone()
    order, offsets = index.new_empty((rows,)), index.new_empty((num_groups + 2,))
    work = index.new_empty((_group_rows_workspace(rows, num_groups),), dtype=torch.uint8)
    _call(device, _lib_functions().smx_group_rows, rows, num_groups, index.data_ptr(), order.data_ptr(), offsets.data_ptr(), work.data_ptr(), work.numel())
    return RowGroups(index, num_groups, order, offsets)


# ---- rows of a table

def embedding_forward(table, index, scale=1.0):
    """scale table[index] for every row of index (int32; -1: a row of zeros).  A row whose index is out of range is NaN.

    scale: 0 or a normal number of single precision, which it is rounded to."""
    kind = _type(table, "table")
    shape = table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError("table: [entries, dim] expected")
    entries, dim = shape
    if entries > MAX_ENTRIES or not math.isfinite(scale):
        raise ValueError(f"entries: up to {MAX_ENTRIES}; scale: a finite number")
    index, groups = _index(index)
    if groups is not None:
        groups.of(entries)
    device = _on(table, index)
    table, _, stride = _rows(table, dim, "table")
    y = table.new_empty(index.shape + (dim,))
    _call(device, _lib_functions().smx_embedding_forward, kind, index.numel(), entries, dim, table.data_ptr(), stride, index.data_ptr(), scale, y.data_ptr(), dim)
    return y


@functools.lru_cache(maxsize=1024)
def _embedding_workspace(kind, rows, entries, dim):
    size = C.c_long()
    _lib.check(_lib_functions().smx_embedding_backward_workspace(kind, rows, entries, dim, C.byref(size)))
    return size.value


def embedding_backward(dy, index, entries, scale=1.0):
    """The gradient of a table [entries, dim]: scale times the sum of the rows of dy of every entry, in the type of dy."""
    kind = _type(dy, "dy")
    _need(dy.dim() >= 1 and dy.shape[-1] >= 1, "dy: rows of at least one number expected")
    dim = dy.shape[-1]
    _need(0 <= entries <= MAX_ENTRIES and math.isfinite(scale), f"entries: 0 to {MAX_ENTRIES}; scale: a finite number")
    index, groups = _index(index, dy.shape[:-1])
    device = _on(dy, index)
    order = offsets = 0
    if groups is not None:
        groups.of(entries)
        order, offsets = groups.order.data_ptr(), groups.offsets.data_ptr()
    dy_rows, rows, stride = _rows(dy, dim, "dy")
    dtable = dy.new_empty((entries, dim))
    work = dy.new_empty((_embedding_workspace(kind, rows, entries, dim),), dtype=torch.uint8)
    _call(device, _lib_functions().smx_embedding_backward, kind, rows, entries, dim, dy_rows.data_ptr(), stride, index.data_ptr(), order, offsets, scale,
          dtable.data_ptr(), work.data_ptr(), work.numel())
    return dtable


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale):
        y = embedding_forward(table, index, scale)
        ctx.groups = index if isinstance(index, RowGroups) else None
        ctx.save_for_backward(index.index if ctx.groups else index)
        ctx.entries, ctx.scale = table.shape[0], scale
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return embedding_backward(dy, ctx.groups or ctx.saved_tensors[0], ctx.entries, ctx.scale), None, None


def embedding(table, index, scale=1.0):
    """embedding_forward, differentiable once with respect to table."""
    return _Embedding.apply(table, index, scale)


# ---- a product with a matrix of the row's own group

def _grouped(x, weight, bias, index):
    kind, shape, rows_shape = _type(x, "x"), weight.shape, x.shape
    if len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        raise ValueError("weight: [groups, d_out, d_in] expected")
    n, d_out, d_in = shape
    if not rows_shape or rows_shape[-1] != d_in:
        raise ValueError("x: rows of d_in numbers expected")
    if n > MAX_GROUPS:
        raise ValueError(f"groups: up to {MAX_GROUPS}")
    if weight.dtype is not x.dtype or (bias is not None and bias.dtype is not x.dtype):
        raise TypeError("x, weight and bias: one type expected")
    if bias is not None and (bias.shape != (n, d_out) or not bias.is_contiguous()):
        raise ValueError("bias: contiguous, [groups, d_out] expected")
    index, groups = _index(index, rows_shape[:-1])
    device = _on(x, weight, bias, index)
    order = offsets = 0
    if groups is not None:
        groups.of(n)
        order, offsets = groups.order.data_ptr(), groups.offsets.data_ptr()
    rows_of, rows, stride = _rows(x, d_in, "x")
    each, weight_stride, along = weight.stride()
    if (d_in > 1 and along != 1) or (d_out > 1 and weight_stride < d_in):
        weight = weight.contiguous()
        each, weight_stride, along = weight.stride()
    if d_out == 1:
        weight_stride = d_in
    p = _GROUPED.pack(kind, d_in, d_out, n, rows, rows_of.data_ptr(), stride, weight.data_ptr(), weight_stride, each, 0 if bias is None else bias.data_ptr(),
                      index.data_ptr(), order, offsets)
    # (the copies live until the call is made)
    return device, p, (kind, d_in, d_out, n, rows, stride, weight_stride, each), (rows_of, weight)


@functools.lru_cache(maxsize=1024)
def _grouped_workspace(sizes, backward):
    """Bytes of a call's workspace, which depends on sizes alone."""
    kind, d_in, d_out, n, rows, stride, weight_stride, each = sizes
    size, some = C.c_long(), 256
    _lib.check(_lib_functions().smx_grouped_linear_workspace(
        _GROUPED.pack(kind, d_in, d_out, n, rows, some, stride, some, weight_stride, each, 0, some, 0, 0), backward, C.byref(size)))
    return size.value


def grouped_linear_forward(x, weight, bias, index):
    """y = weight[g] x + bias[g] for every row of x, g = index of the row (int32; -1: no group, zeros), or RowGroups of it.

    x[..., d_in], weight[groups, d_out, d_in] and bias[groups, d_out] (or None) are of one type.  Rows may come in any order, groups may
    have none.  A row whose index is out of range is NaN."""
    device, p, sizes, keep = _grouped(x, weight, bias, index)
    y = x.new_empty(x.shape[:-1] + (sizes[2],))
    size = _grouped_workspace(sizes, 0)
    work = x.new_empty((size,), dtype=torch.uint8) if size else None
    _call(device, _lib_functions().smx_grouped_linear_forward, p, y.data_ptr(), sizes[2], work.data_ptr() if size else 0, size)
    return y


def grouped_linear_backward(dy, x, weight, index, need=(True, True, True)):
    """Gradients of x, weight and bias (None where `need` says so); zeros for groups without a row."""
    device, p, sizes, keep = _grouped(x, weight, None, index)
    d_in, d_out, n = sizes[1:4]
    _need(dy.shape == x.shape[:-1] + (d_out,), "dy: a row of d_out numbers for every row of x expected")
    if dy.dtype != x.dtype:
        raise TypeError("dy: the type of x expected")
    _on(x, dy)
    dy_rows, _, dy_stride = _rows(dy, d_out, "dy")
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need[1] else None
    db = x.new_empty((n, d_out)) if need[2] else None
    work = x.new_empty((_grouped_workspace(sizes, 1),), dtype=torch.uint8)
    _call(device, _lib_functions().smx_grouped_linear_backward, p, dy_rows.data_ptr(), dy_stride, 0 if dx is None else dx.data_ptr(), d_in,
          0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(), work.data_ptr(), work.numel())
    return dx, dw, db


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, index):
        ctx.groups = index if isinstance(index, RowGroups) else None
        ctx.save_for_backward(x, weight, index.index if ctx.groups else index)
        ctx.biased = bias is not None
        return grouped_linear_forward(x, weight, bias, index)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, index = ctx.saved_tensors
        need = ctx.needs_input_grad
        return *grouped_linear_backward(dy, x, weight, ctx.groups or index, (need[0], need[1], ctx.biased and need[2])), None


def grouped_linear(x, weight, bias, index):
    """grouped_linear_forward, differentiable once with respect to x, weight and bias."""
    return _GroupedLinear.apply(x, weight, bias, index)


# ---- the norm of gradients

@functools.lru_cache(maxsize=64)
def _grad_tensors(count):
    return struct.Struct("@" + "iPPq" * count)


def _describe_grads(grads, outs=None):
    """The descriptions of tensors that are there (not None), their device, how many, and what has to live until the call is made."""
    numbers, keep, device, types = [], [], None, _TYPES
    for g, o in zip(grads, outs or grads):
        if g is None:
            continue
        dtype = g.dtype
        kind = types.get(dtype)
        if kind is None:
            _type(g, "gradients")
        at, n = g.get_device(), g.numel()
        if at != device:
            if device is not None:
                raise ValueError("gradients on one device expected")
            device = _on(g)
        to = 0
        if outs is not None and o is not g:
            if o is None:
                raise ValueError("out: a tensor for every gradient expected")
            if o.dtype is not dtype:
                raise TypeError("out: the types of the gradients expected")
            if o.get_device() != at or o.shape != g.shape or not o.is_contiguous():
                raise ValueError("out: contiguous, of the gradients' shapes and on their device, expected")
            to = o.data_ptr()
        if not g.is_contiguous():
            g = g.contiguous()
            keep.append(g)
        from_ = g.data_ptr()
        numbers += (kind, from_, to or from_, n)
    count = len(numbers) // 4
    return _grad_tensors(count).pack(*numbers), device, count, keep


def _span(t):
    """Where the tensor's numbers begin and end in memory."""
    at = t.data_ptr()
    return at, at + (1 + sum((n - 1) * step for n, step in zip(t.shape, t.stride()))) * t.element_size() if t.numel() else at


def _norm_call(described, max_norm, clip, factor=False):
    """The norm, a float32 number, and with `factor` what keeps the factor, where its memory begins."""
    packed, device, count, keep = described
    place, size = torch.device("cuda", device), (8 * (_NORM_PARTS + count) + 255) // 256 * 256
    norm = torch.empty((), dtype=torch.float32, device=place)
    work = torch.empty((size + 256 if factor else size,), dtype=torch.uint8, device=place)
    at = work.data_ptr()
    if clip:
        _call(device, _lib_functions().smx_clip_grads, packed, count, max_norm, norm.data_ptr(), at, size)
    else:
        _call(device, _lib_functions().smx_grad_norm, packed, count, max_norm, norm.data_ptr(), at if factor else 0, at + 256 if factor else at, size)
    return (norm, work) if factor else norm


def grad_norm(grads):
    """The norm of all numbers of the tensors together, sqrt(sum g^2), as a float32 tensor of no dimensions.

    Tensors may be of different types and shapes; None stands for a gradient that is not there."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    described = _describe_grads(grads)
    if not described[2]:
        return torch.zeros((), device="cuda")
    return _norm_call(described, math.inf, False)


def clip_grads(grads, max_norm, out=None):
    """Brings the gradients to a norm of at most max_norm together, g min(1, max_norm / norm), in place or into out (tensors like
    grads, each with memory of its own), and returns the norm that they had.  Where the norm is not finite they stay as they are."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    _need(max_norm >= 0, "max_norm: a number from 0 on")
    there = list(grads)
    if out is not None:
        there = [out] if isinstance(out, torch.Tensor) else list(out)
        _need(len(there) == len(grads), "out: a tensor for every gradient expected")
    back, out = [], list(there)          # gradients that are clipped in place by way of a contiguous copy, and the copies
    for k, g in enumerate(there):
        if g is not None and g is grads[k] and not g.is_contiguous():
            _need(all(n <= 1 or step for n, step in zip(g.shape, g.stride())), "gradients that are clipped in place: numbers with memory of their own expected")
            grads[k] = out[k] = g.detach().contiguous()
            back.append((g.detach(), out[k]))
    if back:          # (of what is written as it is, the call itself finds out)
        spans = {(g.data_ptr(), g.shape, g.stride()): _span(g) for g, _ in back}
        _need(len(spans) == len(back), "tensors that are written: every one once expected, each with memory of its own")
        for g, o in zip(grads, out):
            if g is not None and o is not None and o is not g:
                from_, to = _span(o)
                _need(all(to <= a or b <= from_ for a, b in spans.values()), "tensors that are written: every one once expected, each with memory of its own")
    described = _describe_grads(grads, out)
    if not described[2]:
        return torch.zeros((), device="cuda")
    norm = _norm_call(described, max_norm, True)
    for g, copy in back:
        g.copy_(copy)
    # (as torch's own operations in place do)
    torch.autograd.graph.increment_version([o for o, g in zip(there, grads) if g is not None])
    return norm


# ---- AdamW

def moment_values(code_avg, scale_avg, code_avg_sq, scale_avg_sq):
    """The numbers that moments in 8 bits stand for: codes (int8, uint8) of one tensor and a float32 scale for every 256 of them."""
    n = code_avg.numel()
    if code_avg.dtype != torch.int8 or code_avg_sq.dtype != torch.uint8 or not scale_avg.dtype == scale_avg_sq.dtype == torch.float32:
        raise TypeError("codes in int8 and uint8, scales in float32 expected")
    blocks = -(-n // MOMENT_BLOCK)
    _need(code_avg_sq.numel() == n and scale_avg.numel() == scale_avg_sq.numel() == blocks, f"{n} codes and {blocks} scales expected")
    _need(all(t.is_contiguous() for t in (code_avg, scale_avg, code_avg_sq, scale_avg_sq)), "contiguous tensors expected")
    device = _on(code_avg, scale_avg, code_avg_sq, scale_avg_sq)
    m = torch.empty_like(code_avg, dtype=torch.float32)
    v = torch.empty_like(m)
    _call(device, _lib_functions().smx_moment_values, n, code_avg.data_ptr(), scale_avg.data_ptr(), code_avg_sq.data_ptr(), scale_avg_sq.data_ptr(),
          m.data_ptr(), v.data_ptr())
    return m, v


class AdamW:
    """AdamW over many tensors at once, a launch for up to 56 of them.

    state_bits 32: moments in single precision; 8: in codes of 8 bits, 256 to a scale.  masters: parameters in single
    precision for params in 16 bits, a list like params; True makes them from params.  states: moments to go on with, a tuple a
    tensor, (exp_avg, exp_avg_sq) or (code_avg, scale_avg, code_avg_sq, scale_avg_sq); they are used in place, as params and
    masters are, and so is what self.states holds otherwise (zeros at first).  Both attributes can be assigned anew as a whole, under
    the same checks; what a tensor of theirs or a parameter holds is looked at in every step.  step: steps taken before, a number or
    one for every parameter, as self.steps has them: a parameter takes only those steps that it has a gradient in."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, masters=None, states=None, step=0):
        self.params = tuple(params)
        _need(state_bits in (32, 8), "state_bits: 32 or 8")
        _need(0 <= betas[0] < 1 and 0 <= betas[1] < 1, "betas: 0 up to, not including, 1")
        _need(lr >= 0 and eps >= 0 and weight_decay >= 0, "lr, eps and weight_decay: numbers from 0 on")
        taken = list(step) if isinstance(step, (list, tuple)) else [step] * len(self.params)
        _need(len(taken) == len(self.params) and all(t >= 0 for t in (taken or [step])), "step: steps taken before, none or more, a number or one for every parameter")
        self.lr, self.betas, self.eps, self.weight_decay, self._bits = lr, tuple(betas), eps, weight_decay, state_bits
        self.step_count = max(taken, default=0)
        self._missed = [self.step_count - t for t in taken]          # steps without a gradient
        for p in self.params:
            _type(p, "parameters")
            _need(p.is_contiguous(), "parameters: contiguous tensors expected")
            _need(p.is_cuda and p.device == self.params[0].device, "parameters on one GPU expected: there is no CPU path")
            if p.dtype != self.params[0].dtype:
                raise TypeError("parameters of one type expected: an optimizer for each")
        self._apart(self.params, "parameters")
        # what every parameter has to be in every step
        self._shapes = [p.shape for p in self.params]
        self._dtype, self._device = (self.params[0].dtype, self.params[0].get_device()) if self.params else (None, None)
        self._masters = None
        self.states = [self._zeros(p) for p in self.params] if states is None else states
        self.masters = [p.detach().float() for p in self.params] if masters is True else masters

    @property
    def state_bits(self):
        return self._bits

    @property
    def steps(self):
        """The steps that every parameter has taken."""
        return tuple(self.step_count - m for m in self._missed)

    @property
    def states(self):
        """Moments, a tuple of tensors for every parameter."""
        return self._states

    @states.setter
    def states(self, states):
        states = tuple(tuple(s) for s in states)
        _need(len(states) == len(self.params), "states: a tuple for every parameter expected")
        self._apart([t for s in states for t in s], "states")
        self._hold_all(states, self._masters)

    @property
    def masters(self):
        """Parameters in single precision, a tuple like params, or None."""
        return self._masters

    @masters.setter
    def masters(self, masters):
        if masters is not None:
            masters = tuple(masters)
            _need(len(masters) == len(self.params), "masters: one for every parameter expected")
            self._apart(masters, "masters")
        self._hold_all(self._states, masters)

    @staticmethod
    def _apart(tensors, what):
        """(A step goes over all tensors at once: memory that two of them name would be written by both.)"""
        starts = [t.data_ptr() for t in tensors if t.numel()]
        _need(len(set(starts)) == len(starts), f"{what}: every tensor once expected, each with memory of its own")

    # What is held of the tensors: the descriptions that a step hands on, all but the parameters' and gradients' addresses, the addresses
    # in them, and aliases of the tensors.  The aliases keep the memory, so that none of the addresses is ever that of memory that others
    # use; a tensor that was given other memory has another address, which is compared in every step.
    def _hold_all(self, states, masters):
        held = [self._hold(i, states, masters) for i in range(len(self.params))]
        self._table = bytearray(b"".join(_ADAMW_TENSOR.pack(0, 0, *h[0]) for h in held))
        self._held, self._states, self._masters = held, states, masters

    def _hold(self, i, states, masters):
        """A parameter's part of smx_adamw_tensor from its master on, and the aliases."""
        n, bits, s = self._shapes[i].numel(), self._bits, states[i]
        kinds = (torch.float32, torch.float32) if bits == 32 else (torch.int8, torch.float32, torch.uint8, torch.float32)
        counts = (n, n) if bits == 32 else (n, -(-n // MOMENT_BLOCK)) * 2
        _need(len(s) == len(kinds) and all(t.dtype == k and t.numel() == c and t.is_contiguous() and t.get_device() == self._device
                                           for t, k, c in zip(s, kinds, counts)),
              "states: (exp_avg, exp_avg_sq) in float32, or (code_avg int8, scale_avg float32, code_avg_sq uint8, scale_avg_sq float32), "
              "contiguous and on the parameters' device, expected")
        held = s
        if masters is not None:
            m = masters[i]
            _need(self._dtype != torch.float32, "masters are for parameters in 16 bits")
            _need(m.dtype == torch.float32 and m.shape == self._shapes[i] and m.is_contiguous() and m.get_device() == self._device,
                  "masters: contiguous, float32, of the parameters' shapes and on their device expected")
            held = (*s, m)
        at = (0, 1) if bits == 32 else (0, 2, 1, 3)          # of a state: moments, then their scales
        return (0 if masters is None else m.data_ptr(), *(s[k].data_ptr() for k in at), *((0, 0) if bits == 32 else ()), n), [t.detach() for t in held]

    def _zeros(self, p):
        n, blocks = p.numel(), -(-p.numel() // MOMENT_BLOCK)
        make = lambda k, dtype: torch.zeros(k, dtype=dtype, device=p.device)          # noqa: E731
        if self._bits == 32:
            return make(n, torch.float32), make(n, torch.float32)
        return make(n, torch.int8), make(blocks, torch.float32), make(n, torch.uint8), make(blocks, torch.float32)

    def step(self, grads=None, max_norm=None):
        """One step with the given gradients, one for every parameter (None: the parameters' own).  A parameter without a gradient
        (None) is left as it is, and does not count the step.  Gradients are of the parameters' type or all in float32.

        max_norm: the step goes by gradients clipped to this norm together, as clip_grads does, but without writing them; returned is
        their norm before (a norm that is not finite clips nothing)."""
        norm = None
        if grads is None:
            grads = [p.grad for p in self.params]
        _need(max_norm is None or max_norm >= 0, "max_norm: a number from 0 on")
        _need(len(grads) == len(self.params), "a gradient (or None) for every parameter expected")
        taken = [i for i, g in enumerate(grads) if g is not None]
        if taken:
            params, device, own = self.params, self._device, self._dtype
            kind = grads[taken[0]].dtype
            if kind != own and kind != torch.float32:
                raise TypeError(f"gradients: {own} or float32, not {kind}")
            keep, wide, size, described = [], self._bits == 32, _ADAMW_TENSOR.size, []
            shapes, held, states, masters, table, first = self._shapes, self._held, self._states, self._masters, self._table, _ADAMW_FIRST.pack_into
            for i in taken:
                p, g, shape, s = params[i], grads[i], shapes[i], states[i]
                if p.dtype is not own or g.dtype is not kind:
                    raise TypeError(f"parameters in {own}, as they were at first, and gradients of one type expected")
                if p.shape != shape or p.get_device() != device or not p.is_contiguous():
                    raise ValueError("parameters contiguous, and of the shapes and on the device they had at first, expected")
                if g.shape != shape or g.get_device() != device:
                    raise ValueError("gradients of the parameters' shapes and on their device expected")
                if not g.is_contiguous():
                    g = g.contiguous()
                    keep.append(g)
                master, m, v, scale_m, scale_v, _ = held[i][0]
                if (s[0].data_ptr() != m or (s[1].data_ptr() != v if wide else s[2].data_ptr() != v or s[1].data_ptr() != scale_m or s[3].data_ptr() != scale_v)
                        or (masters is not None and masters[i].data_ptr() != master)):
                    held[i] = self._hold(i, states, masters)
                    _ADAMW_TENSOR.pack_into(table, i * size, 0, 0, *held[i][0])
                first(table, i * size, p.data_ptr(), g.data_ptr())
                if max_norm is not None:
                    described.append(_GRAD_TENSOR.pack(_TYPES[kind], g.data_ptr(), 0, g.numel()))
            missed = self._missed
            if any(missed):
                _need(all(missed[i] <= self.step_count for i in taken), "step_count: less than the steps that a parameter has missed")
                calls = {}          # descriptions by the number of the step that it is for their tensors
                for i in taken:
                    calls[missed[i]] = calls.get(missed[i], b"") + table[i * size:(i + 1) * size]
            else:          # (no parameter has missed a step so far; some may have no gradient in this one)
                calls = {0: bytes(table) if len(taken) == len(params) else b"".join(table[i * size:(i + 1) * size] for i in taken)}
            if max_norm is not None:
                norm, factor = _norm_call((b"".join(described), device, len(described), keep), max_norm, False, factor=True)
            for late, some in calls.items():
                of = (_TYPES[own], _TYPES[kind], self._bits, some, len(some) // size, self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay,
                      self.step_count + 1 - late)
                if norm is None:
                    _call(device, _lib_functions().smx_adamw_step, *of)
                else:
                    _call(device, _lib_functions().smx_adamw_step_scaled, *of, factor.data_ptr())
            # (as torch's own operations in place do: a backward pass that saved the old values says so)
            torch.autograd.graph.increment_version(params if len(taken) == len(params) else [params[i] for i in taken])
        if len(taken) < len(grads):
            for i, g in enumerate(grads):
                if g is None:
                    self._missed[i] += 1
        self.step_count += 1
        if max_norm is not None:
            return norm if norm is not None else torch.zeros((), device=torch.device("cuda", self._device) if self.params else "cuda")
