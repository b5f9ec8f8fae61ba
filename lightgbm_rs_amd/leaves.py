"""The operators around a forest's leaves, as methods of `HipBackend` over torch tensors:
rows grouped by leaf, the leaves' linear maps and their gradients, dropout and class scores
(include/lgbm_hip.h has the definitions).

Tensors are on the backend's device; matrices have a row stride (a matrix whose columns
are strided is copied first).  A call queues its work on torch's current stream of that
device and returns, so calls follow each other like torch's own operations and can be
captured into a graph.  Gradients are entries of their own: nothing is recorded for
torch's autograd, so a floating-point tensor that requires gradients is refused while they are
recorded (call under torch.no_grad(), as the methods of a torch.autograd.Function are, or
on detached tensors).

Import torch before the first `HipBackend`: torch brings a HIP runtime of its own, which
the library then shares.  (The other way round torch finds no device.)
"""
import ctypes as C
from typing import Any, NamedTuple

import numpy as np

from .backend import PREDICT_KINDS, HipBackend, load_library

_DTYPES = {}  # torch's element types -> LGBM_HIP_DTYPE_*
_PRODUCT, _DX, _DW = 0, 1, 2


class _Maps(C.Structure):
    """`lgbm_leaf_maps`."""

    _fields_ = [("order", C.c_void_p), ("begin", C.c_void_p), ("count", C.c_void_p),
                ("num_rows", C.c_int64), ("num_trees", C.c_int32), ("num_leaves", C.c_int32),
                ("inputs", C.c_int32), ("outputs", C.c_int32), ("dtype", C.c_int32),
                ("_pad", C.c_int32)]


class _Scores(C.Structure):
    """`lgbm_score_args`."""

    _fields_ = [("x", C.c_void_p), ("ldx", C.c_int64), ("num_rows", C.c_int64),
                ("num_classes", C.c_int32), ("dtype", C.c_int32), ("kind", C.c_int32),
                ("num_masks", C.c_int32), ("bias", C.c_void_p), ("mask", C.c_void_p),
                ("mask_rows", C.c_void_p), ("ids", C.c_void_p), ("offsets", C.c_void_p),
                ("num_ids", C.c_int64), ("repetition", C.c_double), ("frequency", C.c_double),
                ("presence", C.c_double), ("penalties", C.c_void_p), ("out", C.c_void_p),
                ("ldo", C.c_int64)]


class LeafGroups(NamedTuple):
    """The rows of every leaf: order int32 [trees, rows], begin and count int32 [trees,
    leaves] (each leaf's range of its tree's order)."""

    order: Any
    begin: Any
    count: Any

    @classmethod
    def from_layout(cls, layout, device="cuda"):
        """The groups of a grown tree's layout (`HipBackend.grow_tree_on_device_with_cfg`)."""
        import torch
        up = lambda v: torch.from_numpy(np.ascontiguousarray(v).astype(np.int32))[None].to(device)
        return cls(up(layout["indices"]), up(layout["leaf_begin"]), up(layout["leaf_count"]))


_torch = None  # the module, once a method has been called


def _module():
    """torch, the library's entries with their argument types declared, and the element types:
    set up by the first call, so that the package itself does not need torch."""
    global _torch
    if _torch is None:
        import torch
        p, i32, i64, u64, size = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64, C.c_size_t
        lib = load_library()
        for name, types in (
                ("leaf_groups_workspace", (i64, i32, i32, p)),
                ("leaf_groups", (p, p, i64, i64, i32, i32, p, p, p, p, size, p)),
                ("leaf_product_workspace", (p, i32, p)),
                ("leaf_product", (p, p, p, i64, p, p, p, i64, p, size, p)),
                ("leaf_product_dx", (p, p, p, i64, p, p, i64, p, size, p)),
                ("leaf_product_dw", (p, p, p, i64, p, i64, p, p, p, size, p)),
                ("dropout", (p, p, i64, i64, i64, i32, C.c_double, u64, u64, i32, p, i64, p)),
                ("adjust_scores_workspace", (p, p)),
                ("adjust_scores", (p, p, p, size, p))):
            getattr(lib, "lgbm_hip_" + name).argtypes = types
        for name, code in (("float32", 0), ("float64", 1), ("bfloat16", 2), ("float16", 3)):
            _DTYPES[getattr(torch, name)] = code
        _torch = torch
    return _torch


def _stream(self, torch):
    """The `stream` argument: torch's current stream of the backend's device."""
    return C.byref(C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream))


def _dtype(t, what, double=False):
    code = _DTYPES.get(t.dtype)
    if code is None or (code == 1 and not double):
        raise ValueError(f"{what} is {t.dtype}: a floating-point type of the device is needed"
                         + ("" if double else ", of at most 32 bits"))
    return code


def _here(self, **tensors):
    """Every tensor on the backend's device, and none that autograd would have to record."""
    for name, t in tensors.items():
        if t is not None and t.requires_grad and _torch.is_grad_enabled():
            raise ValueError(f"{name} requires gradients, which this call does not record")
    for name, t in tensors.items():
        if t is not None and (not t.is_cuda or t.get_device() != self.device):
            raise ValueError(f"{name} is on {t.device}: cuda:{self.device} is needed")


def _shape(t, shape, what):
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}: {tuple(shape)} is needed")


def _typed(t, what, dtype):
    """t without gaps, of a type."""
    if t.dtype is not dtype:
        raise ValueError(f"{what} is {t.dtype}: {dtype} is needed")
    return t.contiguous()


def _ld(t):
    """The row stride of a matrix; one row or none has no stride that matters."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _rows(t):
    """t with unit column stride and rows that do not overlap."""
    if not t.is_contiguous():
        rows, cols = t.shape
        if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
            t = t.contiguous()
    return t


def _out(out, like, shape):
    """The output: the caller's, checked, or a new tensor."""
    if out is None:
        return like.new_empty(shape)
    _shape(out, shape, "out")
    if out.dtype is not like.dtype:
        raise ValueError(f"out is {out.dtype}: {like.dtype} is needed")
    if _rows(out) is not out:
        raise ValueError("out has strided columns or rows that overlap")
    return out


def _written(*tensors):
    """Tells autograd of the caller's tensors that were written, as torch's own in-place
    operations do: a graph that saved one refuses its backward pass."""
    for t in tensors:
        if t is not None and not t.is_inference():
            _torch.autograd.graph.increment_version(t)


def _workspace(self, torch, entry, *args):
    """(pointer, bytes, the tensor that holds them) of an entry's working memory."""
    size = C.c_size_t(0)
    self._check_plain(entry(*args, C.byref(size)))
    if not size.value:
        return None, 0, None
    t = torch.empty(size.value, dtype=torch.uint8, device=f"cuda:{self.device}")
    return t.data_ptr(), size.value, t


def _leaf_groups(self, leaf, num_leaves):
    """The rows of every leaf (`lgbm_hip_leaf_groups`) from leaf int32 [rows, trees] or
    [rows], as `predict(kind="leaf")` gives it; an index outside [0, num_leaves) means that
    the row is in no leaf of that tree.  Returns LeafGroups."""
    torch = _module()
    if leaf.dim() == 1:
        leaf = leaf[:, None]
    if leaf.dim() != 2 or leaf.shape[1] == 0:
        raise ValueError("leaf has to be [rows, trees]")
    if leaf.dtype is not torch.int32:
        raise ValueError(f"leaf is {leaf.dtype}: int32 is needed")
    _here(self, leaf=leaf)
    leaf = _rows(leaf)
    rows, trees = leaf.shape
    ws, nbytes, hold = _workspace(self, torch, self.lib.lgbm_hip_leaf_groups_workspace, rows,
                                  trees, num_leaves)
    order = leaf.new_empty((trees, rows))
    begin, count = leaf.new_empty((2, trees, num_leaves))
    self._check(self.lib.lgbm_hip_leaf_groups(
        self.ctx, leaf.data_ptr(), _ld(leaf), rows, trees, num_leaves, order.data_ptr(),
        begin.data_ptr(), count.data_ptr(), ws, nbytes, _stream(self, torch)))
    return LeafGroups(order, begin, count)


def _maps(self, torch, rows, inputs, outputs, dtype, groups, leaves=None):
    """(lgbm_leaf_maps, the tensors it points to)"""
    order, begin, count = groups
    trees, num = begin.shape
    _shape(order, (trees, rows), "order")
    _shape(count, (trees, num), "count")
    if leaves is not None and leaves != trees * num:
        raise ValueError(f"weights of {leaves} leaves for {trees} x {num}")
    hold = [_typed(t, n, torch.int32) for t, n in ((order, "order"), (begin, "begin"), (count, "count"))]
    _here(self, order=order, begin=begin, count=count)
    return _Maps(*[t.data_ptr() for t in hold], rows, trees, num, inputs, outputs, dtype, 0), hold


def _leaf_product(self, x, weight, groups, bias=None, out=None):
    """y[n] = sum over trees of weight[t, leaf] x[n] + bias[t, leaf]
    (`lgbm_hip_leaf_product`): x [rows, inputs], weight [trees * leaves, outputs, inputs],
    bias [trees * leaves, outputs] or None, all float32, bfloat16 or float16.  Returns y
    [rows, outputs]."""
    torch = _module()
    if x.dim() != 2 or weight.dim() != 3:
        raise ValueError("x has to be [rows, inputs], weight [leaves, outputs, inputs]")
    dtype, (rows, inputs) = _dtype(x, "x"), x.shape
    leaves, outputs = weight.shape[:2]
    _shape(weight, (leaves, outputs, inputs), "weight")
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise ValueError("x, weight and bias differ in type")
    if bias is not None:
        _shape(bias, (leaves, outputs), "bias")
        bias = bias.contiguous()
    _here(self, x=x, weight=weight, bias=bias, out=out)
    m, keep = _maps(self, torch, rows, inputs, outputs, dtype, groups, leaves)
    given = out
    x, weight, out = _rows(x), weight.contiguous(), _out(out, x, (rows, outputs))
    ws, nbytes, hold = _workspace(self, torch, self.lib.lgbm_hip_leaf_product_workspace,
                                  C.byref(m), _PRODUCT)
    self._check(self.lib.lgbm_hip_leaf_product(
        self.ctx, C.byref(m), x.data_ptr(), _ld(x), weight.data_ptr(),
        None if bias is None else bias.data_ptr(), out.data_ptr(), _ld(out), ws, nbytes,
        _stream(self, torch)))
    _written(given)
    return out


def _leaf_product_dx(self, dy, weight, groups, out=None):
    """The gradient of `leaf_product`'s x (`lgbm_hip_leaf_product_dx`): dy [rows, outputs]
    gives dx [rows, inputs], the sum over the trees."""
    torch = _module()
    if dy.dim() != 2 or weight.dim() != 3:
        raise ValueError("dy has to be [rows, outputs], weight [leaves, outputs, inputs]")
    dtype, (rows, outputs) = _dtype(dy, "dy"), dy.shape
    leaves, inputs = weight.shape[0], weight.shape[2]
    _shape(weight, (leaves, outputs, inputs), "weight")
    if weight.dtype != dy.dtype:
        raise ValueError("dy and weight differ in type")
    _here(self, dy=dy, weight=weight, out=out)
    m, keep = _maps(self, torch, rows, inputs, outputs, dtype, groups, leaves)
    given = out
    dy, weight, out = _rows(dy), weight.contiguous(), _out(out, dy, (rows, inputs))
    ws, nbytes, hold = _workspace(self, torch, self.lib.lgbm_hip_leaf_product_workspace,
                                  C.byref(m), _DX)
    self._check(self.lib.lgbm_hip_leaf_product_dx(
        self.ctx, C.byref(m), dy.data_ptr(), _ld(dy), weight.data_ptr(), out.data_ptr(), _ld(out),
        ws, nbytes, _stream(self, torch)))
    _written(given)
    return out


def _leaf_product_dw(self, dy, x, groups, bias=True, out=None, bias_out=None):
    """The gradients of `leaf_product`'s weight and bias (`lgbm_hip_leaf_product_dw`):
    dw [trees * leaves, outputs, inputs] and db [trees * leaves, outputs] (None without
    `bias`), float32 whatever the type of dy [rows, outputs] and x [rows, inputs]."""
    torch = _module()
    if dy.dim() != 2 or x.dim() != 2:
        raise ValueError("dy has to be [rows, outputs], x [rows, inputs]")
    dtype, (rows, outputs) = _dtype(dy, "dy"), dy.shape
    inputs = x.shape[1]
    _shape(x, (rows, inputs), "x")
    if x.dtype != dy.dtype:
        raise ValueError("dy and x differ in type")
    if bias_out is not None and not bias:
        raise ValueError("bias_out without bias")
    _here(self, dy=dy, x=x, out=out, bias_out=bias_out)
    m, keep = _maps(self, torch, rows, inputs, outputs, dtype, groups)
    leaves = m.num_trees * m.num_leaves
    for name, t, shape in (("out", out, (leaves, outputs, inputs)),
                           ("bias_out", bias_out, (leaves, outputs))):
        if t is not None:
            _shape(t, shape, name)
            if t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError(f"{name} has to be contiguous float32")
    dw = dy.new_empty((leaves, outputs, inputs), dtype=torch.float32) if out is None else out
    db = bias_out
    if bias and db is None:
        db = dy.new_empty((leaves, outputs), dtype=torch.float32)
    dy, x = _rows(dy), _rows(x)
    ws, nbytes, hold = _workspace(self, torch, self.lib.lgbm_hip_leaf_product_workspace,
                                  C.byref(m), _DW)
    self._check(self.lib.lgbm_hip_leaf_product_dw(
        self.ctx, C.byref(m), dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), dw.data_ptr(),
        None if db is None else db.data_ptr(), ws, nbytes, _stream(self, torch)))
    _written(out, bias_out)
    return dw, db


def _dropout(self, x, p, seed, offset=0, by="element", out=None):
    """x with elements, or with by="row" whole rows, dropped with probability p and the
    others divided by the share kept (`lgbm_hip_dropout`): the mask follows from seed and
    offset (64 bits each), so the gradient is the same call on the outputs' gradient.
    x [rows, cols] or [rows] float32, bfloat16 or float16; out may be x."""
    torch = _module()
    if by not in ("element", "row"):
        raise ValueError("by is neither 'element' nor 'row'")
    if x.dim() not in (1, 2):
        raise ValueError("x has to be [rows, cols] or [rows]")
    dtype = _dtype(x, "x")
    _here(self, x=x, out=out)
    if x.dim() == 1:
        if out is not None:
            _shape(out, x.shape, "out")
            _dropout(self, x[:, None], p, seed, offset, by, out[:, None])
            return out
        return _dropout(self, x[:, None], p, seed, offset, by)[:, 0]
    inplace = out is x
    src = _rows(x)
    if inplace and src is not x:
        raise ValueError("out has strided columns or rows that overlap")
    dst = _out(out, x, tuple(x.shape))
    self._check(self.lib.lgbm_hip_dropout(
        self.ctx, src.data_ptr(), _ld(src), x.shape[0], x.shape[1], dtype, p, seed & (2 ** 64 - 1),
        offset & (2 ** 64 - 1), by == "row", dst.data_ptr(), _ld(dst), _stream(self, torch)))
    _written(out)
    return dst


def _adjust_scores(self, scores, kind="raw", bias=None, mask=None, mask_rows=None, ids=None,
                   offsets=None, repetition=1.0, frequency=0.0, presence=0.0, penalties=None,
                   out=None):
    """Class scores to answers (`lgbm_hip_adjust_scores`): penalties for the classes that
    stand in a row's history, a bias for every class, the mask of the classes that a row
    may have, and with kind="transformed" the softmax.

    scores [rows, classes] float32, float64, bfloat16 or float16; bias [classes] of the same
    type; mask int32 [masks, ceil(classes / 32)] whose bits are the classes allowed, mask_rows
    int32 [rows] the mask of every row (-1: none; left out: one mask, or one for each row);
    ids int32 and offsets int64 [rows + 1]: row n's history is ids[offsets[n]:offsets[n +
    1]]; penalties float32 [rows, 3] instead of the three numbers.  out may be scores."""
    torch = _module()
    if scores.dim() != 2:
        raise ValueError("scores has to be [rows, classes]")
    if kind not in ("raw", "transformed"):
        raise ValueError("kind is neither 'raw' nor 'transformed'")
    dtype, (rows, classes) = _dtype(scores, "scores", True), scores.shape
    if bias is not None:
        _shape(bias, (classes,), "bias")
        if bias.dtype != scores.dtype:
            raise ValueError("scores and bias differ in type")
        bias = bias.contiguous()
    if mask is not None:
        if mask.dim() == 1:
            mask = mask[None]
        _shape(mask, (mask.shape[0], (classes + 31) // 32), "mask")
        mask = _typed(mask, "mask", torch.int32)
        if mask_rows is None and mask.shape[0] == 0 < rows:
            raise ValueError("a mask table without masks")
    elif mask_rows is not None:
        raise ValueError("mask_rows without mask")
    if mask_rows is not None:
        _shape(mask_rows, (rows,), "mask_rows")
        mask_rows = _typed(mask_rows, "mask_rows", torch.int32)
    if (ids is None) != (offsets is None):
        raise ValueError("a history needs ids and offsets")
    if ids is not None:
        _shape(ids, (ids.numel(),), "ids")
        _shape(offsets, (rows + 1,), "offsets")
        ids, offsets = _typed(ids, "ids", torch.int32), _typed(offsets, "offsets", torch.int64)
    if penalties is not None:
        _shape(penalties, (rows, 3), "penalties")
        penalties = _typed(penalties, "penalties", torch.float32)
    _here(self, scores=scores, bias=bias, mask=mask, mask_rows=mask_rows, ids=ids,
          offsets=offsets, penalties=penalties, out=out)
    src = _rows(scores)
    if out is scores and src is not scores:
        raise ValueError("out has strided columns or rows that overlap")
    given = out
    out = _out(out, scores, (rows, classes))
    at = lambda t: None if t is None else t.data_ptr()
    a = _Scores(at(src), _ld(src), rows, classes, dtype, PREDICT_KINDS[kind],
                0 if mask is None else mask.shape[0], at(bias), at(mask), at(mask_rows), at(ids),
                at(offsets), 0 if ids is None else ids.numel(), repetition, frequency, presence,
                at(penalties), at(out), _ld(out))
    ws, nbytes, hold = _workspace(self, torch, self.lib.lgbm_hip_adjust_scores_workspace, C.byref(a))
    self._check(self.lib.lgbm_hip_adjust_scores(self.ctx, C.byref(a), ws, nbytes,
                                                _stream(self, torch)))
    _written(given)
    return out


HipBackend.leaf_groups = _leaf_groups
HipBackend.leaf_product = _leaf_product
HipBackend.leaf_product_dx = _leaf_product_dx
HipBackend.leaf_product_dw = _leaf_product_dw
HipBackend.dropout = _dropout
HipBackend.adjust_scores = _adjust_scores

__all__ = ["LeafGroups"]
