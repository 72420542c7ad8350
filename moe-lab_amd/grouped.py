"""Products of 16-bit matrices grouped by expert, with ragged sizes, and their gradients (moe_grouped_mm, _dx, _dw).

Slots are sorted by expert: expert e holds the slots offsets[e] <= p < offsets[e + 1] (router.group and router.route_group
return offsets, and the slots' order). x, w and bias are bf16 or fp16, all of one type; sums are fp32 in a fixed order and
rounded once.

    y = mm(x, w, offsets, bias=b)            x [M, K], w [E, N, K] -> y [M, N], differentiable
    y = mm(x, w, offsets, rows=tokens)       x [T, K], the row of each slot by index: no gathered copy of x

The reference multiplies quantised experts only; its unquantised form is a loop over the experts (reference
moelab/variants/cuda/torch_loop.py:11-17).
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib

# A matrix read through an index list is addressed with 32 bits from its start; past this many bytes its rows are gathered
# first.
MAX_INDEXED_BYTES = 0xB0000000


def _index(t, name, device, n=None):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name}: int32 [{'slots' if n is None else n}] expected, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other operands on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _offsets(t, device, E):
    if t is None and E != 1:
        raise ValueError(f"offsets None: one expert expected, not {E}")
    return _index(t, "offsets", device, E + 1)


def _weights(w, name="w"):
    if w.dim() != 3:
        raise ValueError(f"{name} has shape {tuple(w.shape)}: [experts, N, K] expected")
    E, N, K = w.shape
    _lib.multiple_of(N, 8, "N")
    _lib.multiple_of(K, 8, "K")
    _lib.require_device(w, name)
    if w.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} is {w.dtype}: bf16 or fp16 expected")
    if not w.is_contiguous() or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    return w, E, N, K


def _far(x):
    return x.shape[0] * x.stride(0) * 2 > MAX_INDEXED_BYTES


def _taken(x, rows):
    """x[rows], an index outside x as a row of zeros."""
    ok = (rows >= 0) & (rows < x.shape[0])
    return torch.where(ok[:, None], x[torch.where(ok, rows, 0).long()], 0)


def _gathered(x, rows):
    """x and its index list, or the rows themselves where 32 bits cannot address x."""
    return (_taken(x, rows), None) if rows is not None and _far(x) else (x, rows)


def _slots(x, rows, what):
    if rows is not None and x.shape[0] == 0 and rows.shape[0] > 0:
        raise ValueError(f"{what} has no rows to index")
    return x.shape[0] if rows is None else rows.shape[0]


def _mm(x, w, offsets, bias, rows, out, out_dtype):
    w, E, N, K = _weights(w)
    x = _lib.half_matrix(x, "x", K, w.device, w.dtype)
    offsets = _offsets(offsets, w.device, E)
    rows = _index(rows, "rows", w.device)
    bias = _lib.plain(bias, "bias", (E, N), w.device, w.dtype)
    M = _slots(x, rows, "x")
    y = _lib.result(out, (M, N), w.dtype, out_dtype, w.device)
    x, rows = _gathered(x, rows)
    _lib.call("moe_grouped_mm", w.device, x.data_ptr(), w.data_ptr(), _lib.ptr(bias), _lib.ptr(offsets), _lib.ptr(rows), M,
              x.shape[0], x.stride(0), E, N, K, _lib.DTYPE[w.dtype], y.data_ptr(), _lib.DTYPE[y.dtype], int(out is None))
    return y


class _Mm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, bias, rows, out_dtype):
        ctx.save_for_backward(x, w, offsets, rows)
        return _mm(x, w, offsets, bias, rows, None, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets, rows = ctx.saved_tensors
        dy = dy.to(w.dtype)
        dx = mm_dx(dy, w, offsets) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[3]:
            dw, db = mm_dw(dy, x, offsets, w.shape[0], x_rows=rows, bias=True)
        return dx, dw if ctx.needs_input_grad[1] else None, None, db if ctx.needs_input_grad[3] else None, None, None


def mm(x, w, offsets, bias=None, rows=None, out=None, out_dtype=None):
    """y[p] = x[p] . w[e]^T (+ bias[e]) for the slots p of expert e; with rows (int32 [M]) x[rows[p]] in place of x[p] (an
    index outside x reads as zeros).
    x [M or any, K], w [E, N, K], offsets int32 [E + 1] (or None with E = 1: all slots), bias [E, N]; N and K multiples of 8.
    Slots behind the last expert: zeros in a new result, left as they are in `out`. out_dtype: the operands' type or fp32.
    Differentiable in x, w and bias (x not with rows: its gradient would add several slots' rows); gradients of a result in
    fp32 are rounded to the operands' type first."""
    if not _lib.wants_grad(x, w, bias):
        return _mm(x, w, offsets, bias, rows, out, out_dtype)
    if out is not None:
        raise ValueError("out= takes no gradient")
    if rows is not None and x.requires_grad:
        raise ValueError("x read through rows takes no gradient: index it first, or use dense.experts_mlp")
    return _Mm.apply(x, w, offsets, bias, rows, out_dtype)


def mm_dx(dy, w, offsets, rows=None, out=None, out_dtype=None):
    """dx[p] = dy[p] . w[e]: the gradient of mm in x. dy [M, N] (with rows: dy[rows[p]]), w [E, N, K] -> [M, K]."""
    w, E, N, K = _weights(w)
    dy = _lib.half_matrix(dy, "dy", N, w.device, w.dtype)
    offsets = _offsets(offsets, w.device, E)
    rows = _index(rows, "rows", w.device)
    M = _slots(dy, rows, "dy")
    dx = _lib.result(out, (M, K), w.dtype, out_dtype, w.device)
    dy, rows = _gathered(dy, rows)
    _lib.call("moe_grouped_mm_dx", w.device, dy.data_ptr(), w.data_ptr(), _lib.ptr(offsets), _lib.ptr(rows), M, dy.shape[0],
              dy.stride(0), E, N, K, _lib.DTYPE[w.dtype], dx.data_ptr(), _lib.DTYPE[dx.dtype], int(out is None))
    return dx


def mm_dw(dy, x, offsets, E, dy_rows=None, x_rows=None, bias=False, out=None, out_dtype=None):
    """dw[e] = sum of dy[p]^T x[p] over the slots of expert e (zeros where it has none): the gradient of mm in w, [E, N, K].
    dy_rows, x_rows: int32 [M] row of each slot. bias: also return db [E, N], the sums of dy, as (dw, db)."""
    for t, name, n in ((dy, "dy", "N"), (x, "x", "K")):
        _lib.require_device(t, name)
        if t.dim() != 2:
            raise ValueError(f"{name} has shape {tuple(t.shape)}: [rows, {n}] expected")
        _lib.multiple_of(t.shape[1], 8, n)
    dy = _lib.half_matrix(dy, "dy")
    x = _lib.half_matrix(x, "x", None, dy.device, dy.dtype)
    N, K = dy.shape[1], x.shape[1]
    offsets = _offsets(offsets, dy.device, E)
    dy_rows, x_rows = _index(dy_rows, "dy_rows", dy.device), _index(x_rows, "x_rows", dy.device)
    M = _slots(dy, dy_rows, "dy")
    if _slots(x, x_rows, "x") != M:
        raise ValueError(f"{M} slots of dy and {_slots(x, x_rows, 'x')} of x")
    dw = _lib.result(out, (E, N, K), dy.dtype, out_dtype, dy.device)
    db = torch.empty((E, N), dtype=dy.dtype, device=dy.device) if bias else None
    if (dy_rows is not None or x_rows is not None) and (_far(dy) or _far(x)):
        # with a list for either operand the kernel addresses both with 32 bits from their start
        dy, dy_rows = (dy if dy_rows is None else _taken(dy, dy_rows)), None
        x, x_rows = (x if x_rows is None else _taken(x, x_rows)), None
    _lib.call("moe_grouped_mm_dw", dy.device, dy.data_ptr(), x.data_ptr(), _lib.ptr(offsets), _lib.ptr(dy_rows),
              _lib.ptr(x_rows), M, dy.shape[0], dy.stride(0), x.shape[0], x.stride(0), E, N, K, _lib.DTYPE[dy.dtype],
              dw.data_ptr(), _lib.DTYPE[dw.dtype], _lib.ptr(db))
    return (dw, db) if bias else dw
