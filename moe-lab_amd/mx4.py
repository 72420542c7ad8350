"""MXFP4 operands made on the GPU, and products of two of them on the block-scaled matrix cores (moe_mx4_*).

    q = quantize(x)                                     x [..., K] bf16, fp16 or fp32 -> Mx4; dequantize(q) gives the values
    y = linear(x, w, bias=b, act=SILU, residual=r)      linear.linear with both operands in MXFP4; w an Mx4, or 16-bit numbers
    y = grouped_mm(x, w, offsets, rows=tokens)          grouped.mm likewise, by expert

An element is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign), 32 neighbours share a power of two (formats.py's MXFP4, whose
packed weights from_packed and to_packed take and give). A product of two such numbers is exact and sums are fp32, so what a call
adds to the exact product of its 16-bit operands is their rounding to MXFP4: for normal numbers about 12% of an element, and of
a product's result. The reference multiplies MXFP4 weights by 16-bit activations in its expert kernels only (reference
metal_mxfp4_moe.py); experts.run_experts is that form.

Gradients go straight through the roundings, in 16 bits: dx = dz w and dw = dz^T x at the values that the product used, of which
x's are kept in 4 bits. For fp16 operands those values are rounded to fp16 there (bf16 holds them): what 16-bit fp16 weights and
activations become is exact in it, but weights from a checkpoint whose exponents leave its range give infinities past 65504 in dx, and
nothing up to 2^-25, where the product itself takes them as they are.
With an activation z is kept, and dz rounded, in the operands' 16 bits: dz because the 16-bit matrix instructions take it so, z because its
32 bits would be as large as the result in fp32 for little. Errors of the gradients in the norm (1024^3, SiLU, bf16, against 64 bits):
1.66e-3 from their own rounding, 1.74e-3 with z's, 2.35e-3 with dz's, 2.40e-3 with both; fp16 2.1e-4, 2.2e-4, 2.9e-4, 3.0e-4.
"""
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib, formats, grouped as _grouped
from .linear import GELU, NONE, SILU   # noqa: F401

BLOCK = formats.GS_MXFP4   # elements that share an exponent
STEP = 256                 # columns whose exponents lie together: 8 bytes of a row


class Mx4:
    """A matrix [rows, K], or several [E, rows, K], in MXFP4. codes: uint8 [..., rows, K / 2], two codes to a byte, the low half
    first; scales: the E8M0 bytes as the products read them (include/moe_mi355x.h). Neither can be replaced."""
    __slots__ = ("codes", "scales", "shape", "device")

    def __init__(self, codes, scales):
        shape = (*codes.shape[:-1], 2 * codes.shape[-1])
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() not in (2, 3) or shape[-1] % BLOCK or not shape[-1]:
            raise ValueError(f"uint8 codes [rows, K / 2] or [E, rows, K / 2] with K a multiple of {BLOCK}, and uint8 scales expected")
        n = _scale_bytes(shape)
        if scales.device != codes.device or tuple(scales.shape) != (n,) or not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError(f"contiguous codes, and {n} bytes of scales on the same device expected")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("16-byte aligned codes and scales expected")
        _set(self, codes, scales, shape)

    def __setattr__(self, name, value):
        raise AttributeError("an Mx4 is not changed: its products rely on the sizes it was made with")

    def __reduce__(self):
        return Mx4, (self.codes, self.scales)

    def __repr__(self):
        return f"Mx4({list(self.shape)}, device='{self.device}')"


def _set(q, codes, scales, shape):
    for name, value in (("codes", codes), ("scales", scales), ("shape", shape), ("device", codes.device)):
        object.__setattr__(q, name, value)


def _of(codes, scales):
    """The Mx4 of tensors that came from one."""
    q = Mx4.__new__(Mx4)
    _set(q, codes, scales, (*codes.shape[:-1], 2 * codes.shape[-1]))
    return q


def _scale_bytes(shape):
    E = shape[0] if len(shape) == 3 else 1
    return 8 * E * shape[-2] * (-(-shape[-1] // STEP)) + 16


def _new(shape, device):
    q = Mx4.__new__(Mx4)
    _set(q, torch.empty(*shape[:-1], shape[-1] // 2, dtype=torch.uint8, device=device),
         torch.empty(_scale_bytes(shape), dtype=torch.uint8, device=device), tuple(shape))
    return q


def _quantize(x):
    """x [rows, K] (rows may be apart) or contiguous [E, rows, K], 16-byte aligned -> Mx4."""
    q = _new(x.shape, x.device)
    E = x.shape[0] if x.dim() == 3 else 1
    _lib.call("moe_mx4_quantize", x.device, x.data_ptr(), x.stride(-2) if x.shape[-2] > 1 else x.shape[-1], E, x.shape[-2], x.shape[-1],
              _lib.DTYPE[x.dtype], q.codes.data_ptr(), q.scales.data_ptr())
    return q


def quantize(x):
    """x [..., K] (bf16, fp16 or fp32; K a multiple of 32) -> Mx4, of one matrix [rows, K], or for x [E, rows, K] of E matrices.
    Per 32 neighbours the exponent is that of their largest magnitude less 2, so that it lies in [4, 8) steps of E2M1's 6;
    elements go to the nearest code, ties to the even one, past 6 to 6. Blocks below 2^-124 become zeros, blocks with an
    infinity or NaN read as NaN. No gradient (linear and grouped_mm have one)."""
    _lib.require_device(x, "x")
    if x.dtype not in _lib.DTYPE:
        raise TypeError(f"x is {x.dtype}: bf16, fp16 or fp32 expected")
    if x.dim() < 1:
        raise ValueError("x [..., K] expected")
    _lib.multiple_of(x.shape[-1], BLOCK, "K")
    if _lib.wants_grad(x):
        raise NotImplementedError("quantize has no gradient: detach x, or multiply by linear or grouped_mm")
    x = x.detach()
    if x.dim() not in (2, 3):
        x = x.reshape(-1, x.shape[-1])
    apart = x.dim() == 2 and x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.shape[1] <= x.stride(0) <= 1 << 21
    if not (apart or x.is_contiguous()) or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return _quantize(x)


def dequantize(q, dtype=torch.bfloat16):
    """The values of an Mx4, in its shape: exact in bf16 and fp32 (from 2^-126 on), rounded to fp16."""
    _lib.require_device(q.codes, "q")
    if dtype not in _lib.DTYPE:
        raise TypeError(f"dtype {dtype}: bf16, fp16 or fp32 expected")
    out = torch.empty(*q.shape, dtype=dtype, device=q.device)
    E = q.shape[0] if len(q.shape) == 3 else 1
    _lib.call("moe_mx4_dequantize", q.device, q.codes.data_ptr(), q.scales.data_ptr(), E, q.shape[-2], q.shape[-1], out.data_ptr(),
              _lib.DTYPE[dtype])
    return out


def _steps_of(shape):
    return -(-shape[-1] // STEP)


def from_packed(codes, scales):
    """The packed form of formats.py (and of MXFP4 checkpoints): codes int32 [..., N, K / 8], scales uint8 [..., N, K / 32] ->
    Mx4. A scale byte of 0, which reads as 0 there, takes its codes along."""
    if codes.dtype != torch.int32 or scales.dtype != torch.uint8 or codes.dim() not in (2, 3) or codes.device != scales.device:
        raise ValueError("codes int32 [N, K / 8] or [E, N, K / 8] and uint8 scales on the same device expected")
    if tuple(scales.shape) != (*codes.shape[:-1], codes.shape[-1] // 4) or codes.shape[-1] % 4 or codes.shape[-1] == 0:
        raise ValueError(f"codes {tuple(codes.shape)}, scales {tuple(scales.shape)}: [..., K / 8] and [..., K / 32] expected")
    shape = (*codes.shape[:-1], 8 * codes.shape[-1])
    c = codes.contiguous().view(torch.uint8)
    if bool((scales == 0).any()):
        c = torch.where((scales == 0).repeat_interleave(16, -1), torch.zeros_like(c), c)
    E, N, S = shape[0] if len(shape) == 3 else 1, shape[-2], _steps_of(shape)
    s = torch.full((E, N, 8 * S), 127, dtype=torch.uint8, device=codes.device)
    s[..., :shape[-1] // BLOCK] = scales.reshape(E, N, shape[-1] // BLOCK)
    flat = torch.zeros(_scale_bytes(shape), dtype=torch.uint8, device=codes.device)
    flat[:-16] = s.reshape(E, N, S, 4, 2).permute(0, 2, 1, 4, 3).reshape(-1)
    return Mx4(c.clone() if c.data_ptr() == codes.data_ptr() else c, flat)


def to_packed(q):
    """(codes int32 [..., K / 8], scales uint8 [..., K / 32]) of an Mx4."""
    E, N, S = q.shape[0] if len(q.shape) == 3 else 1, q.shape[-2], _steps_of(q.shape)
    s = q.scales[:-16].reshape(E, S, N, 2, 4).permute(0, 2, 1, 4, 3).reshape(E, N, 8 * S)[..., :q.shape[-1] // BLOCK]
    return q.codes.clone().view(torch.int32), s.reshape(*q.shape[:-1], q.shape[-1] // BLOCK).contiguous()


# ------------------------------------------------------------------------------------------------------ products
def _weights(w, dims, what):
    """w as an Mx4 of that many dimensions (16-bit numbers are quantised), and its type if it was 16-bit."""
    if isinstance(w, Mx4):
        _lib.require_device(w.codes, "w")
        if len(w.shape) != dims:
            raise ValueError(f"w has shape {w.shape}: {what} expected")
        _lib.multiple_of(w.shape[-2], 8, "N")
        return w, None
    _lib.require_device(w, "w")
    if w.dim() != dims:
        raise ValueError(f"w has shape {tuple(w.shape)}: {what} expected")
    if w.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"w is {w.dtype}: an Mx4, bf16 or fp16 expected")
    _lib.multiple_of(w.shape[-2], 8, "N")
    _lib.multiple_of(w.shape[-1], BLOCK, "K")
    return quantize(w.detach()), w.dtype


def _type_of(x, w_type, out_dtype, *others):
    """The call's 16-bit type: x's, or for an Mx4 that of w or the other operands, else out_dtype if that is one, else bf16."""
    types = set()
    for t in others:
        if t is not None:
            types.add(t.dtype)
    if w_type is not None:
        types.add(w_type)
    if not isinstance(x, Mx4):
        types.add(x.dtype)
    if len(types) > 1:
        raise TypeError(f"operands in {', '.join(sorted(map(str, types)))}: one 16-bit type expected")
    t = types.pop() if types else out_dtype if out_dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
    if t not in (torch.bfloat16, torch.float16):
        raise TypeError(f"operands in {t}: bf16 or fp16 expected")
    return t


def _operand(x, K, device, dims=None):
    """x as the library takes it: (16-bit rows or None, Mx4 or None, rows)."""
    if isinstance(x, Mx4):
        if len(x.shape) != 2 or x.shape[1] != K:
            raise ValueError(f"x has shape {x.shape}: [rows, {K}] expected")
        if x.device != device:
            raise ValueError(f"x is on {x.device}, the other operands on {device}")
        return None, x, x.shape[0]
    _lib.require_device(x, "x")
    if x.dim() < 1 or x.shape[-1] != K or (dims is not None and x.dim() != dims):
        raise ValueError(f"x has shape {tuple(x.shape)}: [{'rows' if dims == 2 else '...'}, {K}] expected")
    x2 = _lib.half_matrix(x if x.dim() == 2 else x.reshape(-1, K), "x", K, device)
    return x2, None, x2.shape[0]


def _pointers(x2, q):
    rows = (None, 0) if x2 is None else (x2.data_ptr(), x2.stride(0) if x2.shape[0] > 1 else x2.shape[1])
    return rows + ((None, None) if q is None else (q.codes.data_ptr(), q.scales.data_ptr()))


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name, *sizes):
    return getattr(_lib.lib(), name)(*sizes)


def _workspace(device, name, *sizes):
    n = _workspace_bytes(name, *sizes)
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


def _run_linear(x, w, bias, act, residual, out_dtype, keep_z, keep_x):
    """y, z (None unless keep_z), x's Mx4 (keep_x: made for a 16-bit x too) and w's."""
    if act not in (NONE, SILU, GELU):
        raise ValueError(f"act {act}: NONE, SILU or GELU expected")
    w4, w_type = _weights(w, 2, "[N, K]")
    N, K = w4.shape
    device = w4.device
    dtype = _type_of(x, w_type, out_dtype, bias, residual)
    lead = (x.shape[0],) if isinstance(x, Mx4) else x.shape[:-1]
    x2, q, T = _operand(x, K, device)
    bias = _lib.plain(bias, "bias", (N,), device, dtype)
    residual = _lib.plain(residual, "residual", (*lead, N), device, dtype)
    y = _lib.result(None, (T, N), dtype, out_dtype, device)
    z = torch.empty((T, N), dtype=dtype, device=device) if keep_z else None
    if keep_x and q is None:
        q = _new((T, K), device)
    ws, nws = _workspace(device, "moe_mx4_linear_workspace_bytes", T, N, K)
    _lib.call("moe_mx4_linear", device, *_pointers(x2, q), w4.codes.data_ptr(), w4.scales.data_ptr(), _lib.ptr(bias),
              _lib.ptr(residual), int(act), T, N, K, _lib.DTYPE[dtype], y.data_ptr(), _lib.DTYPE[y.dtype], _lib.ptr(z), _lib.ptr(ws), nws)
    return y if len(lead) == 1 else y.view(*lead, N), z, q, w4


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w4, bias, act, residual, out_dtype):
        need_x, need_w, _, need_b = ctx.needs_input_grad[:4]
        y, z, q, w4 = _run_linear(x, w if w4 is None else w4, bias, act, residual, out_dtype,
                                  act != NONE and (need_x or need_w or need_b), need_w)
        # the weights' 4-bit form stands for w from here on, also where w changes before the backward pass
        ctx.save_for_backward(*((q.codes, q.scales) if need_w else (None, None)),
                              *((w4.codes, w4.scales) if need_x else (None, None)), z)
        ctx.act, ctx.x_shape, ctx.dtype = int(act), x.shape, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xc, xs, wc, ws, z = ctx.saved_tensors
        need_x, need_w, _, need_b = ctx.needs_input_grad[:4]
        dy = dy.to(ctx.dtype)
        dx = dw = db = None
        if need_x or need_w or need_b:
            d, K = _lib.half_matrix(dy.reshape(-1, dy.shape[-1]), "dy"), ctx.x_shape[-1]
            T, N = d.shape
            if need_x:
                dx = torch.empty(ctx.x_shape, dtype=d.dtype, device=d.device)
            if need_w:
                dw = torch.empty((N, K), dtype=d.dtype, device=d.device)
            if need_b:
                db = torch.empty(N, dtype=d.dtype, device=d.device)
            work, n = _workspace(d.device, "moe_mx4_linear_bwd_workspace_bytes", T, N, K, ctx.act, int(need_x), int(need_w), int(need_b))
            _lib.call("moe_mx4_linear_bwd", d.device, d.data_ptr(), d.stride(0), _lib.ptr(z), ctx.act, _lib.ptr(xc), _lib.ptr(xs),
                      _lib.ptr(wc), _lib.ptr(ws), T, N, K, _lib.DTYPE[d.dtype], _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db),
                      _lib.ptr(work), n)
        return dx, dw, None, db, None, dy if ctx.needs_input_grad[5] else None, None


def _bias_grad(dy, offsets, E):
    """Sums of dy's rows by group [E, N]."""
    M, N = dy.shape
    db = torch.empty((E, N), dtype=dy.dtype, device=dy.device)
    ws, nws = _workspace(dy.device, "moe_mx4_bias_grad_workspace_bytes", M, E, N)
    _lib.call("moe_mx4_bias_grad", dy.device, dy.data_ptr(), dy.stride(0), _lib.ptr(offsets), M, E, N, _lib.DTYPE[dy.dtype],
              db.data_ptr(), _lib.ptr(ws), nws)
    return db


def _grouped_dx(dy, w4, offsets):
    M, (E, N, K) = dy.shape[0], w4.shape
    dx = torch.empty((M, K), dtype=dy.dtype, device=dy.device)
    _lib.call("moe_mx4_grouped_mm_dx", dy.device, dy.data_ptr(), dy.stride(0), w4.codes.data_ptr(), w4.scales.data_ptr(),
              _lib.ptr(offsets), M, E, N, K, _lib.DTYPE[dy.dtype], dx.data_ptr(), _lib.DTYPE[dy.dtype], 1)
    return dx


def linear(x, w, bias=None, act=NONE, residual=None, out_dtype=None):
    """act(x w^T + bias) + residual, x and w in MXFP4. x [..., K] bf16 or fp16 (quantised in the call) or an Mx4 [rows, K];
    w an Mx4 [N, K], or 16-bit weights that are quantised in the call; bias [N] and residual [..., N] of x's type (with an Mx4
    x: of one 16-bit type). K a multiple of 32, N of 8. out_dtype: that type or fp32.
    Differentiable in 16-bit x and w, bias and residual, straight through the quantisation: dx = dz w, dw = dz^T x with the MXFP4
    values (in fp16 rounded to it), 16-bit products and z = x w^T + bias kept in 16 bits. Gradients of a result in fp32 are rounded
    to the operands' type first."""
    x_grad, w_grad = (None if isinstance(t, Mx4) else t for t in (x, w))
    if not _lib.wants_grad(x_grad, w_grad, bias, residual):
        return _run_linear(x, w, bias, act, residual, out_dtype, False, False)[0]
    if x_grad is None:
        raise ValueError("an Mx4 x takes no part in a backward pass: give its 16-bit form")
    return _Linear.apply(x, w_grad, w if w_grad is None else None, bias, act, residual, out_dtype)


def _run_grouped(x, w, offsets, bias, rows, out, out_dtype, keep):
    """y, x's Mx4 (keep: made for a 16-bit x too), w's, the offsets as the library reads them, and the list of x's rows (None also
    where x was indexed first)."""
    w4, w_type = _weights(w, 3, "[experts, N, K]")
    E, N, K = w4.shape
    device = w4.device
    dtype = _type_of(x, w_type, out_dtype if out is None else out.dtype, bias)
    offsets = _grouped._offsets(offsets, device, E)
    rows = _grouped._index(rows, "rows", device)
    bias = _lib.plain(bias, "bias", (E, N), device, dtype)
    x2, q, n = _operand(x, K, device, 2)
    M = n if rows is None else rows.shape[0]
    if rows is not None and n == 0 and M > 0:
        raise ValueError("x has no rows to index")
    if rows is not None and n * (K // 2) > _grouped.MAX_INDEXED_BYTES:
        if x2 is None:
            raise ValueError(f"an Mx4 of {n * (K // 2)} bytes cannot be read through rows: at most {_grouped.MAX_INDEXED_BYTES}")
        x2, rows, n = _grouped._taken(x2, rows), None, M
    y = _lib.result(out, (M, N), dtype, out_dtype, device)
    if keep and q is None:
        q = _new((n, K), device)
    ws, nws = _workspace(device, "moe_mx4_grouped_mm_workspace_bytes", M, n, E, K, int(q is not None))
    _lib.call("moe_mx4_grouped_mm", device, *_pointers(x2, q), n, w4.codes.data_ptr(), w4.scales.data_ptr(), _lib.ptr(bias),
              _lib.ptr(offsets), _lib.ptr(rows), M, E, N, K, _lib.DTYPE[dtype], y.data_ptr(), _lib.DTYPE[y.dtype], int(out is None),
              _lib.ptr(ws), nws)
    return y, q, w4, offsets, rows


class _GroupedMm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w4, offsets, bias, rows, out_dtype):
        need_x, need_w = ctx.needs_input_grad[:2]
        y, q, w4, offsets, rows = _run_grouped(x, w if w4 is None else w4, offsets, bias, rows, None, out_dtype, need_w)
        ctx.save_for_backward(*((q.codes, q.scales) if need_w else (None, None)), *((w4.codes, w4.scales) if need_x else (None, None)),
                              offsets, rows)
        ctx.dtype, ctx.experts = x.dtype, w4.shape[0]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xc, xs, wc, ws, offsets, rows = ctx.saved_tensors
        need_x, need_w, _, _, need_b = ctx.needs_input_grad[:5]
        dy = _lib.half_matrix(dy.to(ctx.dtype), "dy")
        dx = dw = db = None
        if need_x:
            dx = _grouped_dx(dy, _of(wc, ws), offsets)
        if need_w:
            dw, db = _grouped.mm_dw(dy, dequantize(_of(xc, xs), ctx.dtype), offsets, ctx.experts, x_rows=rows, bias=True)
        elif need_b:
            db = _bias_grad(dy, offsets, ctx.experts)
        return dx, dw, None, None, db if need_b else None, None, None


def grouped_mm(x, w, offsets, bias=None, rows=None, out=None, out_dtype=None):
    """y[p] = x[p] . w[e]^T (+ bias[e]) for the slots p of expert e, x and w in MXFP4; with rows x[rows[p]] in place of x[p] (an
    index outside x reads as zeros). x [M or any, K] bf16 or fp16 (quantised in the call) or an Mx4; w an Mx4 [E, N, K], or
    16-bit weights that are quantised in the call; offsets int32 [E + 1] (or None with E = 1), bias [E, N] of x's type. K a
    multiple of 32, N of 8. Slots behind the last expert: zeros in a new result, left as they are in `out`. out_dtype: the
    operands' 16-bit type or fp32.
    Differentiable as linear is, in x (not with rows: its gradient would add several slots' rows), 16-bit w and bias."""
    x_grad, w_grad = (None if isinstance(t, Mx4) else t for t in (x, w))
    if not _lib.wants_grad(x_grad, w_grad, bias):
        return _run_grouped(x, w, offsets, bias, rows, out, out_dtype, False)[0]
    if out is not None:
        raise ValueError("out= takes no gradient")
    if x_grad is None:
        raise ValueError("an Mx4 x takes no part in a backward pass: give its 16-bit form")
    if rows is not None and x.requires_grad:
        raise ValueError("x read through rows takes no gradient: index it first")
    return _GroupedMm.apply(x, w_grad, w if w_grad is None else None, offsets, bias, rows, out_dtype)
