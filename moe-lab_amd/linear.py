"""One product of 16-bit matrices with bias, activation and residual in its epilogue, and its gradients (moe_linear):

    y = linear(x, w, bias=b, act=SILU, residual=r)        act(x w^T + b) + r, differentiable in x, w, b and r

for the dense parts beside the experts: shared experts, projections. Sums, bias, activation and residual are fp32, rounded
once. The reference runs these as stock modules (reference e2e.py:66-68, 146-147).
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib, act8

NONE, SILU, GELU = 0, 1, 2   # no activation; z * sigmoid(z); tanh-GELU


def _rows(t, name, cols, device, dtype):
    return _lib.half_matrix(t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t, name, cols, device, dtype)


def _workspace(size, T, N, K, device):
    n = getattr(_lib.lib(), size)(T, N, K)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None, n


# dz, x and w as half_matrix and plain return them
def _dx(dz, w):
    (T, N), K = dz.shape, w.shape[1]
    dx = torch.empty((T, K), dtype=w.dtype, device=w.device)
    ws, nws = _workspace("moe_linear_dx_workspace_bytes", T, N, K, w.device)
    _lib.call("moe_linear_dx", w.device, dz.data_ptr(), w.data_ptr(), T, dz.stride(0), N, K, _lib.DTYPE[w.dtype], dx.data_ptr(),
              _lib.ptr(ws), nws)
    return dx


def _dw(dz, x, bias):
    (T, N), K = dz.shape, x.shape[1]
    dw = torch.empty((N, K), dtype=dz.dtype, device=dz.device)
    db = torch.empty(N, dtype=dz.dtype, device=dz.device) if bias else None
    ws, nws = _workspace("moe_linear_dw_workspace_bytes", T, N, K, dz.device)
    _lib.call("moe_linear_dw", dz.device, dz.data_ptr(), x.data_ptr(), T, dz.stride(0), x.stride(0), N, K, _lib.DTYPE[dz.dtype],
              dw.data_ptr(), _lib.ptr(db), _lib.ptr(ws), nws)
    return dw, db


def _forward(x, w, bias, act, residual, out_dtype, keep_z):
    """y [..., N] and z [T, N] (None unless keep_z)."""
    return _run(x, w, bias, act, residual, out_dtype, keep_z)[:2]


def _run(x, w, bias, act, residual, out_dtype, keep_z):
    """y, z, and x [T, K] and w as the kernels read them."""
    _lib.require_device(w, "w")
    if w.dim() != 2:
        raise ValueError(f"w has shape {tuple(w.shape)}: [N, K] expected")
    if w.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"w is {w.dtype}: bf16 or fp16 expected")
    N, K = w.shape
    _lib.multiple_of(N, 8, "N")
    _lib.multiple_of(K, 8, "K")
    if act not in (NONE, SILU, GELU):
        raise ValueError(f"act {act}: NONE, SILU or GELU expected")
    w = _lib.plain(w, "w", (N, K), w.device, w.dtype)
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x has shape {tuple(x.shape)}: [..., {K}] expected")
    x2 = _rows(x, "x", K, w.device, w.dtype)
    bias = _lib.plain(bias, "bias", (N,), w.device, w.dtype)
    residual = _lib.plain(residual, "residual", (*x.shape[:-1], N), w.device, w.dtype)
    T = x2.shape[0]
    y = _lib.result(None, (T, N), w.dtype, out_dtype, w.device)
    z = torch.empty((T, N), dtype=w.dtype, device=w.device) if keep_z else None
    ws, nws = _workspace("moe_linear_workspace_bytes", T, N, K, w.device)
    _lib.call("moe_linear", w.device, x2.data_ptr(), w.data_ptr(), _lib.ptr(bias), _lib.ptr(residual), int(act), T,
              x2.stride(0), N, K, _lib.DTYPE[w.dtype], y.data_ptr(), _lib.DTYPE[y.dtype], _lib.ptr(z), _lib.ptr(ws), nws)
    return y.view(*x.shape[:-1], N), z, x2, w


def act_backward(dy, z, act, codes=None, scales=None):
    """dz = dy act'(z) [T, N] from z, or (z None) from its 8-bit form."""
    dy = _lib.half_matrix(dy, "dy")
    T, N = dy.shape
    _lib.multiple_of(N, 8, "N")
    if act not in (SILU, GELU):
        raise ValueError(f"act {act}: SILU or GELU expected")
    if (z is None) != (codes is not None) or (codes is None) != (scales is None):
        raise ValueError("either z, or codes and scales")
    z = _lib.plain(z, "z", (T, N), dy.device, dy.dtype)
    if codes is not None:
        codes, scales = act8.check_codes(codes, scales, (T, N), dy.device)
    return _act_backward(dy, z, act, codes, scales)


def _act_backward(dy, z, act, codes, scales):
    T, N = dy.shape
    dz = torch.empty((T, N), dtype=dy.dtype, device=dy.device)
    _lib.call("moe_linear_act_bwd", dy.device, dy.data_ptr(), dy.stride(0), _lib.ptr(z), _lib.ptr(codes), _lib.ptr(scales),
              int(act), T, N, _lib.DTYPE[dy.dtype], dz.data_ptr())
    return dz


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, act, residual, out_dtype, checkpoint):
        need_z = act != NONE and any(ctx.needs_input_grad[:3])
        y, z, x2, w2 = _run(x, w, bias, act, residual, out_dtype, need_z)
        codes = scales = None
        if need_z and checkpoint:
            codes, scales = act8.pack(z)
            z = None
        # the inputs themselves where the kernels read them in place, so that a change before the backward pass is noticed
        in_place = x2.data_ptr() == x.data_ptr() and x.is_contiguous()
        ctx.save_for_backward(x if in_place else x2, w2, z, codes, scales)
        ctx.act, ctx.x_shape = act, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, z, codes, scales = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = dy.to(w.dtype)
        dx = dw = db = None
        if need_x or need_w or need_b:
            dz = _rows(dy, "dy", w.shape[0], w.device, w.dtype)
            if ctx.act != NONE:
                dz = _act_backward(dz, z, ctx.act, codes, scales)
            if need_x:
                dx = _dx(dz, w).view(ctx.x_shape)
            if need_w or need_b:
                dw, db = _dw(dz, x.view(-1, w.shape[1]) if x.dim() != 2 else x, need_b)
        return dx, dw if need_w else None, db, None, dy if ctx.needs_input_grad[4] else None, None, None


def linear(x, w, bias=None, act=NONE, residual=None, out_dtype=None, checkpoint=False):
    """act(x w^T + bias) + residual. x [..., K], w [N, K], bias [N], residual [..., N], all bf16 or all fp16; N and K
    multiples of 8. out_dtype: the operands' type or fp32.
    Differentiable; the backward pass of an activation needs z = x w^T + bias, which is kept in 16 bits, or with checkpoint in
    8 (act8.pack; N a multiple of 32). Gradients of a result in fp32 are rounded to the operands' type first."""
    if checkpoint and act != NONE:
        _lib.multiple_of(w.shape[0], 32, "N with checkpoint")
    if not _lib.wants_grad(x, w, bias, residual):
        return _forward(x, w, bias, act, residual, out_dtype, False)[0]
    return _Linear.apply(x, w, bias, act, residual, out_dtype, checkpoint)
