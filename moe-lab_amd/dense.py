"""The expert layer on 16-bit weights, forward and backward (moe_mlp_fwd, moe_mlp_bwd): what experts.run_experts computes from
packed weights, for a model before it is quantised, or in training.

    y = experts_mlp(x, idx, wts, w_gate_up, w_down)     differentiable in x, wts, w_gate_up, w_down and residual
    y = glu_mlp(x, w_gate, w_up, w_down)                a dense GLU layer (shared experts) on linear.linear

The forward call groups the slots by expert (the stable grouping of router.group), multiplies gate and up for each slot with
token rows read through the slot list (no gathered copy of x), applies the GLU, multiplies down, and sums each token's slots
in fp32 in their order; the backward call reads dy through the same list. Between two launches h and the gradients
of gate and up are in 16 bits (the matrix cores' operands); dh and the slots' rows of y and dx are fp32. For the
backward pass the gate/up rows are kept in 8 bits (act8) or 16.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib, act8, linear as _linear


def _desc(x, w_gate_up, w_down, act):
    _lib.require_device(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x has shape {tuple(x.shape)}: [T, d] expected")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x is {x.dtype}: bf16 or fp16 expected")
    T, d = x.shape
    if w_gate_up.dim() != 3 or w_down.dim() != 3:
        raise ValueError("w_gate_up [E, 2 F, d] and w_down [E, d, F] expected")
    E, F = w_down.shape[0], w_down.shape[2]
    _lib.multiple_of(d, 8, "d")
    act8._check_glu(act, F)
    w_gate_up = _lib.plain(w_gate_up, "w_gate_up", (E, 2 * F, d), x.device, x.dtype)
    w_down = _lib.plain(w_down, "w_down", (E, d, F), x.device, x.dtype)
    return _lib.Mlp(E, d, F, int(act), _lib.DTYPE[x.dtype], w_gate_up.data_ptr(), w_down.data_ptr()), w_gate_up, w_down


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _slot_lists(x, idx, wts):
    _lib.require_device(x, "x")
    T = x.shape[0]
    if idx.dim() != 2 or idx.shape[0] != T or idx.shape[1] < 1 or tuple(wts.shape) != tuple(idx.shape):
        raise ValueError(f"idx {tuple(idx.shape)} and wts {tuple(wts.shape)}: [{T}, k] expected")
    if idx.dtype not in (torch.int32, torch.int64) or wts.dtype not in _lib.DTYPE:
        raise TypeError(f"idx {idx.dtype} and wts {wts.dtype}: int32 (or int64) and a floating type expected")
    if idx.device != x.device or wts.device != x.device:
        raise ValueError("idx and wts must be on x's device")
    if idx.dtype == torch.int64:   # an id past 32 bits stays outside [0, E)
        idx = idx.clamp(-1, 2 ** 31 - 1)
    return _lib.dense(idx, torch.int32), _lib.dense(wts, torch.float32)


def _forward(x, idx, wts, w_gate_up, w_down, act, residual, out_dtype, keep):
    """keep: None (inference), "8" or "16". Returns y and what the backward pass reads: (x, keep buffer, gu, codes, scales)."""
    desc, w_gate_up, w_down = _desc(x, w_gate_up, w_down, act)
    x = _lib.plain(x, "x", tuple(x.shape), x.device, x.dtype)
    T, d = x.shape
    k, F = idx.shape[1], desc.F
    residual = _lib.plain(residual, "residual", (T, d), x.device, x.dtype)
    y = _lib.result(None, (T, d), x.dtype, out_dtype, x.device)
    if T == 0:
        return y, (x, None, None, None, None)
    L = _lib.lib()
    nkeep, nws = L.moe_mlp_keep_bytes(desc, T, k), L.moe_mlp_fwd_workspace_bytes(desc, T, k)
    gu = codes = scales = None
    if keep is None:   # one buffer: the grouping is scratch too
        ws = _bytes(nkeep + nws, x.device)
        kept, ws_ptr = None, ws.data_ptr() + nkeep
        keep_ptr = ws.data_ptr()
    else:
        ws, kept = _bytes(nws, x.device), _bytes(nkeep, x.device)
        ws_ptr, keep_ptr = ws.data_ptr(), kept.data_ptr()
        if keep == "8":
            codes = torch.empty((T * k, 2 * F), dtype=torch.int8, device=x.device)
            scales = torch.empty((T * k, 2 * F // act8.BLOCK), dtype=torch.uint8, device=x.device)
        else:
            gu = torch.empty((T * k, 2 * F), dtype=x.dtype, device=x.device)
    _lib.call("moe_mlp_fwd", x.device, desc, x.data_ptr(), idx.data_ptr(), wts.data_ptr(), T, k, _lib.ptr(residual),
              y.data_ptr(), _lib.DTYPE[y.dtype], keep_ptr, _lib.ptr(gu), _lib.ptr(codes), _lib.ptr(scales), ws_ptr, nws)
    return y, (x, kept, gu, codes, scales)


class _Experts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, idx, wts, w_gate_up, w_down, act, residual, out_dtype, checkpoint):
        idx32, wts32 = _slot_lists(x, idx, wts)
        needed = any(ctx.needs_input_grad[i] for i in (0, 2, 3, 4))
        y, (x2, kept, gu, codes, scales) = _forward(x, idx32, wts32, w_gate_up, w_down, act, residual, out_dtype,
                                                    ("8" if checkpoint else "16") if needed else None)
        ctx.save_for_backward(x if x2.data_ptr() == x.data_ptr() else x2, wts, w_gate_up, w_down, kept, gu, codes, scales)
        ctx.act, ctx.k = act, idx.shape[1]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, wts, w_gate_up, w_down, kept, gu, codes, scales = ctx.saved_tensors
        need_x, _, need_wts, need_gu, need_dn = ctx.needs_input_grad[:5]
        T, d = x.shape
        dy = dy.to(x.dtype)
        dx = torch.empty((T, d), dtype=x.dtype, device=x.device) if need_x else None
        # slots of an id outside [0, E) have no gradient; the kernel writes the others
        dwts = torch.zeros((T, ctx.k), dtype=torch.float32, device=x.device) if need_wts else None
        new = torch.empty if T else torch.zeros
        dwgu = new(w_gate_up.shape, dtype=x.dtype, device=x.device) if need_gu else None
        dwd = new(w_down.shape, dtype=x.dtype, device=x.device) if need_dn else None
        if T and (need_x or need_wts or need_gu or need_dn):
            desc, w_gate_up, w_down = _desc(x, w_gate_up, w_down, ctx.act)
            w32 = _lib.dense(wts.detach(), torch.float32)
            g = _lib.plain(dy, "dy", (T, d), x.device, x.dtype)
            nws = _lib.lib().moe_mlp_bwd_workspace_bytes(desc, T, ctx.k)
            ws = _bytes(nws, x.device)
            _lib.call("moe_mlp_bwd", x.device, desc, x.data_ptr(), w32.data_ptr(), g.data_ptr(), T, ctx.k, kept.data_ptr(),
                      _lib.ptr(gu), _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(dx), _lib.ptr(dwts), _lib.ptr(dwgu),
                      _lib.ptr(dwd), ws.data_ptr(), nws)
        return (dx, None, None if dwts is None else dwts.to(wts.dtype), dwgu, dwd, None,
                dy if ctx.needs_input_grad[6] else None, None, None)


def experts_mlp(x, idx, wts, w_gate_up, w_down, act=_lib.ACT_SWIGLU, residual=None, out_dtype=None, checkpoint=True):
    """y[t] = residual[t] + sum_j wts[t, j] w_down[e] . act(w_gate_up[e] . x[t]),  e = idx[t, j].
    x [T, d], w_gate_up [E, 2 F, d] (gate rows, then up), w_down [E, d, F], residual [T, d], all bf16 or all fp16; idx [T, k]
    int32 (int64 is converted), wts [T, k] floating. d a multiple of 8, F of 32. A slot whose id is outside [0, E) adds
    nothing. out_dtype: x's type or fp32.
    Differentiable; checkpoint: the gate/up rows are kept in 8 bits for the backward pass (half the memory; its gradients are
    the layer's at these values, about 1% off its own in the norm), else in 16 (0.3% off in bf16, 0.04% in fp16). Gradients of
    a result in fp32 are rounded to x's type first."""
    if not _lib.wants_grad(x, wts, w_gate_up, w_down, residual):
        idx, wts = _slot_lists(x, idx, wts)
        y = _forward(x, idx, wts, w_gate_up, w_down, act, residual, out_dtype, None)[0]
        return y
    return _Experts.apply(x, idx, wts, w_gate_up, w_down, act, residual, out_dtype, checkpoint)


def glu_mlp(x, w_gate, w_up, w_down, act=_lib.ACT_SWIGLU, residual=None, checkpoint=False):
    """residual + (a(x w_gate^T) * (x w_up^T)) w_down^T, a = SiLU (ACT_SWIGLU) or tanh-GELU (ACT_GEGLU): a dense GLU layer, as a
    model's shared experts are. x [..., d], w_gate and w_up [F, d], w_down [d, F]; differentiable."""
    acts = {_lib.ACT_SWIGLU: _linear.SILU, _lib.ACT_GEGLU: _linear.GELU}
    if act not in acts:
        raise ValueError(f"act {act}: ACT_SWIGLU or ACT_GEGLU expected")
    h = _linear.linear(x, w_gate, act=acts[act], checkpoint=checkpoint) * _linear.linear(x, w_up)
    return _linear.linear(h, w_down, residual=residual)
