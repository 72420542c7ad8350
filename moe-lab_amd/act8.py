"""Activations kept in 8 bits between a forward and its backward pass (moe_act8_*, moe_glu_fwd, moe_glu_bwd).

    codes, scales = pack(x)                  int8 codes like x, one exponent byte per 32 neighbours of a row (uint8)
    x = unpack(codes, scales, dtype)
    h = glu(gu)                              act(gate) * up of rows [gate | up], differentiable: its backward pass reads 8 bits
                                             (pack, unpack, glu_forward and glu_backward have no gradient themselves)

A value is code * 2^(scale - 133), off by at most half a step 2^(scale - 134). The exponent is the block's largest, one more
where that one would round to 128 steps, so half a step is at most 1/127.5 of the block's largest value, and a block is as
exact at 1e-30 as at 1e30; 255 marks a block that held an infinity or NaN and reads as NaN.
Against 16 bits this halves what a GLU keeps: 8.25 bits per value. int8 rather than an 8-bit float: activations of one
neighbourhood are of one size, and over a block a uniform step errs by about 0.7% of its rms, e4m3 by 2.6%.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib

BLOCK = 32


def check_codes(codes, scales, shape, device):
    """codes [rows, C] and scales [rows, C / 32], checked and contiguous."""
    _lib.require_device(codes, "codes")
    _lib.multiple_of(shape[1], BLOCK, "columns")
    return (_lib.plain(codes, "codes", shape, device, torch.int8),
            _lib.plain(scales, "scales", (shape[0], shape[1] // BLOCK), device, torch.uint8))


def pack(x):
    """x [M, C] in bf16 or fp16, C a multiple of 32 -> (codes int8 [M, C], scales uint8 [M, C / 32])."""
    x = _lib.half_matrix(x, "x")
    M, C = x.shape
    _lib.multiple_of(C, BLOCK, "columns")
    codes = torch.empty((M, C), dtype=torch.int8, device=x.device)
    scales = torch.empty((M, C // BLOCK), dtype=torch.uint8, device=x.device)
    _lib.call("moe_act8_pack", x.device, x.data_ptr(), x.stride(0), M, C, _lib.DTYPE[x.dtype], codes.data_ptr(),
              scales.data_ptr())
    return codes, scales


def unpack(codes, scales, dtype=torch.bfloat16):
    """The values that codes and scales stand for, in bf16, fp16 or fp32: exact in the type they came from and in fp32, but
    for 65536 in fp16, to which fp16 values from 65280 on are kept: 65504 there, not infinity."""
    if dtype not in _lib.DTYPE:
        raise TypeError(f"dtype {dtype}: bf16, fp16 or fp32 expected")
    if codes.dim() != 2:
        raise ValueError(f"codes have shape {tuple(codes.shape)}: [rows, columns] expected")
    codes, scales = check_codes(codes, scales, tuple(codes.shape), codes.device)
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    _lib.call("moe_act8_unpack", codes.device, codes.data_ptr(), scales.data_ptr(), codes.shape[0], codes.shape[1],
              out.data_ptr(), _lib.DTYPE[dtype])
    return out


def _check_glu(act, F):
    if act not in (_lib.ACT_SWIGLU, _lib.ACT_GEGLU, _lib.ACT_GPTOSS):
        raise ValueError(f"act {act}: ACT_SWIGLU, ACT_GEGLU or ACT_GPTOSS expected")
    _lib.multiple_of(F, BLOCK, "F")


def _glu_rows(gu):
    gu = _lib.half_matrix(gu, "gu")
    if gu.shape[1] % 2:
        raise ValueError(f"gu has {gu.shape[1]} columns: gate and up halves expected")
    return gu, gu.shape[0], gu.shape[1] // 2


def glu_forward(gu, act=_lib.ACT_SWIGLU, keep=True):
    """gu [M, 2 F] (gate columns, then up), F a multiple of 32 -> (h [M, F] = act(gate, up), codes, scales), the last two gu's
    8-bit form from the same pass (None without keep)."""
    gu, M, F = _glu_rows(gu)
    _check_glu(act, F)
    h = torch.empty((M, F), dtype=gu.dtype, device=gu.device)
    codes = scales = None
    if keep:
        codes = torch.empty((M, 2 * F), dtype=torch.int8, device=gu.device)
        scales = torch.empty((M, 2 * F // BLOCK), dtype=torch.uint8, device=gu.device)
    _lib.call("moe_glu_fwd", gu.device, gu.data_ptr(), gu.stride(0), M, F, int(act), _lib.DTYPE[gu.dtype], h.data_ptr(),
              _lib.ptr(codes), _lib.ptr(scales))
    return h, codes, scales


def glu_backward(codes, scales, dh, act=_lib.ACT_SWIGLU, wts=None, gu=None):
    """The GLU's backward pass from its kept input (codes and scales, or both None and gu itself), dh [M, F] in bf16, fp16 or,
    with codes, fp32, and a weight per row wts fp32 [M] (None: 1), for rows that are summed with these weights later on:
    (dgu [M, 2 F] = wts dh act'(gate, up), h [M, F] times wts, dwts fp32 [M] = sum of dh h). Results in gu's type, from codes in
    dh's (bf16 for fp32 dh)."""
    _lib.require_device(dh, "dh")
    if dh.dim() != 2 or dh.dtype not in _lib.DTYPE:
        raise TypeError(f"dh is {dh.dtype} {tuple(dh.shape)}: [M, F] in bf16, fp16 or fp32 expected")
    M, F = dh.shape
    _check_glu(act, F)
    dt = torch.bfloat16 if dh.dtype == torch.float32 else dh.dtype
    if gu is not None:
        if codes is not None or scales is not None:
            raise ValueError("either codes and scales, or gu")
        dt = gu.dtype
        gu = _lib.half_matrix(gu, "gu", 2 * F, dh.device, None if dh.dtype == torch.float32 else dt)
        if gu.shape[0] != M:
            raise ValueError(f"gu has {gu.shape[0]} rows, dh {M}")
    else:
        if codes is None or scales is None:
            raise ValueError("either codes and scales, or gu")
        codes, scales = check_codes(codes, scales, (M, 2 * F), dh.device)
    dh = _lib.plain(dh, "dh", (M, F), dh.device, dh.dtype)
    wts = _lib.plain(wts, "wts", (M,), dh.device, torch.float32)
    dgu = torch.empty((M, 2 * F), dtype=dt, device=dh.device)
    hw = torch.empty((M, F), dtype=dt, device=dh.device)
    dwts = torch.empty(M, dtype=torch.float32, device=dh.device)
    _lib.call("moe_glu_bwd", dh.device, _lib.ptr(codes), _lib.ptr(scales), _lib.ptr(gu), 0 if gu is None else gu.stride(0),
              dh.data_ptr(), _lib.DTYPE[dh.dtype], _lib.ptr(wts), M, F, int(act), _lib.DTYPE[dt], dgu.data_ptr(),
              hw.data_ptr(), dwts.data_ptr())
    return dgu, hw, dwts


class _Glu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu, act, checkpoint):
        h, codes, scales = glu_forward(gu, act, keep=checkpoint)
        ctx.save_for_backward(codes, scales, None if checkpoint else gu)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        codes, scales, gu = ctx.saved_tensors
        return glu_backward(codes, scales, dh, act=ctx.act, gu=gu)[0], None, None


def glu(gu, act=_lib.ACT_SWIGLU, checkpoint=True):
    """h [M, F] = act(gate, up) of gu [M, 2 F], differentiable. checkpoint: the backward pass keeps gu in 8 bits, so that its
    gradient is the function's at these values; else in 16."""
    if not _lib.wants_grad(gu):
        return glu_forward(gu, act, keep=False)[0]
    return _Glu.apply(gu, act, checkpoint)
