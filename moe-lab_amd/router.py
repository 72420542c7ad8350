"""Fused router on gfx950: logits [T, E] -> top-k ids [T, k] int32 + weights [T, k] fp32.

Mirrors reference moelab/router.py (semantics :1-12, ``topk_norm`` :71-80):
  * norm=True: weights = softmax over the top-k logits (= the renormalised full softmax);
    norm=False: the full-softmax probabilities of the chosen experts (DeepSeek-V2 greedy);
  * ties: the lowest expert id wins; NaN logits count as -inf; with fewer than k finite logits the
    remaining slots take the lowest unused ids with weight 0;
  * E <= 1024, k <= min(E, 32).
``topk_scored`` and ``route_scored`` are the routers that the reference leaves to the stock gate (reference e2e.py:129-150):
softmax or sigmoid scores, a bias that only ranks, groups of experts of which the best few are kept, and a gradient.
``route`` adds what the reference leaves to the stock gate GEMV (reference e2e.py:57-59): the logits
x . Wr^T (+ bias) are computed in the same kernel, in fp32, in one fixed reduction order, so a CPU
restatement reproduces them bit for bit and the chosen ids are exact.
"""
import functools
import math
import operator

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_SCORES = {"softmax": 0, "sigmoid": 1}   # MOE_SCORE_*
_GROUP_SCORES = {"max": 0, "top2": 1}    # MOE_GROUP_*


def topk_norm(logits, k, norm=True, scale=1.0):
    """logits [..., E] (fp32, bf16 or fp16, on the GPU) -> (idx [T, k] int32, wts [T, k] fp32)."""
    E = logits.shape[-1]
    assert E <= 1024 and k <= min(E, 32), (E, k)
    _lib.require_device(logits, "logits")
    lg = logits.reshape(-1, E).contiguous()
    T = lg.shape[0]
    if lg.dtype not in _lib.DTYPE:
        lg = lg.float()
    idx = torch.empty((T, k), dtype=torch.int32, device=lg.device)
    wts = torch.empty((T, k), dtype=torch.float32, device=lg.device)
    rc = _lib.lib().moe_topk(_lib.ptr(lg), _lib.DTYPE[lg.dtype], T, E, k, int(bool(norm)), float(scale),
                             _lib.ptr(idx), _lib.ptr(wts), _lib.stream_of(lg.device))
    _lib.check("moe_topk", rc)
    return idx, wts


def reserve(device, T):
    """Nothing to size: the router's launches need no scratch of their own (kept for callers that size every buffer
    before capturing a HIP graph)."""
    return None


def route(x, wr, k, bias=None, norm=True, scale=1.0, return_logits=False):
    """Gate GEMV, then the router tails (two launches). x [T, d] bf16, wr [E, d] bf16, bias [E] (any float) or None.
    Returns (idx [T, k] int32, wts [T, k] fp32[, logits [T, E] fp32])."""
    _lib.require_device(x, "x")
    assert x.dtype == torch.bfloat16 and wr.dtype == torch.bfloat16, "router takes bf16 x and Wr"
    T, d = x.shape
    E = wr.shape[0]
    assert wr.shape[1] == d and E <= 1024 and 1 <= k <= min(E, 32), (x.shape, wr.shape, k)
    x = x.contiguous()
    wr = wr.contiguous()
    b = None if bias is None else bias.to(torch.float32).contiguous()
    logits = torch.empty((T, E), dtype=torch.float32, device=x.device)
    idx = torch.empty((T, k), dtype=torch.int32, device=x.device)
    wts = torch.empty((T, k), dtype=torch.float32, device=x.device)
    rc = _lib.lib().moe_router(_lib.ptr(x), _lib.ptr(wr), _lib.ptr(b), T, d, E, k, int(bool(norm)), float(scale),
                               _lib.ptr(logits), _lib.ptr(idx), _lib.ptr(wts), None, _lib.stream_of(x.device))
    _lib.check("moe_router", rc)
    return (idx, wts, logits) if return_logits else (idx, wts)


def route_group(x, wr, k, bias=None, norm=True, scale=1.0):
    """route() plus the stable slot grouping, built by the router's own launches (moe_router_group: after the logits
    launch, the launch that runs the tails sorts the T*k slots by expert with a wave prefix sum of the counts).
    Returns (idx, wts, logits, (counts [E], offsets [E+1], sorted [T*k], active [E], meta [2])), the grouping as
    group(idx, E) returns it."""
    _lib.require_device(x, "x")
    assert x.dtype == torch.bfloat16 and wr.dtype == torch.bfloat16, "router takes bf16 x and Wr"
    T, d = x.shape
    E = wr.shape[0]
    assert wr.shape[1] == d and E <= 1024 and 1 <= k <= min(E, 32), (x.shape, wr.shape, k)
    L = _lib.lib()
    x = x.contiguous()
    wr = wr.contiguous()
    b = None if bias is None else bias.to(torch.float32).contiguous()
    dev = x.device
    logits = torch.empty((T, E), dtype=torch.float32, device=dev)
    idx = torch.empty((T, k), dtype=torch.int32, device=dev)
    wts = torch.empty((T, k), dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    srt = torch.empty(max(T * k, 1), dtype=torch.int32, device=dev)
    active = torch.empty(E, dtype=torch.int32, device=dev)
    meta = torch.empty(2, dtype=torch.int32, device=dev)
    rc = L.moe_router_group(_lib.ptr(x), _lib.ptr(wr), _lib.ptr(b), T, d, E, k, int(bool(norm)), float(scale),
                            _lib.ptr(logits), _lib.ptr(idx), _lib.ptr(wts), _lib.ptr(counts), _lib.ptr(offsets),
                            _lib.ptr(srt), _lib.ptr(active), _lib.ptr(meta), _lib.stream_of(dev))
    _lib.check("moe_router_group", rc)
    return idx, wts, logits, (counts, offsets, srt[:T * k], active, meta)


def group(idx, E):
    """Stable slot grouping on the GPU: returns (counts [E], offsets [E+1], sorted [T*k], active [E], meta [2])."""
    _lib.require_device(idx, "idx")
    flat = idx.reshape(-1).to(torch.int32).contiguous()
    n = flat.numel()
    dev = flat.device
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
    srt = torch.empty(max(n, 1), dtype=torch.int32, device=dev)
    active = torch.empty(E, dtype=torch.int32, device=dev)
    meta = torch.empty(2, dtype=torch.int32, device=dev)
    rc = _lib.lib().moe_group(_lib.ptr(flat), n, E, _lib.ptr(counts), _lib.ptr(offsets), _lib.ptr(srt),
                              _lib.ptr(active), _lib.ptr(meta), _lib.stream_of(dev))
    _lib.check("moe_group", rc)
    return counts, offsets, srt[:n], active, meta


@functools.lru_cache(maxsize=1024)
def _settings(E, k, score, groups, top_groups, group_score, norm, scale):
    """The descriptor of these settings, checked, without a bias."""
    kind, by = _SCORES.get(score), _GROUP_SCORES.get(group_score)
    if kind is None or by is None:
        raise ValueError(f"score {score!r}, group_score {group_score!r}: one of {list(_SCORES)}, one of {list(_GROUP_SCORES)} expected")
    if not 1 <= E <= 1024 or not 1 <= groups <= 64 or E % groups or not 1 <= top_groups <= groups:
        raise ValueError(f"{E} experts in {groups} groups, {top_groups} kept: at most 1024 in at most 64 equal groups expected")
    if groups > 1 and group_score == "top2" and E < 2 * groups:
        raise ValueError("group_score 'top2': groups of two experts at least expected")
    if not 1 <= k <= min(32, top_groups * (E // groups)):
        raise ValueError(f"k = {k}: 1 to {min(32, top_groups * (E // groups))} expected (32, or the experts in the kept groups)")
    if not math.isfinite(scale):
        raise ValueError(f"scale {scale}: a finite number expected")
    return _lib.Scored(E, k, kind, groups, top_groups, by, norm, scale, None)


def _scored(E, k, score, bias, groups, top_groups, group_score, norm, scale, device):
    """The call's descriptor, its arguments checked, and the bias that it points to."""
    desc = _settings(E, operator.index(k), score, operator.index(groups), operator.index(top_groups), group_score,
                     1 if norm else 0, float(scale))
    if bias is None:
        return desc, None
    if bias.dtype not in _lib.DTYPE or tuple(bias.shape) != (E,) or bias.device != device:
        raise ValueError(f"bias {bias.dtype} {tuple(bias.shape)} on {bias.device}: floating [{E}] on {device} expected")
    bias = _lib.dense(bias.detach(), torch.float32)
    return _with_bias(desc, bias), bias


def _with_bias(desc, bias):
    desc = _lib.Scored.from_buffer_copy(desc)
    desc.bias = bias.data_ptr()
    return desc


def _topk_scored(lg, desc):
    T = lg.shape[0]
    k, device = desc.k, lg.device
    idx = torch.empty(T, k, dtype=torch.int32, device=device)
    wts = torch.empty(T, k, dtype=torch.float32, device=device)
    _lib.call("moe_topk_scored", device, desc, lg.data_ptr(), _lib.DTYPE[lg.dtype], T, idx.data_ptr(), wts.data_ptr())
    return idx, wts


class _TopkScored(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, desc, bias):
        lg = _lib.dense(logits)
        idx, wts = _topk_scored(lg, desc)
        # the backward pass reads in the bias which experts it took out: as it was here, also where its owner moves it in between
        ctx.save_for_backward(lg, None if bias is None else bias.clone(), idx)
        ctx.desc = desc
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return idx, wts

    @staticmethod
    @once_differentiable
    def backward(ctx, _, dwts):
        if dwts is None:
            return None, None, None
        lg, bias, idx = ctx.saved_tensors
        desc = ctx.desc
        if bias is not None:
            desc = _with_bias(desc, bias)
        dw, dl = _lib.dense(dwts, torch.float32), torch.empty_like(lg)
        _lib.call("moe_topk_scored_bwd", lg.device, desc, lg.data_ptr(), _lib.DTYPE[lg.dtype], lg.shape[0], idx.data_ptr(),
                  dw.data_ptr(), dl.data_ptr())
        return dl, None, None


def topk_scored(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", norm=True, scale=1.0):
    """logits [..., E] (fp32, bf16 or fp16) -> (idx [T, k] int32, wts [T, k] fp32); differentiable: wts in logits.
    score: "softmax" or "sigmoid" of the logits. bias [E]: added to the scores for ranking only (without one the logits rank).
    groups: experts E / groups * g .. form group g; only the top_groups groups of largest value stay, a group's value being its
    largest ranking value (group_score "max") or the sum of its two largest ("top2"). idx: the k experts that rank highest, best
    first, of equals the lowest id. wts: scale * score, with norm divided by the k scores' sum (0 where that is 0).
    NaN logits count as -inf; experts at -inf are chosen last, with weight 0 and no gradient. E <= 1024, groups <= 64, k <= 32.
    Scores are ranked in fp64. The bias and the choice have no gradient; the bias may change before the backward pass."""
    _lib.require_device(logits, "logits")
    if logits.dim() < 1:
        raise ValueError("logits [..., E] expected")
    if logits.dtype not in _lib.DTYPE:
        raise TypeError(f"logits are {logits.dtype}: fp32, bf16 or fp16 expected")
    lg = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    desc, bias = _scored(lg.shape[1], k, score, bias, groups, top_groups, group_score, norm, scale, lg.device)
    if _lib.wants_grad(logits):
        return _TopkScored.apply(lg, desc, bias)
    return _topk_scored(_lib.dense(lg), desc)


def route_scored(x, wr, k, wr_bias=None, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", norm=True,
                 scale=1.0, return_logits=False):
    """topk_scored on the logits x . wr^T (+ wr_bias), which are route's: fp32, in one fixed order. x [T, d] bf16, wr [E, d]
    bf16, wr_bias [E] (any float) or None, the other arguments as topk_scored's. Returns (idx, wts[, logits [T, E] fp32]).
    No gradient: for training, topk_scored on logits of linear.linear(x, wr, out_dtype=torch.float32)."""
    _lib.require_device(x, "x")
    if x.dim() != 2 or wr.dim() != 2 or x.shape[1] != wr.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and wr {tuple(wr.shape)}: [T, d] and [E, d] expected")
    if x.dtype != torch.bfloat16 or wr.dtype != torch.bfloat16:
        raise TypeError(f"x {x.dtype} and wr {wr.dtype}: bf16 expected")
    if wr.device != x.device:
        raise ValueError(f"wr is on {wr.device}, x on {x.device}")
    if _lib.wants_grad(x, wr, wr_bias):
        raise NotImplementedError("route_scored has no gradient: topk_scored on linear.linear's logits has one")
    (T, d), E = x.shape, wr.shape[0]
    _lib.multiple_of(d, 8, "d")
    desc, bias = _scored(E, k, score, bias, groups, top_groups, group_score, norm, scale, x.device)
    x, wr = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format) for t in (x, wr))
    if wr_bias is not None:
        if wr_bias.dtype not in _lib.DTYPE or tuple(wr_bias.shape) != (E,) or wr_bias.device != x.device:
            raise ValueError(f"wr_bias {wr_bias.dtype} {tuple(wr_bias.shape)} on {wr_bias.device}: floating [{E}] on {x.device} expected")
        wr_bias = _lib.dense(wr_bias, torch.float32)
    logits = torch.empty((T, E), dtype=torch.float32, device=x.device)
    idx = torch.empty((T, k), dtype=torch.int32, device=x.device)
    wts = torch.empty((T, k), dtype=torch.float32, device=x.device)
    _lib.call("moe_router_scored", x.device, desc, x.data_ptr(), wr.data_ptr(), _lib.ptr(wr_bias), T, d, logits.data_ptr(),
              idx.data_ptr(), wts.data_ptr())
    return (idx, wts, logits) if return_logits else (idx, wts)
