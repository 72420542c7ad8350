"""Plain 64-bit forms of MXFP4 and of the routing by scores, for the tests."""
import math

import torch

import dense_helpers as H
from moelab_amd import _lib, mx4

MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def nearest(x):
    """x [..., K] -> (codes 0 .. 15, exponent bytes, values) of its MXFP4 form in 64 bits, from the borders between neighbours."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(top)
    safe = torch.where(bad | (top == 0), torch.ones_like(top), top)
    e = torch.frexp(safe)[1].to(torch.int64) - 1 - 2          # floor(log2) - 2
    byte = torch.where(top == 0, torch.zeros_like(e), (e + 127).clamp(min=0))
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    r = torch.where((bad | (byte == 0))[..., None], torch.zeros_like(b), b * H.pow2(-(byte - 127).clamp(-127, 127))[..., None])
    a = r.abs()
    code = torch.zeros_like(a, dtype=torch.int64)
    for i in range(7):   # on the border the even code wins
        mid = (MAGS[i] + MAGS[i + 1]) / 2
        code += (a >= mid) if i % 2 else (a > mid)
    v = torch.tensor(MAGS, dtype=torch.float64, device=x.device)[code] * torch.sign(r) * H.pow2(byte.clamp(1, 254) - 127)[..., None]
    v = torch.where(bad[..., None], torch.full_like(v, math.nan), v)
    code = code + 8 * (torch.signbit(r) & ~bad[..., None] & (byte > 0)[..., None])
    return code.reshape(x.shape), byte, v.reshape(x.shape)


def values(x):
    return nearest(x)[2]


def unpacked(q):
    """Codes [..., K] and exponent bytes [..., K / 32] of an Mx4."""
    codes = torch.stack([q.codes & 15, q.codes >> 4], -1).reshape(q.shape).to(torch.int64)
    return codes, mx4.to_packed(q)[1].to(torch.int64)


def random_mx4(E, N, K, seed=0):
    """Random codes and exponents around 1 / sqrt(K) as an Mx4 [E, N, K] and its values in 64 bits."""
    g = torch.Generator(device=H.DEV).manual_seed(seed + 31 * N + K)
    words = torch.randint(-2 ** 31, 2 ** 31, (E, N, K // 8), generator=g, device=H.DEV).to(torch.int32)
    e = 126 - int(math.log2(K) / 2)
    scales = torch.randint(e - 2, e + 2, (E, N, K // 32), generator=g, device=H.DEV).to(torch.uint8)
    q = mx4.from_packed(words, scales)
    codes = torch.stack([q.codes & 15, q.codes >> 4], -1).reshape(E, N, K).long()
    table = torch.tensor(MAGS + tuple(-m for m in MAGS), dtype=torch.float64, device=H.DEV)
    return q, table[codes] * H.pow2(scales.long() - 127).repeat_interleave(32, -1)


def first(q):
    """The one matrix of an Mx4 [1, N, K]."""
    return mx4.Mx4(q.codes[0].contiguous(), q.scales)


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", norm=True, scale=1.0):
    """ids, weights and the scores in 64 bits, token by token."""
    ids, wts, scores = [], [], []
    E = logits.shape[1]
    n = E // groups
    for row in logits.double().cpu():
        row = torch.where(torch.isnan(row), torch.full_like(row, -math.inf), row)
        if score == "softmax":
            m = row.max()
            p = torch.where(row == m, torch.ones_like(row), torch.exp(row - m)) if m > -math.inf else torch.zeros_like(row)
            p = torch.where(row == -math.inf, torch.zeros_like(p), p)
            p = p / p.sum() if p.sum() > 0 else p
        else:
            p = torch.sigmoid(row)
        c = row if bias is None else p + bias.double().cpu()
        c = torch.where((row == -math.inf) | torch.isnan(c), torch.full_like(c, -math.inf), c)
        vals = c if group_score == "max" or bias is not None else torch.where(c == -math.inf, c, p)
        gv = []
        for g in range(groups):
            top = sorted(vals[g * n:(g + 1) * n].tolist(), reverse=True)
            gv.append(top[0] if group_score == "max" or groups == 1 else top[0] + top[1])
        gv = [v if v == v else -math.inf for v in gv]
        kept = sorted(range(groups), key=lambda g: (-gv[g], g))[:top_groups]
        order = sorted((e for g in kept for e in range(g * n, (g + 1) * n)), key=lambda e: (-float(c[e]), e))[:k]
        live = torch.tensor([c[e] > -math.inf for e in order])
        if norm and score == "softmax":
            lv = row[order]
            m = lv[live].max() if live.any() else 0.0
            s = torch.where(live, torch.where(lv == m, torch.ones_like(lv), torch.exp(lv - m)), torch.zeros_like(lv))
        else:
            s = torch.where(live, p[order], torch.zeros(k, dtype=torch.float64))
        if norm:
            s = s / s.sum() if s.sum() > 0 else torch.zeros_like(s)
        ids.append(torch.tensor(order))
        wts.append(s * scale)
    return torch.stack(ids).to(logits.device), torch.stack(wts).to(logits.device)


def linear_dx(dz, w4):
    """The library's call by itself."""
    (T, N), K = dz.shape, w4.shape[1]
    dx = torch.empty((T, K), dtype=dz.dtype, device=dz.device)
    ws, nws = mx4._workspace(dz.device, "moe_mx4_linear_dx_workspace_bytes", T, N, K)
    _lib.call("moe_mx4_linear_dx", dz.device, dz.data_ptr(), dz.stride(0), w4.codes.data_ptr(), w4.scales.data_ptr(), T, N, K,
              _lib.DTYPE[dz.dtype], dx.data_ptr(), _lib.ptr(ws), nws)
    return dx
