"""Plain 64-bit forms of the 16-bit expert operators, and error bounds derived from their arithmetic, for the tests.

A result of type t that is rounded once from fp32 sums of R products is off by at most
    half_step(t) |ref|  +  (R + 8) 2^-23 sum |a| |b|  (+ half of fp16's smallest step, where it can be subnormal)
the first term the final rounding, the second the fp32 additions in any order (each off by at most 2^-24 of the running
magnitude; twice that for matrix instructions that truncate). Operands that are themselves rounded inside the call add their
half step once more, which the tests write out where it applies.
"""
import math

import torch

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def product_tol(ref, mags, R, dtype):
    return half_step(dtype) * ref.abs() + (R + 8) * 2.0 ** -23 * mags + tiny(dtype)


def check(got, ref, tol, what=""):
    """got within tol of ref, element by element; inf and NaN in the same places."""
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    rest = ~fine & ~torch.isnan(ref)
    assert torch.equal(got[rest], ref[rest]), f"{what}: infinities differ"
    gap = ((got - ref).abs() - tol)[fine]
    if gap.numel():
        worst = float(gap.max())
        assert worst <= 0, f"{what}: {int((gap > 0).sum())} of {gap.numel()} out of tolerance, by up to {worst:.3e}"


def randn(*shape, dtype, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 17 * sum(shape))
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def offsets_of(counts):
    return torch.tensor([0] + list(counts), device=DEV).cumsum(0).to(torch.int32)


def ranges(counts):
    lo = 0
    for e, n in enumerate(counts):
        yield e, slice(lo, lo + n)
        lo += n


def gelu(z):
    """tanh-GELU as z sigmoid(2 t): 1 + tanh(t) loses its digits far out on the negative side, also in 64 bits."""
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


def silu(z):
    return z * torch.sigmoid(z)


def glu(act, g, u):
    if act == 0:
        return silu(g) * u
    if act == 1:
        return gelu(g) * u
    g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
    return g * torch.sigmoid(1.702 * g) * (u + 1)


def pow2(e):
    """2^e in 64 bits from its bits (a library's pow need not be exact)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantise(v):
    """The 8-bit form's definition in 64 bits: v [M, C] -> codes, scales."""
    b = v.double().reshape(v.shape[0], -1, 32)
    a = b.abs().amax(-1)
    bad = ~torch.isfinite(a)
    a = torch.where(bad, torch.ones_like(a), a)
    s = torch.where(a > 0, torch.frexp(a)[1].double() + 126, torch.zeros_like(a)).clamp(0, 254)
    s = torch.where(torch.round(a * pow2(133 - s)) > 127, (s + 1).clamp(max=254), s)
    q = torch.round(b * pow2(133 - s)[..., None]).clamp(-127, 127)
    q = torch.where(bad[..., None], torch.zeros_like(q), q)
    return q.to(torch.int8).reshape(v.shape), torch.where(bad, torch.full_like(s, 255), s).to(torch.uint8)


def values(codes, scales):
    f = torch.where(scales == 255, math.nan, pow2(scales.to(torch.int64) - 133))
    return (codes.double().reshape(*scales.shape, 32) * f[..., None]).reshape(codes.shape)


def experts(x, idx, wts, wgu, wd, act, residual=None, kept=None):
    """The expert layer in the inputs' precision, slot by slot; kept: what the GLU reads in place of the gate/up rows [T, k, 2F]."""
    T, k = idx.shape
    E, F = wd.shape[0], wd.shape[2]
    out = []
    for t in range(T):
        acc = torch.zeros_like(x[t]) if residual is None else residual[t]
        for j in range(k):
            e = int(idx[t, j])
            if 0 <= e < E:
                gu = wgu[e] @ x[t] if kept is None else kept(t, j, wgu[e] @ x[t])
                acc = acc + wts[t, j] * (wd[e] @ glu(act, gu[:F], gu[F:]))
        out.append(acc)
    return torch.stack(out)
