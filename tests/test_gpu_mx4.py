"""MXFP4 on the GPU against 64-bit arithmetic: the quantisation code by code, products on every path (few rows quantised in the call,
few rows, the three tiles, split sums), ragged and empty groups, index lists, epilogues, gradients, layouts, captured calls."""
import math

import pytest
import torch

import dense_helpers as H
import mx4_helpers as M
from dense_helpers import DEV, TYPES
from moelab_amd import formats, grouped, mx4
from moelab_amd.linear import GELU, NONE, SILU
from test_gpu_linear import act_of, act_tol

pytestmark = pytest.mark.gpu
IDS = ["bf16", "fp16"]


def activations(T, K, dtype, seed=0):
    """Rows and channels of different size."""
    x = H.randn(T, K, dtype=torch.float32, seed=seed) * torch.exp(H.randn(1, K, dtype=torch.float32, seed=seed + 1))
    return x.to(dtype)


# -------------------------------------------------------------------------------------------------- quantisation
def check_form(x):
    q = mx4.quantize(x)
    codes, byte, v = M.nearest(x)
    got_codes, got_byte = M.unpacked(q)
    assert torch.equal(got_byte, byte)
    assert torch.equal(got_codes, codes)
    for dtype in (torch.bfloat16, torch.float32):
        H.check(mx4.dequantize(q, dtype), v, torch.zeros_like(v))
    with_inf = torch.isnan(v) | (v.abs() < 65520)
    H.check(mx4.dequantize(q, torch.float16)[with_inf], v[with_inf], (v.abs() * 2.0 ** -11 + 2.0 ** -25)[with_inf])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M_,K", [(1, 32), (3, 64), (5, 2880), (7, 256), (130, 288), (64, 4096), (1000, 160)])
def test_quantise(M_, K, dtype):
    x = activations(M_, K, dtype)
    x[::3, :32] = 0
    check_form(x)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_quantise_every_number(dtype):
    """Every 16-bit number next to a largest of every exponent it can have there; infinities and NaN in blocks of their own."""
    bits = torch.arange(65536, device=DEV).to(torch.int32).to(torch.int16).view(dtype)
    fine = bits[torch.isfinite(bits)]
    check_form(torch.cat([fine, torch.zeros((-len(fine)) % 32, dtype=dtype, device=DEV)]).reshape(-1, 32))
    mag = fine[fine > 0]
    for shift in (1, 2, 5, 40):   # each number with a larger one: other codes of the same numbers
        x = torch.zeros((len(mag), 32), dtype=dtype, device=DEV)
        x[:, 3], x[:, 17] = mag, -mag
        x[:, 30] = (mag.double() * 2.0 ** shift).clamp(max=float(torch.finfo(dtype).max)).to(dtype)
        check_form(x)
    x = torch.ones((4, 96), dtype=dtype, device=DEV)
    x[0, 40], x[1, 95], x[2, 0] = math.inf, -math.inf, math.nan
    check_form(x)
    assert torch.isnan(mx4.dequantize(mx4.quantize(x))[0, 32:64]).all()


def test_quantise_fp32_borders():
    """Numbers on each border between codes and an ulp to either side, for exponents over the whole range."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    near = torch.cat([mids, torch.nextafter(mids, mids * 0), torch.nextafter(mids, mids * 9)])
    near = torch.cat([near, -near[:10]])[:31]
    for e in (-140, -127, -125, -124, -123, -60, 0, 1, 90, 124):
        x = torch.zeros((2, 32), device=DEV)
        for i, top in enumerate((4.0, 7.9999995)):
            x[i, :31] = (near.double() * 2.0 ** e).float()
            x[i, 31] = (torch.tensor(top, dtype=torch.float64) * 2.0 ** e).float()
        check_form(x)


@pytest.mark.parametrize("shape", [(2, 3, 64), (0, 64), (3, 0, 64), (64,), (2, 2, 2, 96)])
def test_quantise_shapes(shape):
    x = H.randn(*shape, dtype=torch.bfloat16)
    q = mx4.quantize(x)
    want = x if x.dim() in (2, 3) else x.reshape(-1, x.shape[-1])
    assert q.shape == tuple(want.shape)
    H.check(mx4.dequantize(q), M.values(want) if want.numel() else want.double(), torch.zeros(want.shape, device=DEV, dtype=torch.float64))


def test_layouts_and_packed_form():
    x = H.randn(9, 3 * 96, dtype=torch.bfloat16)
    plain = mx4.quantize(x[:, 96:192].contiguous())
    for t in (x[:, 96:192], x[:, 96:192].t().contiguous().t(), H.randn(9, 97, dtype=torch.bfloat16)[:, 1:].copy_(x[:, 96:192])):
        q = mx4.quantize(t)
        assert torch.equal(q.codes, plain.codes) and torch.equal(q.scales[:-16], plain.scales[:-16])
    w = H.randn(5, 16, 288, dtype=torch.float32)
    words, scales = formats.quantize_mxfp4(w)
    q = mx4.quantize(w)
    a, b = mx4.to_packed(q)
    assert torch.equal(b, scales)
    assert torch.equal(formats.dequant_mxfp4(a, b), formats.dequant_mxfp4(words, scales))
    r = mx4.from_packed(a, b)
    assert torch.equal(r.codes, q.codes) and torch.equal(r.scales[:-16], q.scales[:-16])
    b[0, 0, 0] = 0   # reads as 0 in the packed form
    r = mx4.dequantize(mx4.from_packed(a, b), torch.float32)
    assert torch.equal(r, formats.dequant_mxfp4(a, b))


# ------------------------------------------------------------------------------------------------------ products
SIZES = [(1, 8, 32), (1, 200, 1056), (2, 1024, 4096), (4, 264, 96), (5, 1024, 544), (16, 136, 2880), (17, 136, 288), (32, 264, 1056), (24, 8200, 96), (33, 2056, 160),
         (65, 520, 352), (130, 264, 1440), (237, 2048, 2816), (700, 136, 96), (1000, 1032, 224), (2048, 2048, 64), (513, 4104, 160),
         (300, 512, 8192), (3, 64, 20480), (2049, 4104, 288)]


def linear_reference(xv, wv, b, r, act):
    K = xv.shape[-1]
    z = xv @ wv.T
    mags = xv.abs() @ wv.abs().T
    if b is not None:
        z, mags = z + b.double(), mags + b.double().abs()
    y = act_of(act, z)
    tol = act_tol(act, z, (K + 8) * 2.0 ** -23 * mags)
    if r is not None:
        y, tol = y + r.double(), tol + 2.0 ** -23 * (y.abs() + r.double().abs())
    return z, mags, y, tol


@pytest.mark.parametrize("act", [NONE, SILU, GELU])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,N,K", SIZES)
def test_linear(T, N, K, dtype, act):
    x = activations(T, K, dtype)
    w, wv = M.random_mx4(1, N, K)
    w, wv = M.first(w), wv[0]
    b, r = H.randn(N, dtype=dtype, seed=2), H.randn(T, N, dtype=dtype, seed=3)
    xv = M.values(x)
    for bias, res in ((b, r), (None, None)):
        _, _, y, tol = linear_reference(xv, wv, bias, res, act)
        got = mx4.linear(x, w, bias=bias, act=act, residual=res)
        H.check(got, y, tol + H.half_step(dtype) * y.abs() + H.tiny(dtype))
        out = mx4.linear(x, w, bias=bias, act=act, residual=res, out_dtype=torch.float32)
        H.check(out, y, tol + 2.0 ** -23 * y.abs())
        if bias is not None:   # from x's form, and from 16-bit weights
            out = mx4.linear(mx4.quantize(x), w, bias=bias, act=act, residual=res, out_dtype=torch.float32)
            H.check(out, y, tol + 2.0 ** -23 * y.abs())


def test_linear_quantises_weights():
    x, w = activations(40, 160, torch.bfloat16), H.randn(72, 160, dtype=torch.bfloat16)
    assert torch.equal(mx4.linear(x, w), mx4.linear(x, mx4.quantize(w)))


@pytest.mark.parametrize("act", [NONE, SILU, GELU])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T,N,K", [(1, 64, 96), (5, 96, 160), (65, 544, 352), (300, 1056, 224), (1024, 1024, 64), (130, 72, 1056)])
def test_linear_gradients(T, N, K, dtype, act):
    """At the MXFP4 values of both operands; as for linear.linear, z may land on the other side of a border of its 16 bits."""
    x, w = activations(T, K, dtype), H.randn(N, K, dtype=dtype, scale=K ** -0.5, seed=1)
    b, r = H.randn(N, dtype=dtype, seed=2), H.randn(T, N, dtype=dtype, seed=3)
    dy = H.randn(T, N, dtype=dtype, seed=4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y = mx4.linear(leaves[0], leaves[1], bias=leaves[2], act=act, residual=leaves[3])
    plain = mx4.linear(x, w, bias=b, act=act, residual=r)
    xv, wv = M.values(x), M.values(w)
    z, mags, ref, tol = linear_reference(xv, wv, b, r, act)
    H.check(y.detach(), ref, tol + H.half_step(dtype) * ref.abs() + H.tiny(dtype))
    H.check(plain, ref, tol + H.half_step(dtype) * ref.abs() + H.tiny(dtype))
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dr, dy)
    if act == NONE:
        dz, dz_tol = dy.double(), torch.zeros_like(z)
    else:
        step = 2 * H.half_step(dtype) * z.abs() + 2 * H.tiny(dtype) + (K + 8) * 2.0 ** -23 * mags
        kept = z.to(dtype).double().requires_grad_()
        (slope,) = torch.autograd.grad(act_of(act, kept).sum(), kept)
        dz = dy.double() * slope
        dz_tol = dy.double().abs() * (step + 2.0 ** -17) + H.half_step(dtype) * dz.abs() + H.tiny(dtype)
    # the values in fp16: those below its normal range are rounded (at most half of its smallest step)
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for got, ref, tol, m, R in (
            (dx, dz @ wv, dz_tol @ wv.abs() + (dz.abs() + dz_tol).sum(1, keepdim=True) * sub, dz.abs() @ wv.abs(), N),
            (dw, dz.T @ xv, dz_tol.T @ xv.abs() + (dz.abs() + dz_tol).sum(0)[:, None] * sub, dz.abs().T @ xv.abs(), T),
            (db, dz.sum(0), dz_tol.sum(0), dz.abs().sum(0), T)):
        ref = ref.detach()
        H.check(got, ref, (tol * (1 + H.half_step(dtype)) + H.product_tol(ref, m, R, dtype)).detach())


def test_gradient_against_differences():
    """Along steps of E2M1 numbers that stay in one binade the quantisation is the identity, so differences of the product itself
    are the gradient's: x of whole numbers 0 .. 4 in blocks whose largest is 4, moved by 1/2 where its code is below 2."""
    T, N, K = 6, 40, 96
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, 4, (T, K), generator=g).double().to(DEV)
    x[:, ::32] = 4
    v = torch.where(x < 2, 0.5, 0.0) * torch.randint(0, 2, (T, K), generator=g).to(DEV)
    w, wv = M.random_mx4(1, N, K)
    w = M.first(w)
    dy = H.randn(T, N, dtype=torch.bfloat16, seed=4)
    f = lambda t: mx4.linear(t.to(torch.bfloat16), w, out_dtype=torch.float32).double()   # noqa: E731
    xr = x.to(torch.bfloat16).requires_grad_()
    (dx,) = torch.autograd.grad(mx4.linear(xr, w), xr, dy)
    d = float(((f(x + v) - f(x)) * dy.double()).sum())
    dx64 = dy.double() @ wv[0]
    sums = float((((x + v).abs() @ wv[0].abs().T) * 2 * (K + 8) * 2.0 ** -23 * dy.double().abs()).sum())
    assert abs(d - float((dx.double() * v).sum())) <= sums + float((dx64.abs() * v).sum()) * 2.0 ** -8 + 1e-5


GROUPS = [[1], [5], [0, 3, 0], [1] * 8, [40, 0, 1, 17, 0], [0, 0, 0], [130, 64, 1, 65, 2], [33] * 20, [700, 0, 300], [256] * 9,
          [3, 1, 0, 0, 200, 0, 5, 31] * 4, [3, 0, 40, 1] * 20]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("N,K", [(8, 32), (264, 160), (1032, 1056)])
def test_grouped(counts, N, K, dtype):
    E, n = len(counts), sum(counts)
    w, wv = M.random_mx4(E, N, K)
    x = activations(n, K, dtype)
    b = H.randn(E, N, dtype=dtype, seed=2)
    off = H.offsets_of(counts)
    xv = M.values(x) if n else x.double()
    ref, mags = torch.zeros(2, n, N, dtype=torch.float64, device=DEV)
    for e, r in H.ranges(counts):
        ref[r], mags[r] = xv[r] @ wv[e].T + b[e].double(), xv[r].abs() @ wv[e].abs().T + b[e].double().abs()
    got = mx4.grouped_mm(x, w, off, bias=b)
    H.check(got, ref, H.product_tol(ref, mags, K, dtype))
    H.check(mx4.grouped_mm(x, w, off, bias=b, out_dtype=torch.float32), ref, (K + 8) * 2.0 ** -23 * mags + 2.0 ** -23 * ref.abs())
    if n:
        H.check(mx4.grouped_mm(mx4.quantize(x), w, off, bias=b), ref, H.product_tol(ref, mags, K, dtype))


@pytest.mark.parametrize("T,k,E,N,K", [(1, 8, 128, 264, 256), (3, 4, 32, 136, 2880), (40, 6, 64, 72, 96), (700, 4, 16, 264, 160),
                                       (2000, 8, 32, 520, 288)])
@pytest.mark.parametrize("form", ["16-bit", "mx4"])
def test_grouped_rows(T, k, E, N, K, form):
    """Token rows through the slot list, with indices outside x, and slots behind the last group."""
    dtype = torch.bfloat16
    g = torch.Generator().manual_seed(T)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).reshape(-1)
    order = torch.argsort(ids, stable=True)
    tail = 3
    rows = torch.cat([order // k, torch.zeros(tail, dtype=torch.int64)]).to(torch.int32).to(DEV)
    rows[0], rows[len(order) // 2] = -1, T
    off = H.offsets_of(torch.bincount(ids, minlength=E).tolist())
    x = activations(T, K, dtype)
    w, wv = M.random_mx4(E, N, K)
    xv = torch.cat([M.values(x), torch.zeros(1, K, dtype=torch.float64, device=DEV)])
    src = rows[:-tail].long()
    xs = xv[torch.where((src < 0) | (src >= T), T, src)]
    ref, mags = torch.zeros(2, T * k + tail, N, dtype=torch.float64, device=DEV)
    for e, r in H.ranges(torch.bincount(ids, minlength=E).tolist()):
        ref[r], mags[r] = xs[r] @ wv[e].T, xs[r].abs() @ wv[e].abs().T
    operand = x if form == "16-bit" else mx4.quantize(x)
    H.check(mx4.grouped_mm(operand, w, off, rows=rows), ref, H.product_tol(ref, mags, K, dtype))
    out = torch.full((T * k + tail, N), 7.0, dtype=dtype, device=DEV)
    got = mx4.grouped_mm(operand, w, off, rows=rows, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[-tail:] == 7).all()
    H.check(out[:-tail], ref[:-tail], H.product_tol(ref, mags, K, dtype)[:-tail])


@pytest.mark.parametrize("frozen", [True, False], ids=["frozen", "master"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("counts", [[1], [0, 3, 0, 70], [130, 64, 0, 65, 2], [160, 161, 500, 0, 33, 1]])
def test_grouped_gradients(counts, dtype, frozen):
    N, K, E, n = 136, 224, len(counts), sum(counts)
    x, b, dy = activations(n, K, dtype), H.randn(E, N, dtype=dtype, seed=2), H.randn(n, N, dtype=dtype, seed=4)
    if frozen:
        w, wv = M.random_mx4(E, N, K)
        leaves = [x.requires_grad_(), b.requires_grad_()]
    else:
        w = H.randn(E, N, K, dtype=dtype, scale=K ** -0.5, seed=1)
        wv = M.values(w)
        w.requires_grad_()
        leaves = [x.requires_grad_(), b.requires_grad_(), w]
    off = H.offsets_of(counts)
    grads = torch.autograd.grad(mx4.grouped_mm(x, w, off, bias=b), leaves, dy)
    xv = M.values(x.detach())
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    d = dy.double()
    for e, r in H.ranges(counts):
        ref, m = d[r] @ wv[e], d[r].abs() @ wv[e].abs()
        H.check(grads[0][r], ref, H.product_tol(ref, m, N, dtype) + d[r].abs().sum(1, keepdim=True) * sub)
        H.check(grads[1][e], d[r].sum(0), H.product_tol(d[r].sum(0), d[r].abs().sum(0), n, dtype))
        if not frozen:
            ref, m = d[r].T @ xv[r], d[r].abs().T @ xv[r].abs()
            H.check(grads[2][e], ref, H.product_tol(ref, m, n, dtype) + d[r].abs().sum(0)[:, None] * sub)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("counts,tail,N", [([0], 5, 8), ([1, 0, 7], 2, 264), ([8, 9, 63, 64, 65, 129], 0, 520), ([0, 5000, 0], 3, 136),
                                           ([1500] * 3, 0, 1024), ([3] * 1024, 1, 8)],
                         ids=["empty", "few", "pieces of 8 rows", "one group has all", "shared by workgroups", "1024 groups"])
def test_bias_gradients_beside_frozen_weights(counts, tail, N, dtype):
    """Rows behind the last group (of NaN here) count for no bias, groups without rows get zeros."""
    E, n, K = len(counts), sum(counts) + tail, 32
    w, _ = M.random_mx4(E, N, K)
    b = H.randn(E, N, dtype=dtype).requires_grad_()
    dy = H.randn(n, N, dtype=dtype, seed=4)
    dy[sum(counts):] = math.nan
    y = mx4.grouped_mm(activations(n, K, dtype), w, H.offsets_of(counts), bias=b)
    (db,) = torch.autograd.grad(y, b, dy)
    ref = torch.zeros((E, N), dtype=torch.float64, device=DEV)
    mags = torch.zeros_like(ref)
    for e, r in H.ranges(counts):
        ref[e], mags[e] = dy[r].double().sum(0), dy[r].double().abs().sum(0)
    H.check(db, ref, H.product_tol(ref, mags, n, dtype))


@pytest.mark.parametrize("T,N", [(0, 64), (1, 8), (100, 2056), (4097, 512)])
def test_linear_bias_gradient_beside_frozen_weights(T, N):
    w = M.first(M.random_mx4(1, N, 64)[0])
    b = H.randn(N, dtype=torch.bfloat16).requires_grad_()
    wide = H.randn(T, N + 24, dtype=torch.bfloat16, seed=4)
    (db,) = torch.autograd.grad(mx4.linear(activations(T, 64, torch.bfloat16), w, bias=b), b, wide[:, 8:8 + N])
    d = wide[:, 8:8 + N].double()
    H.check(db, d.sum(0), H.product_tol(d.sum(0), d.abs().sum(0), T, torch.bfloat16))


def test_grouped_weight_gradient_through_rows():
    T, N, K, E = 30, 64, 96, 4
    x, w = activations(T, K, torch.bfloat16), H.randn(E, N, K, dtype=torch.bfloat16, scale=0.1, seed=1).requires_grad_()
    rows = torch.arange(2 * T, device=DEV).flip(0).to(torch.int32) // 2
    off = H.offsets_of([20, 0, 25, 15])
    dy = H.randn(2 * T, N, dtype=torch.bfloat16, seed=4)
    (dw,) = torch.autograd.grad(mx4.grouped_mm(x, w, off, rows=rows), w, dy)
    xs, d = M.values(x)[rows.long()], dy.double()
    for e, r in H.ranges([20, 0, 25, 15]):
        ref, m = d[r].T @ xs[r], d[r].abs().T @ xs[r].abs()
        H.check(dw[e], ref, H.product_tol(ref, m, 2 * T, torch.bfloat16))


def test_x_that_an_index_list_cannot_address(monkeypatch):
    """Past the bytes that a list's rows can be addressed with, x is indexed first: the same results and weight gradients."""
    T, N, K, E = 30, 64, 96, 4
    x, w = activations(T, K, torch.bfloat16), H.randn(E, N, K, dtype=torch.bfloat16, scale=0.1, seed=1).requires_grad_()
    rows = (torch.arange(2 * T, device=DEV).flip(0) // 2).to(torch.int32)
    rows[3], rows[50] = -1, T
    off, dy = H.offsets_of([20, 0, 25, 15]), H.randn(2 * T, N, dtype=torch.bfloat16, seed=4)
    results = []
    for limit in (grouped.MAX_INDEXED_BYTES, T * K // 2 - 1):
        monkeypatch.setattr(grouped, "MAX_INDEXED_BYTES", limit)
        y = mx4.grouped_mm(x, w, off, rows=rows)
        results.append((y.detach(), torch.autograd.grad(y, w, dy)[0]))
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.any()


# ------------------------------------------------------------------------------------------------ values and use
def test_bad_values_stay_in_their_rows():
    """An infinity or NaN in x makes its row NaN, one in the weights its column; the others are untouched."""
    for T in (2, 16, 40, 300):
        x, w = activations(T, 288, torch.bfloat16), H.randn(264, 288, dtype=torch.bfloat16, scale=0.1, seed=1)
        good = mx4.linear(x, w)
        assert torch.isfinite(good).all()
        x2, w2 = x.clone(), w.clone()
        x2[1, 200], w2[5, 287], w2[263, 3] = math.inf, math.nan, -math.inf
        y = mx4.linear(x2, w2)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[1] = bad[:, 5] = bad[:, 263] = True
        assert torch.isnan(y[bad]).all(), T
        assert torch.equal(y[~bad], good[~bad]), T


def test_wide_range():
    """Rows at the ends of the exponents' range: scales of 2^-126 .. 2^125 on either side."""
    for ex, ew in ((-120, 100), (100, -120), (60, 60), (-60, -60)):
        for T in (3, 100):
            x = (H.randn(T, 64, dtype=torch.float32) * 2.0 ** ex).to(torch.bfloat16)
            w = (H.randn(16, 64, dtype=torch.float32, seed=1) * 2.0 ** ew).to(torch.bfloat16)
            xv, wv = M.values(x), M.values(w)
            ref = xv @ wv.T
            if float(ref.abs().max()) < 1e38:
                H.check(mx4.linear(x, w, out_dtype=torch.float32), ref, 80 * 2.0 ** -23 * (xv.abs() @ wv.abs().T) + 2.0 ** -126)


def test_empty_and_batched():
    w = mx4.quantize(H.randn(64, 96, dtype=torch.bfloat16))
    assert mx4.linear(torch.empty(0, 96, dtype=torch.bfloat16, device=DEV), w).shape == (0, 64)
    x = H.randn(2, 3, 5, 96, dtype=torch.bfloat16).requires_grad_()
    y = mx4.linear(x, w)
    assert y.shape == (2, 3, 5, 64)
    y.sum().backward()
    assert x.grad.shape == x.shape
    x = H.randn(64, 30, dtype=torch.bfloat16).t()
    assert torch.equal(mx4.linear(x, mx4.quantize(H.randn(8, 64, dtype=torch.bfloat16))),
                       mx4.linear(x.contiguous(), mx4.quantize(H.randn(8, 64, dtype=torch.bfloat16))))
    z = torch.zeros(0, 96, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(mx4.linear(z, w).sum(), z)
    assert g.shape == z.shape


def test_captured_calls():
    """A captured product, forward and backward, replayed on new inputs between other work equals the eager call each time."""
    dtype = torch.bfloat16
    for T in (1, 9, 300):
        w, _ = M.random_mx4(1, 264, 288)
        w = M.first(w)
        x, dy = activations(T, 288, dtype), H.randn(T, 264, dtype=dtype)
        xr = x.clone().requires_grad_()

        def step():
            y = mx4.linear(xr, w, act=SILU)
            return y.detach(), torch.autograd.grad(y, xr, dy)[0]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for seed in range(3):
            with torch.no_grad():
                xr.copy_(activations(T, 288, dtype, seed=seed))
            graph.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in got]
            for a, b in zip(kept, step()):
                assert torch.equal(a, b)


def test_other_stream_and_repeat():
    """The same call gives the same bits, also on a stream of its own."""
    for T in (4, 16, 100, 600):
        x, w = activations(T, 2880, torch.bfloat16), M.first(M.random_mx4(1, 520, 2880)[0])
        first = mx4.linear(x, w)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = mx4.linear(x, w)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(first, again)


def test_two_streams_at_once():
    """Calls of every path on two streams, each with its own operands, equal the ones made one after the other."""
    w, _ = M.random_mx4(6, 520, 288)
    dense = [M.first(mx4.Mx4(w.codes[e:e + 1], M.random_mx4(1, 520, 288, seed=e)[0].scales)) for e in (0, 1)]
    counts = ([3, 0, 40, 1, 9, 47], [0, 100, 0, 0, 0, 0])
    xs = [activations(100, 288, torch.bfloat16, seed=s) for s in (0, 1)]
    dy = [H.randn(100, 520, dtype=torch.bfloat16, seed=s) for s in (2, 3)]
    offs = [H.offsets_of(c) for c in counts]

    def calls(i):
        x = xs[i]
        return [mx4.linear(x[:1], dense[i]), mx4.linear(x[:20], dense[i], act=GELU), mx4.linear(x, dense[i]),
                mx4.grouped_mm(x, w, offs[i]), M.linear_dx(dy[i], dense[i]), mx4._grouped_dx(dy[i], w, offs[i]),
                mx4._bias_grad(dy[i], offs[i], 6)]
    want = [calls(0), calls(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


@pytest.mark.parametrize("act", [NONE, SILU])
def test_each_gradient_alone(act):
    """Any one of the operands that can have a gradient, the others without: equal to it among all of them, and no more kept."""
    T, N, K = 70, 136, 96
    x, w, b = activations(T, K, torch.bfloat16), H.randn(N, K, dtype=torch.bfloat16, scale=0.1, seed=1), H.randn(N, dtype=torch.bfloat16)
    r, dy = H.randn(T, N, dtype=torch.bfloat16, seed=2), H.randn(T, N, dtype=torch.bfloat16, seed=3)
    kept = []

    def pack(t):
        kept.append(t.numel() * t.element_size())
        return t

    def grads(needs):
        kept.clear()
        leaves = [t.clone().requires_grad_(i in needs) for i, t in enumerate((x, w, b, r))]
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = mx4.linear(*leaves[:2], bias=leaves[2], act=act, residual=leaves[3])
        return torch.autograd.grad(y, [leaves[i] for i in needs], dy), sum(kept)
    every, _ = grads([0, 1, 2, 3])
    z = T * N * 2 if act != NONE else 0
    form = lambda rows: rows * K // 2 + rows * 8 + 16
    for i, keeps in enumerate((z + form(N), z + form(T), z, 0)):
        (g,), n = grads([i])
        assert torch.equal(g, every[i]) or i == 2   # (the bias's sums have another order beside the weights' gradient)
        assert n == keeps, (i, n, keeps)
    E, off = 2, H.offsets_of([30, 40])
    w, b = H.randn(E, N, K, dtype=torch.bfloat16, scale=0.1, seed=1), H.randn(E, N, dtype=torch.bfloat16)

    def grouped_grads(needs):
        leaves = [t.clone().requires_grad_(i in needs) for i, t in enumerate((x, w, b))]
        y = mx4.grouped_mm(*leaves[:2], off, bias=leaves[2])
        return torch.autograd.grad(y, [leaves[i] for i in needs], dy)
    every = grouped_grads([0, 1, 2])
    for i in range(3):
        assert torch.equal(grouped_grads([i])[0], every[i]) or i == 2


def test_training_calls_without_rows():
    x = torch.zeros(0, 96, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w, b = H.randn(64, 96, dtype=torch.bfloat16).requires_grad_(), H.randn(64, dtype=torch.bfloat16).requires_grad_()
    for g, t in zip(torch.autograd.grad(mx4.linear(x, w, bias=b, act=SILU).sum(), (x, w, b)), (x, w, b)):
        assert g.shape == t.shape and not g.any()
    w, b = H.randn(3, 64, 96, dtype=torch.bfloat16).requires_grad_(), H.randn(3, 64, dtype=torch.bfloat16).requires_grad_()
    for g, t in zip(torch.autograd.grad(mx4.grouped_mm(x, w, H.offsets_of([0, 0, 0]), bias=b).sum(), (x, w, b)), (x, w, b)):
        assert g.shape == t.shape and not g.any()


def test_routed_layer_of_the_operators():
    """Router, grouping, both products of an expert layer and its GLU, as a program would run them, against 64 bits with the
    intermediate rows rounded where the calls round them."""
    from moelab_amd import act8, router
    T, E, k, d, F = 50, 16, 4, 128, 96
    dtype = torch.bfloat16
    x, wr = activations(T, d, dtype), H.randn(E, d, dtype=dtype, scale=d ** -0.5, seed=7)
    idx, wts = router.route_scored(x, wr, k, score="sigmoid", bias=H.randn(E, dtype=torch.float32, scale=0.05), groups=4,
                                   top_groups=2, group_score="top2")
    counts, offsets, srt, _, _ = router.group(idx, E)
    (gu, guv), (dn, dnv) = M.random_mx4(E, 2 * F, d), M.random_mx4(E, d, F, seed=1)
    tokens = torch.div(srt, k, rounding_mode="floor").to(torch.int32)
    h, _, _ = act8.glu_forward(mx4.grouped_mm(x, gu, offsets, rows=tokens))
    ys = mx4.grouped_mm(h, dn, offsets, out_dtype=torch.float32)
    hv = M.values(h)
    for e, r in H.ranges(counts.tolist()):
        m = M.values(x)[tokens[r].long()]
        z = m @ guv[e].T
        ref = H.silu(z[:, :F]) * z[:, F:]
        # z rounded to 16 bits, then h: a step of either, through slopes of at most 1.1 |u| and |g|
        tol = 2.0 ** -7 * (ref.abs() + 1.2 * z[:, :F].abs() * z[:, F:].abs()) + 2.0 ** -20 * (m.abs() @ guv[e].abs().T).amax(1, keepdim=True) ** 2
        H.check(h[r], ref, tol)
        H.check(ys[r], hv[r] @ dnv[e].T, (F + 9) * 2.0 ** -23 * (hv[r].abs() @ dnv[e].abs().T))
    y = torch.zeros(T, d, device=DEV).index_add_(0, tokens.long(), ys * wts.reshape(-1)[srt.long()][:, None])
    assert torch.isfinite(y).all()
