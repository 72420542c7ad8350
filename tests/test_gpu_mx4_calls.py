"""Calls of the MXFP4 products that their documentation allows beside the plain ones: more rows of x than slots, offsets as a view, sums
whose square is past fp32, slots behind the last group in the gradients, values outside fp16's range, one busy group among many of few
slots, captured calls."""
import math

import pytest
import torch

import dense_helpers as H
import mx4_helpers as M
from dense_helpers import DEV, TYPES
from moelab_amd import _lib, mx4
from moelab_amd.linear import GELU, SILU
from test_gpu_mx4 import IDS, activations, linear_reference

pytestmark = pytest.mark.gpu


def grouped_call(x, q, w, off, M_, rows=None):
    """moe_mx4_grouped_mm with as many rows of x as it has and M_ slots."""
    E, N, K = w.shape
    n = (x if q is None else q.codes).shape[0]
    y = torch.full((M_, N), 7.0, dtype=torch.bfloat16, device=DEV)
    ws, nws = mx4._workspace(y.device, "moe_mx4_grouped_mm_workspace_bytes", M_, n, E, K, int(q is not None))
    _lib.call("moe_mx4_grouped_mm", y.device, *mx4._pointers(x, q), n, w.codes.data_ptr(), w.scales.data_ptr(), None, _lib.ptr(off),
              _lib.ptr(rows), M_, E, N, K, 0, y.data_ptr(), 0, 1, _lib.ptr(ws), nws)
    return y


@pytest.mark.parametrize("form", ["16-bit", "mx4"])
@pytest.mark.parametrize("counts,N", [([1] * 8, 264), ([20, 0, 31] * 4, 136), ([300, 0, 90], 264), ([256] * 9, 1032)],
                         ids=["few rows", "64 x 64", "128 x 128", "128 x 256"])
@pytest.mark.parametrize("K", [160, 288, 1056])
def test_more_rows_than_slots(counts, N, K, form):
    """Without an index list slot p reads x's row p, however many rows follow; K past one step of exponents among them."""
    n = sum(counts)
    w, wv = M.random_mx4(len(counts), N, K)
    x = activations(n + 57, K, torch.bfloat16)
    y = grouped_call(*((x, None) if form == "16-bit" else (None, mx4.quantize(x))), w, H.offsets_of(counts), n)
    xv = M.values(x)
    for e, r in H.ranges(counts):
        ref, mags = xv[r] @ wv[e].T, xv[r].abs() @ wv[e].abs().T
        H.check(y[r], ref, H.product_tol(ref, mags, K, torch.bfloat16), (e, r))


@pytest.mark.parametrize("act", [SILU, GELU])
@pytest.mark.parametrize("T", [3, 17, 40, 300, 2048])
def test_sums_whose_square_overflows(T, act):
    """Activations of sums past 2^64, on every path: themselves, or zero on the negative side."""
    N, K = 264, 64
    x = (activations(T, K, torch.float32) * 2.0 ** 40).to(torch.bfloat16)
    w = (H.randn(N, K, dtype=torch.float32, seed=1) * 2.0 ** 40).to(torch.bfloat16)
    b, r = H.randn(N, dtype=torch.bfloat16, seed=2), H.randn(T, N, dtype=torch.bfloat16, seed=3)
    z, _, y, tol = linear_reference(M.values(x), M.values(w), b, r, act)
    assert float(z.abs().max()) > 2.0 ** 64
    for dtype in (torch.bfloat16, torch.float32):
        step = H.half_step(torch.bfloat16) if dtype == torch.bfloat16 else 2.0 ** -23
        H.check(mx4.linear(x, w, bias=b, act=act, residual=r, out_dtype=dtype), y, tol + step * y.abs())


@pytest.mark.parametrize("counts", [[9, 0, 30, 1], [200, 130, 0, 161]])
def test_offsets_with_a_stride(counts):
    """Offsets as a column of a table of counts: the forward pass and every gradient read the view, not what lies behind its first."""
    E, N, K, n = len(counts), 136, 224, sum(counts)
    plain = H.offsets_of(counts)
    view = torch.stack([plain, torch.full_like(plain, n)], 1)[:, 0]
    assert not view.is_contiguous()
    x, dy = activations(n, K, torch.bfloat16), H.randn(n, N, dtype=torch.bfloat16, seed=4)
    b = H.randn(E, N, dtype=torch.bfloat16, seed=2)
    frozen, _ = M.random_mx4(E, N, K)
    for w in (frozen, H.randn(E, N, K, dtype=torch.bfloat16, scale=K ** -0.5, seed=1)):
        got = []
        for off in (plain, view):
            leaves = [t.clone().requires_grad_() for t in ((x, b) if w is frozen else (x, b, w))]
            y = mx4.grouped_mm(leaves[0], w if w is frozen else leaves[2], off, bias=leaves[1])
            got.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
        for i, (p, q) in enumerate(zip(*got)):
            assert torch.equal(p, q), i


def wide_weights(E, N, K):
    """Weights of positive values in blocks of three kinds: some past fp16's largest number, fp16's own, and some below its smallest."""
    q, _ = M.random_mx4(E, N, K)
    codes, _ = mx4.to_packed(q)
    codes &= 0x77777777
    kinds = torch.tensor([127 + 15, 127, 127 - 25], device=DEV).repeat(K // 96)
    q = mx4.from_packed(codes, kinds.to(torch.uint8).expand(E, N, -1).contiguous())
    v = mx4.dequantize(q, torch.float32).double()
    assert float(v.max()) > 65520 and 0 < float(v[v > 0].min()) < 2.0 ** -24
    return q, v


@pytest.mark.parametrize("T", [3, 130, 4100])
def test_gradients_in_fp16_through_weights_outside_its_range(T):
    """The weights' values are rounded to fp16 there: infinity past its largest, what fp16 has below its smallest. The forward
    product takes them as they are."""
    N, K = 72, 288
    w, v = wide_weights(1, N, K)
    x, dy = activations(T, K, torch.float16), H.randn(T, N, dtype=torch.float16, seed=4).abs() + 0.25
    v16 = v[0].half().double()
    with torch.no_grad():
        x[:, (torch.arange(K, device=DEV) // 32) % 3 == 0] *= 2.0 ** -14
    x = x.requires_grad_()
    y = mx4.linear(x, M.first(w))
    xv = M.values(x.detach())
    ref = xv @ v[0].T
    assert torch.isfinite(y).all()
    H.check(y.detach(), ref, H.product_tol(ref, xv.abs() @ v[0].T, K, torch.float16))
    (dx,) = torch.autograd.grad(y, x, dy)
    ref = dy.double() @ v16
    assert torch.isinf(ref).any() and torch.isfinite(ref).any()
    H.check(dx, ref, H.product_tol(ref, ref, N, torch.float16))


@pytest.mark.parametrize("counts", [[9, 0, 30], [200, 130, 0, 161]])
def test_grouped_gradients_in_fp16_through_weights_outside_its_range(counts):
    E, N, K, n = len(counts), 72, 288, sum(counts)
    w, v = wide_weights(E, N, K)
    v16 = v.half().double()
    x, dy = activations(n, K, torch.float16).requires_grad_(), H.randn(n, N, dtype=torch.float16, seed=4).abs() + 0.25
    (dx,) = torch.autograd.grad(mx4.grouped_mm(x, w, H.offsets_of(counts), out_dtype=torch.float32), x, dy.float())
    for e, r in H.ranges(counts):
        ref = dy[r].double() @ v16[e]
        H.check(dx[r], ref, H.product_tol(ref, ref, N, torch.float16))


def test_gradients_through_weights_with_bad_blocks():
    """Blocks with an infinity or NaN read as NaN: their columns of dx are NaN, no others."""
    for T, N, K in ((3, 72, 288), (300, 72, 288), (4100, 64, 96)):
        w = H.randn(N, K, dtype=torch.bfloat16, scale=0.1, seed=1)
        w[5, K - 1], w[N - 1, 3] = math.nan, -math.inf
        x, dy = activations(T, K, torch.bfloat16).requires_grad_(), H.randn(T, N, dtype=torch.bfloat16, seed=4)
        (dx,) = torch.autograd.grad(mx4.linear(x, mx4.quantize(w)), x, dy)
        v = M.values(w)
        bad = torch.isnan(v).any(0)
        assert torch.isnan(dx[:, bad]).all() and int(bad.sum()) == 64
        v = torch.where(torch.isnan(v), 0, v)
        ref = dy.double() @ v
        H.check(dx[:, ~bad], ref[:, ~bad], H.product_tol(ref, dy.double().abs() @ v.abs(), N, torch.bfloat16)[:, ~bad])


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("counts", [[0, 0], [9, 0, 30, 1], [200, 130, 0, 161], [40, 0, 1000]])
def test_gradients_of_slots_behind_the_last_group(counts, out):
    """Their rows of dy (NaN here) are not read. dx is zero there in the backward pass; the library call leaves them as they were
    with fill = 0. Tiles of both heights."""
    E, N, K, n, tail = len(counts), 136, 288, sum(counts), 7
    w, wv = M.random_mx4(E, N, K)
    off, dy = H.offsets_of(counts), H.randn(n + tail, N, dtype=torch.bfloat16, seed=4)
    dy[n:] = math.nan
    x = activations(n + tail, K, torch.bfloat16).requires_grad_()
    (g,) = torch.autograd.grad(mx4.grouped_mm(x, w, off), x, dy)
    ref, mags = torch.zeros(2, n + tail, K, dtype=torch.float64, device=DEV)
    for e, r in H.ranges(counts):
        ref[r], mags[r] = dy[r].double() @ wv[e], dy[r].double().abs() @ wv[e].abs()
    H.check(g, ref, H.product_tol(ref, mags, N, torch.bfloat16))
    for fill in (0, 1):
        dx = torch.full((n + tail, K), 7.0, dtype=out, device=DEV)
        _lib.call("moe_mx4_grouped_mm_dx", dx.device, dy.data_ptr(), dy.stride(0), w.codes.data_ptr(), w.scales.data_ptr(), off.data_ptr(),
                  n + tail, E, N, K, 0, dx.data_ptr(), _lib.DTYPE[out], fill)
        assert (dx[n:] == (0 if fill else 7)).all()
        step = H.half_step(torch.bfloat16) if out == torch.bfloat16 else 2.0 ** -23
        H.check(dx[:n], ref[:n], step * ref[:n].abs() + (N + 8) * 2.0 ** -23 * mags[:n])


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("form", ["16-bit", "mx4"])
@pytest.mark.parametrize("counts,tail", [([0] * 40 + [90] + [0] * 40, 5), ([1] * 30 + [47] + [0, 2] * 20 + [17, 5], 0), ([130] + [0] * 127, 3)])
def test_few_slots_a_group_but_one_busy(counts, tail, form, bias):
    """About one slot a group on average, most of them in one: the kernel of few rows goes through it piece by piece."""
    E, n, N, K = len(counts), sum(counts), 200, 544
    assert (n + tail) // min(E, n + tail) <= 1
    w, wv = M.random_mx4(E, N, K)
    x, b = activations(n + tail, K, torch.bfloat16), H.randn(E, N, dtype=torch.bfloat16, seed=2) if bias else None
    xv = M.values(x)
    ref, mags = torch.zeros(2, n + tail, N, dtype=torch.float64, device=DEV)
    for e, r in H.ranges(counts):
        c = b[e].double() if bias else torch.zeros(N, dtype=torch.float64, device=DEV)
        ref[r], mags[r] = xv[r] @ wv[e].T + c, xv[r].abs() @ wv[e].abs().T + c.abs()
    off, operand = H.offsets_of(counts), x if form == "16-bit" else mx4.quantize(x)
    H.check(mx4.grouped_mm(operand, w, off, bias=b), ref, H.product_tol(ref, mags, K, torch.bfloat16))
    back = torch.arange(n + tail, device=DEV).flip(0).to(torch.int32)
    flipped = x.flip(0) if form == "16-bit" else mx4.quantize(x.flip(0))
    H.check(mx4.grouped_mm(flipped, w, off, bias=b, rows=back), ref, H.product_tol(ref, mags, K, torch.bfloat16))


@pytest.mark.parametrize("M_", [6, 200, 900])
def test_captured_grouped_calls(M_):
    """A captured product and its gradients, replayed on other offsets and rows between eager calls, equal the eager ones each time."""
    E, N, K = 6, 264, 288
    w, _ = M.random_mx4(E, N, K)
    b = H.randn(E, N, dtype=torch.bfloat16, seed=2).requires_grad_()
    x = activations(M_, K, torch.bfloat16).requires_grad_()
    dy, off = H.randn(M_, N, dtype=torch.bfloat16, seed=4), torch.zeros(E + 1, dtype=torch.int32, device=DEV)

    def step():
        y = mx4.grouped_mm(x, w, off, bias=b)
        return (y.detach(), *torch.autograd.grad(y, (x, b), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    g = torch.Generator().manual_seed(M_)
    for case in range(5):
        cuts = torch.randint(0, M_ + 1, (E,), generator=g).sort().values
        cuts = [torch.full((E,), M_), torch.cat([torch.zeros(E - 1), torch.tensor([M_])]), torch.zeros(E)][case] if case < 3 else cuts
        with torch.no_grad():
            off[1:] = cuts.to(DEV, torch.int32)
            x.copy_(activations(M_, K, torch.bfloat16, seed=case))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for p, q in zip(kept, step()):
            assert torch.equal(p, q), case
