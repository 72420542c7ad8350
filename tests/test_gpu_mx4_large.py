"""MXFP4 operands and routing past 32-bit offsets: the last rows and the last expert of tensors of more than 2^32 elements or bytes
equal those of small calls."""
import pytest
import torch

import dense_helpers as H
import mx4_helpers as M
from dense_helpers import DEV
from moelab_amd import mx4, router

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_quantise():
    rows, K, n = (1 << 20) + 13, 4128, 70
    x = torch.zeros((rows, K), dtype=BF, device=DEV)
    x[-n:] = H.randn(n, K, dtype=BF)
    q, small = mx4.quantize(x), mx4.quantize(x[-n:])
    assert torch.equal(q.codes[-n:], small.codes)
    v = mx4.dequantize(q)
    assert torch.equal(v[-n:], mx4.dequantize(small)) and not v[:1000].any() and not v[rows // 2:rows // 2 + 1000].any()


def weights(E, N, K):
    codes = torch.randint(0, 256, (E, N, K // 2), device=DEV, dtype=torch.uint8, generator=torch.Generator(device=DEV).manual_seed(1))
    scales = torch.full((8 * E * N * -(-K // 256) + 16,), 121, dtype=torch.uint8, device=DEV)
    return mx4.Mx4(codes, scales)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_last_expert_of_many(n):
    E, N, K = 66, 16392, 8192
    w = weights(E, N, K)
    last = M.first(mx4.Mx4(w.codes[-1:], w.scales[:8 * N * (K // 256) + 16]))
    wv = mx4.dequantize(last, torch.float32).double()
    counts = [0] * (E - 2) + [2, n]
    x = H.randn(n + 2, K, dtype=BF).requires_grad_()
    dy = H.randn(n + 2, N, dtype=BF, seed=3)
    y = mx4.grouped_mm(x, w, H.offsets_of(counts))
    xv = M.values(x.detach())[2:]
    H.check(y[2:].detach(), xv @ wv.T, H.product_tol(xv @ wv.T, xv.abs() @ wv.T.abs(), K, BF))
    (dx,) = torch.autograd.grad(y, x, dy)
    d = dy[2:].double()
    H.check(dx[2:], d @ wv, H.product_tol(d @ wv, d.abs() @ wv.abs(), N, BF))


def test_last_rows_of_many():
    T, N, K, n = 140003, 16384, 64, 77
    w = weights(1, N, K)
    w = M.first(w)
    x = torch.zeros((T, K), dtype=BF, device=DEV)
    x[-n:] = H.randn(n, K, dtype=BF)
    xv, wv = M.values(x[-n:]), mx4.dequantize(w, torch.float32).double()
    y = mx4.linear(x, w)
    H.check(y[-n:], xv @ wv.T, H.product_tol(xv @ wv.T, xv.abs() @ wv.T.abs(), K, BF))
    assert not y[:5000].any() and not y[T // 2:T // 2 + 5000].any()
    y[-n:] = H.randn(n, N, dtype=BF, seed=5)   # zeros but for the last rows: dy
    d = y[-n:].double()
    for dx in (M.linear_dx(y, w), mx4._grouped_dx(y, mx4.Mx4(w.codes[None], w.scales), H.offsets_of([T]))):
        H.check(dx[-n:], d @ wv, H.product_tol(d @ wv, d.abs() @ wv.abs(), N, BF))
        assert not dx[:-n].any()
    H.check(mx4._bias_grad(y, None, 1)[0], d.sum(0), H.product_tol(d.sum(0), d.abs().sum(0), T, BF))


def test_route():
    T, E, k, n = (1 << 22) + 9, 520, 4, 50
    lg = torch.zeros((T, E), dtype=BF, device=DEV)
    lg[-n:] = H.randn(n, E, dtype=BF)
    kw = dict(score="softmax", norm=False, groups=4, top_groups=2)
    small = lg[-n:].clone().requires_grad_()
    lg.requires_grad_()
    si, sw = router.topk_scored(small, k, **kw)
    idx, wts = router.topk_scored(lg, k, **kw)
    assert torch.equal(idx[-n:], si) and torch.equal(wts[-n:], sw)
    assert (idx[T // 2:T // 2 + 1000] == torch.arange(k, device=DEV)).all()
    dw = torch.zeros_like(wts)
    dw[-n:] = torch.rand(n, k, generator=torch.Generator().manual_seed(1)).to(DEV)
    (dl,) = torch.autograd.grad(wts, lg, dw)
    (ds,) = torch.autograd.grad(sw, small, dw[-n:])
    assert torch.equal(dl[-n:], ds) and not dl[:1000].any()
