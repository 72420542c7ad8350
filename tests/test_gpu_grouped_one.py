"""One group of all slots (offsets None) in the grouped products, rows in slot order and through lists, from one slot to several
rounds of tiles, and the same with the group's offsets given; calls at once from two threads."""
import threading

import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import grouped

pytestmark = pytest.mark.gpu
SIZES = [(1, 8, 8), (3, 264, 72), (5, 72, 4104), (64, 200, 328), (700, 520, 136), (5000, 72, 264), (4200, 1032, 520)]


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_one_group(M, N, K, dtype):
    T = max(1, M // 2)
    x, w, dy = (H.randn(*s, dtype=dtype, seed=i) for i, s in enumerate(((T, K), (1, N, K), (T, N))))
    b = H.randn(1, N, dtype=dtype, seed=4)
    rows = torch.randint(-1, T + 1, (M,), generator=torch.Generator(device=DEV).manual_seed(M), device=DEV).int()
    ok = (rows >= 0) & (rows < T)
    xs, ds = (torch.where(ok[:, None], t[torch.where(ok, rows, 0).long()], 0) for t in (x, dy))
    off = H.offsets_of([M])
    X, W, D = xs.double(), w[0].double(), ds.double()
    for o in (None, off):
        for got, ref, mags, R in (
                (grouped.mm(x, w, o, bias=b, rows=rows), X @ W.T + b.double(), X.abs() @ W.abs().T + b.double().abs(), K),
                (grouped.mm(xs, w, o, bias=b), X @ W.T + b.double(), X.abs() @ W.abs().T + b.double().abs(), K),
                (grouped.mm_dx(dy, w, o, rows=rows), D @ W, D.abs() @ W.abs(), N),
                (grouped.mm_dx(ds, w, o), D @ W, D.abs() @ W.abs(), N),
                (grouped.mm_dw(dy, x, o, 1, dy_rows=rows, x_rows=rows)[0], D.T @ X, D.abs().T @ X.abs(), M),
                (grouped.mm_dw(ds, x, o, 1, x_rows=rows)[0], D.T @ X, D.abs().T @ X.abs(), M),
                (grouped.mm_dw(dy, xs, o, 1, dy_rows=rows)[0], D.T @ X, D.abs().T @ X.abs(), M),
                (grouped.mm_dw(ds, xs, o, 1, bias=True)[1][0], D.sum(0), D.abs().sum(0), M)):
            H.check(got, ref, H.product_tol(ref, mags, R, dtype))


def test_two_threads():
    """Calls and gradients of two threads on streams of their own."""
    from moelab_amd import dense, linear
    x, w = H.randn(300, 136, dtype=torch.bfloat16), H.randn(4, 200, 136, dtype=torch.bfloat16, seed=1)
    off = H.offsets_of([100, 0, 150, 50])
    idx = torch.arange(600, device=DEV).view(300, 2).remainder(4).int()
    wts = torch.full((300, 2), 0.5, device=DEV)
    gu, dn = H.randn(4, 128, 136, dtype=torch.bfloat16, seed=2, scale=0.1), H.randn(4, 136, 64, dtype=torch.bfloat16, seed=3, scale=0.1)

    def step():
        leaves = [t.clone().requires_grad_() for t in (x, w, gu, dn)]
        y = (grouped.mm(leaves[0], leaves[1], off), linear.linear(leaves[0], leaves[1][0], act=linear.SILU),
             dense.experts_mlp(leaves[0], idx, wts, leaves[2], leaves[3]))
        return [t.detach() for t in y], torch.autograd.grad([t.float().sum() for t in y], leaves)
    want, got = step(), [None, None]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = step()
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g in got:
        assert all(torch.equal(p, q) for a, b in zip(g, want) for p, q in zip(a, b))
