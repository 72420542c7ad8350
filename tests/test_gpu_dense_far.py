"""Weight gradients of the expert layer and of grouped.mm_dw where one operand is read through a list and the other, in slot
order, is larger than 32 bits address: between 3 and 4 GiB, and past 4 GiB, against 64-bit sums over an expert's slots."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV
from moelab_amd import dense, grouped
from test_gpu_dense import rel, roundings
from test_gpu_product_shapes import GROUPS

pytestmark = pytest.mark.gpu


# T, k, F: gate/up gradients of 3.2 GiB; of 4.0 GiB; of 8.1 GiB beside weighted h of 4.1 GiB
@pytest.mark.parametrize("T,k,F", [(60_000, 8, 1792), (70_000, 8, 1920), (280_000, 2, 3904)])
def test_weight_gradients(T, k, F):
    E, d, dt = 16, 64, torch.bfloat16
    idx = torch.rand(T, E, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV).topk(k, 1)[1].to(torch.int32)
    wts = torch.softmax(H.randn(T, k, dtype=torch.float32, seed=1), 1)
    x, dy = H.randn(T, d, dtype=dt), H.randn(T, d, dtype=dt, seed=2)
    wgu, wd = H.randn(E, 2 * F, d, dtype=dt, scale=d ** -0.5, seed=3), H.randn(E, d, F, dtype=dt, scale=F ** -0.5, seed=4)
    leaves = [t.requires_grad_() for t in (wgu, wd)]
    y = dense.experts_mlp(x, idx, wts, wgu, wd, checkpoint=False)
    dgu, ddn = torch.autograd.grad(y, leaves, dy)
    for e in (0, E - 1):
        t, j = (idx == e).nonzero(as_tuple=True)
        w = wts[t, j].double()[:, None]
        gu = (x[t].double() @ wgu[e].detach().double().T).to(dt).double().requires_grad_()   # as kept, in 16 bits
        h = H.glu(0, gu[:, :F], gu[:, F:]) * w
        (ref,) = torch.autograd.grad(h, gu, dy[t].double() @ wd[e].detach().double())
        # either sum's operand and its result are rounded
        assert rel(dgu[e], ref.T @ x[t].double()) <= roundings(dt, 2), f"dw_gate_up of expert {e}"
        assert rel(ddn[e], dy[t].double().T @ h.detach()) <= roundings(dt, 2), f"dw_down of expert {e}"


@pytest.mark.parametrize("far", ["dy", "x"])
def test_a_list_beside_a_far_operand(far):
    """The listed operand is gathered first."""
    M, wide, T, dt = 600_000, 4096, 1000, torch.bfloat16
    big = torch.empty(M, wide, dtype=dt, device=DEV)
    for i in range(0, M, 100_000):
        big[i:i + 100_000] = H.randn(100_000, wide, dtype=dt, seed=i)
    small = H.randn(T, 8, dtype=dt, seed=1)
    rows = torch.randint(0, T, (M,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).int()
    counts = [300_000, 0, 299_000, 1000]
    off = H.offsets_of(counts)
    dw = grouped.mm_dw(big, small, off, 4, x_rows=rows) if far == "dy" else grouped.mm_dw(small, big, off, 4, dy_rows=rows)
    assert not dw[1].any()
    r = slice(599_000, 600_000)
    a, b = (big[r].double(), small[rows[r].long()].double()) if far == "dy" else (small[rows[r].long()].double(), big[r].double())
    ref, mags = a.T @ b, a.abs().T @ b.abs()
    H.check(dw[3], ref, H.product_tol(ref, mags, 1000, dt))


@pytest.mark.parametrize("counts,N,K", GROUPS, ids=[f"{len(c)}x{sum(c)}-{n}-{k}" for c, n, k in GROUPS])
def test_one_list(counts, N, K):
    """One operand through a list and the other in slot order, bit for bit the product of both in slot order; rows behind the
    last group are not read."""
    E, M, dt = len(counts), sum(counts), torch.bfloat16
    rows = torch.randint(0, 97, (M,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).int()
    x, dy = H.randn(97, K, dtype=dt), H.randn(97, N, dtype=dt, seed=3)
    xs, ds = (torch.cat([t[rows.long()], torch.full((70, t.shape[1]), float("nan"), dtype=dt, device=DEV)]) for t in (x, dy))
    off, rows = H.offsets_of(counts), torch.cat([rows, torch.full((70,), 2 ** 31 - 1, dtype=torch.int32, device=DEV)])
    want = grouped.mm_dw(ds, xs, off, E, bias=True)
    for a, ar, b, br in ((dy, rows, xs, None), (ds, None, x, rows)):
        assert all(torch.equal(p, q) for p, q in zip(grouped.mm_dw(a, b, off, E, dy_rows=ar, x_rows=br, bias=True), want))
