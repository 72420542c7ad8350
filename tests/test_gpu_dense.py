"""The expert layer on 16-bit weights (dense.experts_mlp, glu_mlp): forward and gradients against 64-bit arithmetic, odd routings,
captured training steps, and transformers' blocks trained through the patch."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import act8, dense, grouped, patch, router

pytestmark = pytest.mark.gpu

# T, k, E, d, F, act
CASES = [(1, 1, 1, 64, 32, 0), (1, 4, 8, 128, 96, 0), (5, 3, 16, 136, 64, 1), (33, 2, 4, 72, 160, 2), (70, 8, 64, 64, 96, 0),
         (150, 2, 3, 264, 128, 0)]


def make(T, k, E, d, F, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + T)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32).to(DEV)
    return (H.randn(T, d, dtype=dtype, seed=seed), idx, torch.softmax(H.randn(T, k, dtype=torch.float32, seed=seed + 1), 1),
            H.randn(E, 2 * F, d, dtype=dtype, scale=d ** -0.5, seed=seed + 2), H.randn(E, d, F, dtype=dtype, scale=F ** -0.5, seed=seed + 3),
            H.randn(T, d, dtype=dtype, seed=seed + 4))


def rel(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


def roundings(dtype, n):
    """2-norm of n independent roundings, each at most half a step of its value (so at most sqrt(n) half steps together, in the
    mean; twice that is allowed for), and the fp32 sums."""
    return 2 * n ** 0.5 * H.half_step(dtype) + 1e-5


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,k,E,d,F,act", CASES)
def test_forward(T, k, E, d, F, act, dtype):
    x, idx, wts, wgu, wd, r = make(T, k, E, d, F, dtype)
    for res in (None, r):
        ref = H.experts(x.double(), idx, wts.double(), wgu.double(), wd.double(), act, None if res is None else res.double())
        y = dense.experts_mlp(x, idx, wts, wgu, wd, act=act, residual=res)
        # gate/up rows (two factors), h, the slots' rows, the result
        assert rel(y, ref) <= roundings(dtype, 5)
        y32 = dense.experts_mlp(x, idx, wts, wgu, wd, act=act, residual=res, out_dtype=torch.float32)
        assert torch.equal(y32.to(dtype), y)
    assert torch.equal(dense.experts_mlp(x, idx.long(), wts, wgu, wd, act=act, residual=r), y)


@pytest.mark.parametrize("checkpoint", [True, False], ids=["8bit", "16bit"])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,k,E,d,F,act", CASES)
def test_gradients(T, k, E, d, F, act, dtype, checkpoint):
    x, idx, wts, wgu, wd, r = make(T, k, E, d, F, dtype)
    dy = H.randn(T, d, dtype=dtype, seed=9)
    leaves = [t.clone().requires_grad_() for t in (x, wts, wgu, wd, r)]
    y = dense.experts_mlp(leaves[0], idx, leaves[1], leaves[2], leaves[3], act=act, residual=leaves[4], checkpoint=checkpoint)
    assert torch.equal(y, dense.experts_mlp(x, idx, wts, wgu, wd, act=act, residual=r))
    got = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(got[4], dy) and got[1].dtype == wts.dtype

    def kept(t, j, gu):   # the values that the backward pass reads, with the gradient passed straight through
        v = gu.to(dtype)
        v = H.values(*H.quantise(v[None]))[0] if checkpoint else v.double()
        return gu + (v - gu).detach()
    refs = [t.double().requires_grad_() for t in (x, wts, wgu, wd)]
    want = torch.autograd.grad(H.experts(refs[0], idx, refs[1], refs[2], refs[3], act, kept=kept), refs, dy.double())
    # dx: gate/up gradients, the slots' rows, the result; weights: one operand and the result. Sums that the 8-bit form rounds
    # to the other side of a border move one value by a step (1/64 of its block's largest) at 1 in 10^3 elements: 2^-6 / 30
    flip = 2e-3 if checkpoint else 0.0
    for name, g, ref, n in zip(("dx", "dwts", "dw_gate_up", "dw_down"), got, want, (3, 1, 2, 2)):
        assert rel(g, ref) <= roundings(dtype, n) + flip, name


def test_slots_without_an_expert():
    """Ids outside [0, E) add nothing and have no gradient; a token with none of its slots left is its residual alone; experts
    without slots get zero gradients; the same expert twice for one token counts twice."""
    T, k, E, d, F = 40, 3, 6, 72, 64
    x, idx, wts, wgu, wd, r = make(T, k, E, d, F, torch.bfloat16)
    idx[:, 2] = torch.where(idx[:, 2] == 5, 0, idx[:, 2])
    idx = torch.where(idx == 5, 1, idx)
    idx[3], idx[7, 1], idx[9, 0] = -1, E, -2 ** 31
    idx[11] = 4
    keep = (idx >= 0) & (idx < E)
    leaves = [t.clone().requires_grad_() for t in (x, wts, wgu, wd)]
    y = dense.experts_mlp(leaves[0], idx, leaves[1], leaves[2], leaves[3], residual=r)
    ref = H.experts(x.double(), idx, wts.double(), wgu.double(), wd.double(), 0, r.double())
    assert rel(y, ref) <= roundings(torch.bfloat16, 5) and torch.equal(y[3], r[3])
    dx, dw, dgu, ddn = torch.autograd.grad(y, leaves, H.randn(T, d, dtype=torch.bfloat16, seed=9))
    assert not dx[3].any() and not dw[~keep].any() and dw[keep].all() and not dgu[5].any() and not ddn[5].any()
    assert all(torch.isfinite(t).all() for t in (dx, dw, dgu, ddn))
    none = torch.full_like(idx, -1)
    y = dense.experts_mlp(leaves[0], none, leaves[1], leaves[2], leaves[3])
    assert not y.any()
    assert all(not g.any() for g in torch.autograd.grad(y, leaves, torch.ones_like(y)))


def test_padded_rows_of_non_finite_values():
    """A token whose slots all have no expert may hold anything."""
    x, idx, wts, wgu, wd, _ = make(20, 2, 4, 64, 64, torch.bfloat16)
    idx[5], x[5] = -1, float("nan")
    leaves = [t.clone().requires_grad_() for t in (x, wts, wgu, wd)]
    y = dense.experts_mlp(*[leaves[0], idx, *leaves[1:]])
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert torch.isfinite(y).all() and all(torch.isfinite(g).all() for g in grads)


def test_parts_one_by_one_are_the_whole():
    """The call is the run of its parts: group, gate/up products through the slot list, GLU, down products; and a token's slots
    in any order are the same sum but for its rounding."""
    T, k, E, d, F = 90, 4, 12, 136, 96
    x, idx, wts, wgu, wd, _ = make(T, k, E, d, F, torch.float16)
    counts, offsets, order, _, _ = router.group(idx, E)
    rows = torch.div(order, k, rounding_mode="floor").to(torch.int32)
    h, codes, scales = act8.glu_forward(grouped.mm(x, wgu, offsets, rows=rows))
    slots = torch.empty(T * k, d, dtype=torch.float64, device=DEV)
    slots[order.long()] = grouped.mm(h, wd, offsets).double()
    want = (slots.view(T, k, d) * wts.double()[..., None]).sum(1)
    y = dense.experts_mlp(x, idx, wts, wgu, wd, out_dtype=torch.float32)
    assert rel(y, want) <= roundings(torch.float16, 2)
    p = torch.arange(k - 1, -1, -1, device=DEV)
    assert rel(dense.experts_mlp(x, idx[:, p], wts[:, p], wgu, wd), y.double()) <= roundings(torch.float16, 2)


def test_no_tokens():
    x, idx, wts, wgu, wd, r = make(4, 2, 4, 64, 64, torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (wgu, wd)]
    y = dense.experts_mlp(x[:0], idx[:0], wts[:0], *leaves, residual=r[:0])
    assert y.shape == (0, 64)
    assert all(g.shape == t.shape and not g.any() for g, t in zip(torch.autograd.grad(y.sum(), leaves), leaves))


def test_streams_in_parallel():
    """Calls on several streams at once, forward and backward, share nothing."""
    args = [make(60, 4, 8, 136, 96, torch.bfloat16, seed=s) for s in range(4)]

    def step(a):
        leaves = [t.clone().requires_grad_() for t in (a[0], a[2], a[3], a[4])]
        y = dense.experts_mlp(leaves[0], a[1], *leaves[1:], residual=a[5])
        return (y.detach(), *torch.autograd.grad(y, leaves, a[5]))
    want = [step(a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = []
    for a, s in zip(args, streams):
        with torch.cuda.stream(s):
            got.append(step(a))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for w, g in zip(want, got) for p, q in zip(w, g))


@pytest.mark.parametrize("T", [1, 30, 400])
def test_captured_training_steps(T):
    """Two graphs of a step, replayed in turn with new tokens, routings and eager steps between."""
    sets = [make(T, 2, 8, 136, 96, torch.bfloat16, seed=s) for s in (0, 50)]
    leaves = [[t.requires_grad_() for t in (a[0], a[2], a[3], a[4])] for a in sets]

    def step(i):
        x, w, gu, dn = leaves[i]
        y = dense.experts_mlp(x, sets[i][1], w, gu, dn, residual=sets[i][5])
        return (y.detach(), *torch.autograd.grad(y, leaves[i], sets[i][5]))
    s = torch.cuda.Stream()
    graphs, outs = [], []
    for i in range(2):
        with torch.cuda.stream(s):
            step(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(step(i))
        graphs.append(graph)
    for n in range(3):
        for i in range(2):
            with torch.no_grad():
                sets[i][0].copy_(H.randn(T, 136, dtype=torch.bfloat16, seed=20 + n))
                sets[i][1].copy_(make(T, 2, 8, 136, 96, torch.bfloat16, seed=30 + n)[1])
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(p, q) for p, q in zip(outs[i], step(i)))


def test_past_32_bit_offsets():
    """Slots' gate/up rows of 4.3 GB: 2^31 values, checked on tokens at the ends and around the borders."""
    T, k, E, d, F = 70_000, 8, 16, 64, 1920
    g = torch.Generator(device=DEV).manual_seed(0)
    idx = torch.rand(T, E, generator=g, device=DEV).topk(k, 1)[1].to(torch.int32)
    x, _, _, wgu, wd, _ = make(8, k, E, d, F, torch.bfloat16)
    x = H.randn(T, d, dtype=torch.bfloat16)
    wts = torch.softmax(torch.randn(T, k, generator=g, device=DEV), 1)
    leaves = [t.requires_grad_() for t in (x, wts)]
    y = dense.experts_mlp(leaves[0], idx, leaves[1], wgu, wd)
    some = torch.tensor([0, 1, T // 2, T - 2, T - 1], device=DEV)
    dy = H.randn(T, d, dtype=torch.bfloat16, seed=1)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    a = [x.detach()[some].double().requires_grad_(), wts.detach()[some].double().requires_grad_()]
    ref = H.experts(a[0], idx[some], a[1], wgu.double(), wd.double(), 0)
    assert rel(y.detach()[some], ref.detach()) <= roundings(torch.bfloat16, 5)
    # 8-bit rows: a rounding of at most 1/127 of a block's largest, about 2% of a value in the mean square, on either factor
    for got, want in zip((dx, dw), torch.autograd.grad(ref, a, dy[some].double())):
        assert rel(got[some], want) <= 0.03


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("T", [1, 50])
def test_glu_mlp(T, act):
    d, F = 136, 96
    dt = torch.bfloat16
    x, r = H.randn(T, d, dtype=dt), H.randn(T, d, dtype=dt, seed=1)
    w = [H.randn(F, d, dtype=dt, scale=d ** -0.5, seed=2), H.randn(F, d, dtype=dt, scale=d ** -0.5, seed=3), H.randn(d, F, dtype=dt, scale=F ** -0.5, seed=4)]
    leaves = [t.clone().requires_grad_() for t in (x, *w, r)]
    y = dense.glu_mlp(*leaves[:4], act=act, residual=leaves[4])
    refs = [t.double().requires_grad_() for t in (x, *w, r)]
    ref = H.glu(act, refs[0] @ refs[1].T, refs[0] @ refs[2].T) @ refs[3].T + refs[4]
    assert rel(y.detach(), ref.detach()) <= roundings(dt, 4)
    dy = H.randn(T, d, dtype=dt, seed=5)
    for g, want, n in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(ref, refs, dy.double()), (6, 5, 5, 5, 1)):
        assert rel(g, want) <= roundings(dt, n)
