"""The expert layer element by element, against 64-bit arithmetic that rounds where the documentation says it does and nowhere else:
h, the gate/up gradients and w h to 16 bits, each result once. So a rounding that comes back into the slots' rows or into the GLU's
input shows.

A value that is rounded inside the call comes from fp32 sums, and next to a border between two 16-bit numbers it can land on the
other side. `rounded` says for each value what that may cost: a step where the border is within the fp32 error, else nothing."""
import ctypes

import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import _lib, act8, dense
from test_gpu_dense import make

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -23

# T, k, E, d, F, act: dot products of single slots; 64-row tiles; 128-row tiles of few experts and of uneven ones; 128 x 256
# tiles with rounds and rests; 300 and 1024 experts; the smallest d; more slots a token than are summed at once
SIZES = [(1, 4, 8, 128, 96, 0), (5, 3, 16, 136, 64, 1), (33, 2, 4, 72, 160, 2), (150, 2, 3, 264, 128, 0), (600, 4, 8, 136, 96, 1),
         (900, 4, 12, 264, 544, 0), (2100, 2, 16, 72, 800, 2), (1500, 8, 64, 136, 160, 0), (40, 8, 300, 72, 64, 1), (3, 8, 1024, 64, 32, 0),
         (700, 8, 1024, 64, 64, 0), (7, 1, 1, 8, 32, 1), (60, 13, 24, 72, 64, 0), (9, 40, 48, 8, 96, 1)]
IDS = ["-".join(map(str, s)) for s in SIZES]


def rounded(v, err, dtype):
    """v to 16 bits, and per element a step where fp32 errors of err can carry it over a border."""
    r = v.to(dtype).double()
    near = torch.maximum((v + err).to(dtype).double(), (v - err).to(dtype).double()) != torch.minimum(
        (v + err).to(dtype).double(), (v - err).to(dtype).double())
    return r, torch.where(near, 2 * H.half_step(dtype) * v.abs() + 2 * H.tiny(dtype) + err, 0.0)


def slope(act, g, u):
    """h of [n, F] halves and its derivatives, in 64 bits."""
    g, u = g.detach().requires_grad_(), u.detach().requires_grad_()
    h = H.glu(act, g, u)
    dg, du = torch.autograd.grad(h.sum(), (g, u))
    return h.detach(), dg, du


def glu_err(act, g, u):
    """fp32 evaluation of the GLU and its derivatives: sigmoid off by (5 |z| + 16) 2^-23 of itself, beside terms of the size of u,
    g and their product."""
    z = {0: g.abs(), 1: 1.6 * (g.abs() + 0.045 * g.abs() ** 3), 2: 1.702 * g.abs()}[act].clamp(max=200)
    return (5 * z + 24) * EPS, (1 + z) * (1 + u.abs())


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,k,E,d,F,act", SIZES, ids=IDS)
def test_forward(T, k, E, d, F, act, dtype):
    """In fp32: only h is rounded. And what each form of the call keeps: the slots' gate/up sums rounded once, and their 8-bit form."""
    x, idx, wts, wgu, wd, r = make(T, k, E, d, F, dtype)
    y = dense.experts_mlp(x, idx, wts, wgu, wd, act=act, residual=r, out_dtype=torch.float32)
    ref, tol = r.double(), EPS * r.double().abs()
    y16, (_, _, gu, _, _) = dense._forward(x, idx, wts, wgu, wd, act, r, None, "16")
    _, (_, _, _, codes, scales) = dense._forward(x, idx, wts, wgu, wd, act, r, None, "8")
    assert torch.equal(y16, dense.experts_mlp(x, idx, wts, wgu, wd, act=act, residual=r)) or k * T <= 2 * E   # other kernels
    order = torch.sort(idx.reshape(-1).long(), stable=True)[1]
    at = torch.empty_like(order)
    at[order] = torch.arange(T * k, device=DEV)
    kept = gu[at].view(T, k, 2 * F)
    pc, ps = act8.pack(gu)
    assert torch.equal(codes, pc) and torch.equal(scales, ps)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        z = x[t].double() @ wgu[e].double().T
        mags = x[t].double().abs() @ wgu[e].double().abs().T
        H.check(kept[t, j], z, H.product_tol(z, mags, d, dtype), "gate/up rows")
        g, u = z[:, :F], z[:, F:]
        h, dg, du = slope(act, g, u)
        err, size = glu_err(act, g, u)
        zerr = (d + 8) * EPS * mags
        herr = dg.abs() * zerr[:, :F] + du.abs() * zerr[:, F:] + err * h.abs() + EPS * size * zerr.amax(1, keepdim=True) + 2.0 ** -118
        h16, step = rounded(h, herr, dtype)
        w, wa = wts[t, j].double()[:, None], wd[e].double().abs().T
        ref = ref.index_put((t,), w * (h16 @ wd[e].double().T), accumulate=True)
        tol = tol.index_put((t,), w.abs() * (step @ wa + (F + k + 8) * EPS * (h16.abs() @ wa)), accumulate=True)
    tol = tol + (k + 2) * EPS * ref.abs()
    H.check(y, ref, tol, "y")
    H.check(y16, ref, tol + H.half_step(dtype) * ref.abs() + H.tiny(dtype), "y in 16 bits")


@pytest.mark.parametrize("checkpoint", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,k,E,d,F,act", SIZES, ids=IDS)
def test_gradients(T, k, E, d, F, act, dtype, checkpoint):
    """From the kept gate/up rows themselves: their gradients and w h are rounded once, and each result."""
    x, idx, wts, wgu, wd, _ = make(T, k, E, d, F, dtype)
    dy = H.randn(T, d, dtype=dtype, seed=9)
    _, (_, _, gu, codes, scales) = dense._forward(x, idx, wts, wgu, wd, act, None, None, "8" if checkpoint else "16")
    gu = H.values(codes, scales) if checkpoint else gu.double()
    leaves = [t.requires_grad_() for t in (x, wts, wgu, wd)]
    y = dense.experts_mlp(leaves[0], idx, *leaves[1:], act=act, checkpoint=checkpoint)
    dx, dwts, dwgu, dwd = torch.autograd.grad(y, leaves, dy)
    x, wts, wgu, wd = (t.detach() for t in leaves)
    order = torch.sort(idx.reshape(-1).long(), stable=True)[1]
    at = torch.empty_like(order)
    at[order] = torch.arange(T * k, device=DEV)
    kept = gu[at].view(T, k, 2 * F)
    half = H.half_step(dtype)
    rx, tx = torch.zeros(T, d, dtype=torch.float64, device=DEV), torch.zeros(T, d, dtype=torch.float64, device=DEV)
    rw, tw = torch.zeros(T, k, dtype=torch.float64, device=DEV), torch.zeros(T, k, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not len(t):
            assert not dwgu[e].any() and not dwd[e].any()
            continue
        n = len(t)
        g, u = kept[t, j][:, :F], kept[t, j][:, F:]
        h, dg, du = slope(act, g, u)
        err, size = glu_err(act, g, u)
        w, dyt, xt = wts[t, j].double()[:, None], dy[t].double(), x[t].double()
        dh, dherr = dyt @ wd[e].double(), (d + 8) * EPS * (dyt.abs() @ wd[e].double().abs())
        s = torch.cat([dg, du], 1)
        serr = (err * size).repeat(1, 2)
        dgu = w * dh.repeat(1, 2) * s
        dguerr = w.abs() * (dherr.repeat(1, 2) * (s.abs() + serr) + dh.abs().repeat(1, 2) * serr) + 4 * EPS * dgu.abs() + 2.0 ** -118
        dgu16, step = rounded(dgu, dguerr, dtype)
        wa = wgu[e].double()
        rx.index_put_((t,), dgu16 @ wa, accumulate=True)
        tx.index_put_((t,), step @ wa.abs() + (2 * F + k + 8) * EPS * (dgu16.abs() @ wa.abs()), accumulate=True)
        rw[t, j] = (dh * h).sum(1)
        tw[t, j] = (dherr * h.abs() + dh.abs() * (err * size + EPS * h.abs())).sum(1) + (F + 8) * EPS * (dh * h).abs().sum(1)
        ref = dgu16.T @ xt
        H.check(dwgu[e], ref, half * ref.abs() + step.T @ xt.abs() + (n + 8) * EPS * (dgu16.abs().T @ xt.abs()) + H.tiny(dtype), f"dw_gate_up {e}")
        hw, step = rounded(w * h, w.abs() * err * size + 4 * EPS * (w * h).abs() + 2.0 ** -118, dtype)
        ref = dyt.T @ hw
        H.check(dwd[e], ref, half * ref.abs() + dyt.abs().T @ step + (n + 8) * EPS * (dyt.abs().T @ hw.abs()) + H.tiny(dtype), f"dw_down {e}")
    H.check(dx, rx, tx + (half + (k + 2) * EPS) * rx.abs() + H.tiny(dtype), "dx")
    H.check(dwts, rw, tw + 2.0 ** -24 * rw.abs(), "dwts")


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_the_result_may_be_the_residual(dtype):
    """moe_mlp_fwd and moe_linear with y the residual's own memory, as their header allows."""
    T, k, E, d, F = 300, 2, 4, 136, 96
    x, idx, wts, wgu, wd, r = make(T, k, E, d, F, dtype)
    L, dt = _lib.lib(), _lib.DTYPE[dtype]
    want = dense.experts_mlp(x, idx, wts, wgu, wd, residual=r)
    m = _lib.Mlp(E, d, F, 0, dt, wgu.data_ptr(), wd.data_ptr())
    buf = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in (L.moe_mlp_keep_bytes(m, T, k), L.moe_mlp_fwd_workspace_bytes(m, T, k))]
    y = r.clone()
    _lib.call("moe_mlp_fwd", y.device, ctypes.byref(m), x.data_ptr(), idx.data_ptr(), wts.data_ptr(), T, k, y.data_ptr(), y.data_ptr(), dt,
              buf[0].data_ptr(), None, None, None, buf[1].data_ptr(), buf[1].numel())
    assert torch.equal(y, want)
    from moelab_amd import linear
    for T, N, K in ((3, 264, 72), (64, 1032, 2056), (700, 136, 72), (2048, 1032, 264)):   # dot products, parts, tiles
        x, w, r = H.randn(T, K, dtype=dtype), H.randn(N, K, dtype=dtype, scale=K ** -0.5, seed=1), H.randn(T, N, dtype=dtype, seed=2)
        for act in (linear.NONE, linear.GELU):
            y, n = r.clone(), L.moe_linear_workspace_bytes(T, N, K)
            ws = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
            _lib.call("moe_linear", y.device, x.data_ptr(), w.data_ptr(), None, y.data_ptr(), act, T, K, N, K, dt, y.data_ptr(), dt, None,
                      ws.data_ptr(), n)
            assert torch.equal(y, linear.linear(x, w, act=act, residual=r)), (T, N, K, act)
