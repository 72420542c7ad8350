"""linear.linear and its gradients against 64-bit arithmetic: sizes on every path (dot products of few rows, the three tiles), odd
ones, every epilogue, z kept in 16 and in 8 bits, batches of more dimensions, layouts, captured calls."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import act8, linear
from moelab_amd.linear import GELU, NONE, SILU

pytestmark = pytest.mark.gpu
SIZES = [(1, 8, 8), (1, 200, 1032), (3, 264, 72), (4, 1024, 520), (7, 2056, 136), (33, 136, 264), (65, 520, 328), (237, 264, 1416),
         (700, 136, 72), (1000, 1032, 200), (2048, 2048, 64), (513, 4104, 136)]


def act_of(act, z):
    return {NONE: lambda t: t, SILU: H.silu, GELU: H.gelu}[act](z)


def z_tol(z, mags, K):
    return (K + 8) * 2.0 ** -23 * mags


def act_tol(act, z, dz):
    """What an error dz in z does to act(z) (slope at most 1.13), and act's own fp32 evaluation."""
    if act == NONE:
        return dz
    big = 1.6 * (z.abs() + 0.045 * z.abs() ** 3) if act == GELU else z.abs()
    return 1.13 * dz + (5 * big.clamp(max=200) + 16) * 2.0 ** -23 * act_of(act, z).abs() + 1e-37


def make(T, N, K, dtype, bias=True, residual=True):
    x, w = H.randn(T, K, dtype=dtype), H.randn(N, K, dtype=dtype, scale=K ** -0.5, seed=1)
    return x, w, H.randn(N, dtype=dtype, seed=2) if bias else None, H.randn(T, N, dtype=dtype, seed=3) if residual else None


def reference(x, w, b, r, act):
    z = x.double() @ w.double().T
    mags = x.double().abs() @ w.double().abs().T
    if b is not None:
        z, mags = z + b.double(), mags + b.double().abs()
    y = act_of(act, z)
    tol = act_tol(act, z, z_tol(z, mags, x.shape[1]))
    if r is not None:
        y, tol = y + r.double(), tol + 2.0 ** -23 * (y.abs() + r.double().abs())
    return z, mags, y, tol


@pytest.mark.parametrize("act", [NONE, SILU, GELU])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K", SIZES)
def test_forward(T, N, K, dtype, act):
    for bias, residual in ((True, True), (False, False)):
        x, w, b, r = make(T, N, K, dtype, bias, residual)
        _, _, y, tol = reference(x, w, b, r, act)
        H.check(linear.linear(x, w, bias=b, act=act, residual=r), y, tol + H.half_step(dtype) * y.abs() + H.tiny(dtype))
        out = linear.linear(x, w, bias=b, act=act, residual=r, out_dtype=torch.float32)
        assert out.dtype == torch.float32
        H.check(out, y, tol + 2.0 ** -23 * y.abs())


@pytest.mark.parametrize("checkpoint", [False, True], ids=["z16", "z8"])
@pytest.mark.parametrize("act", [NONE, SILU, GELU])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K", [(1, 64, 72), (5, 96, 136), (65, 544, 328), (300, 1056, 200), (2048, 2048, 64)])
def test_gradients(T, N, K, dtype, act, checkpoint):
    """From z as it is kept (its rounding is exactly reproduced up to the fp32 sums that it rounds), dz rounded once to the
    operands' type, then products. A sum next to a border of z's rounding can land on its other side; that moves dz by the
    slope's change over one step, which the bound counts for every element."""
    x, w, b, r = make(T, N, K, dtype)
    dy = H.randn(T, N, dtype=dtype, seed=4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y = linear.linear(leaves[0], leaves[1], bias=leaves[2], act=act, residual=leaves[3], checkpoint=checkpoint)
    assert torch.equal(y, linear.linear(x, w, bias=b, act=act, residual=r))
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dr, dy)
    z, mags, _, _ = reference(x, w, b, None, act)
    if act == NONE:
        dz, dz_tol = dy.double(), torch.zeros_like(z)
    else:
        kept, step = z.to(dtype).double(), 2 * H.half_step(dtype) * z.abs() + 2 * H.tiny(dtype) + z_tol(z, mags, K)
        if checkpoint:
            codes, scales = H.quantise(z.to(dtype))
            kept = H.values(codes, scales)
            step = step + (2.0 ** (scales.double() - 132)).repeat_interleave(32, 1)
        kept = kept.requires_grad_()
        (slope,) = torch.autograd.grad(act_of(act, kept).sum(), kept)
        dz = dy.double() * slope
        # |act''| <= 1 (SiLU 0.5, tanh-GELU 0.8); slope in fp32: sums of terms below 2 with a relative error of 2^-18
        dz_tol = dy.double().abs() * (step + 2.0 ** -17) + H.half_step(dtype) * dz.abs() + H.tiny(dtype)
    for got, ref, tol, m, R in (
            (dx, dz @ w.double(), dz_tol @ w.double().abs(), dz.abs() @ w.double().abs(), N),
            (dw, dz.T @ x.double(), dz_tol.T @ x.double().abs(), dz.abs().T @ x.double().abs(), T),
            (db, dz.sum(0), dz_tol.sum(0), dz.abs().sum(0), T)):
        ref = ref.detach()
        H.check(got, ref, (tol * (1 + H.half_step(dtype)) + H.product_tol(ref, m, R, dtype)).detach())


def test_gradient_against_differences():
    """Central differences of the forward pass in fp32 along one direction, against the gradient: the truncation error of the
    same differences in 64 bits, the sums' roundings over the step, and the gradient's own two roundings to bf16."""
    T, N, K, eps = 9, 64, 72, 2.0 ** -3
    x, w, b, _ = make(T, N, K, torch.bfloat16, residual=False)
    x = torch.round(x.float() * 16).div(16).clamp(-3, 3).to(torch.bfloat16)   # x +- eps are bf16 numbers
    v = torch.randint(-1, 2, (T, K), generator=torch.Generator().manual_seed(0)).to(DEV).double()
    dy = H.randn(T, N, dtype=torch.bfloat16, seed=4)
    up, dn = (x.double() + eps * v), (x.double() - eps * v)
    assert torch.equal(up.to(torch.bfloat16).double(), up) and torch.equal(dn.to(torch.bfloat16).double(), dn)
    f = lambda t: linear.linear(t.to(torch.bfloat16), w, bias=b, act=GELU, out_dtype=torch.float32).double()   # noqa: E731
    f64 = lambda t: H.gelu(t @ w.double().T + b.double())   # noqa: E731
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(linear.linear(xr, w, bias=b, act=GELU), xr, dy)
    x64 = x.double().requires_grad_()
    (dx64,) = torch.autograd.grad(f64(x64), x64, dy.double())
    d, d64 = (float(((g(up) - g(dn)) * dy.double()).sum()) / (2 * eps) for g in (f, f64))
    truncation = abs(d64 - float((dx64 * v).sum()))
    _, mags, _, tol = reference(x, w, b, None, GELU)
    sums = float(((2 * tol + 2.0 ** -23 * mags) * dy.double().abs()).sum()) / eps
    grad = float((dx64.abs() * v.abs()).sum()) * 2.0 ** -9 + float((dy.double().abs() @ w.double().abs() * v.abs()).sum()) * 3 * 2.0 ** -9
    assert abs(d - float((dx.double() * v).sum())) <= truncation + sums + grad


def test_only_what_is_asked_for():
    x, w, b, r = make(20, 64, 72, torch.bfloat16)
    dy = H.randn(20, 64, dtype=torch.bfloat16, seed=4)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(linear.linear(full[0], full[1], full[2], SILU, full[3]), full, dy)
    for i in range(4):
        args = [x, w, b, r]
        args[i] = args[i].clone().requires_grad_()
        (g,) = torch.autograd.grad(linear.linear(args[0], args[1], args[2], SILU, args[3]), args[i], dy)
        assert torch.equal(g, want[i]), i


def test_batches_layouts_and_shared_leaves():
    x, w, b, r = make(30, 64, 72, torch.float16)
    y = linear.linear(x, w, b, SILU, r)
    assert torch.equal(linear.linear(x.view(2, 3, 5, 72), w, b, SILU, r.view(2, 3, 5, 64)), y.view(2, 3, 5, 64))
    assert torch.equal(linear.linear(x[0], w, b, SILU, r[0]).view(1, 64), linear.linear(x[:1], w, b, SILU, r[:1]))
    wide = torch.cat([x, x], 1)
    assert torch.equal(linear.linear(wide[:, 72:], w, b, SILU, r), y)
    assert torch.equal(linear.linear(x, w.T.contiguous().T, b, SILU, r.T.contiguous().T), y)
    assert linear.linear(x[:0], w, b, SILU, r[:0]).shape == (0, 64)
    # the same leaf twice in a graph, a broadcast residual and a broadcast gradient
    leaf, res = w.clone().requires_grad_(), H.randn(64, dtype=torch.float16).requires_grad_()
    out = linear.linear(x, leaf, b, SILU, res.expand(30, 64)) + linear.linear(x, leaf, b, SILU)
    out.sum().backward()
    ones = torch.ones(30, 64, dtype=torch.float16, device=DEV)
    one = w.clone().requires_grad_()
    (g,) = torch.autograd.grad(linear.linear(x, one, b, SILU), one, ones)
    assert torch.equal(leaf.grad, g + g) and (res.grad == 30).all()
    empty = w.clone().requires_grad_()
    linear.linear(x[:0], empty, b, SILU).sum().backward()
    assert not empty.grad.any()


def test_act_backward_from_codes():
    z, dy = H.randn(37, 96, dtype=torch.bfloat16, scale=3.0), H.randn(37, 96, dtype=torch.bfloat16, seed=1)
    codes, scales = act8.pack(z)
    for act in (SILU, GELU):
        v = act8.unpack(codes, scales, torch.bfloat16)
        assert torch.equal(linear.act_backward(dy, None, act, codes, scales), linear.act_backward(dy, v, act))


@pytest.mark.parametrize("T", [1, 40, 700])
def test_captured_step(T):
    """Forward and backward in a graph, replayed with new inputs and eager calls between."""
    x, w, b, r = make(T, 264, 136, torch.bfloat16)
    dy = H.randn(T, 264, dtype=torch.bfloat16, seed=4)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def fn():
        y = linear.linear(*leaves, act=GELU, residual=r)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = fn()
    for i in range(3):
        with torch.no_grad():
            x.copy_(H.randn(T, 136, dtype=torch.bfloat16, seed=10 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, fn()))
