"""The 8-bit form of activations and the GLU on it (act8), against its definition in 64 bits."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import act8

pytestmark = pytest.mark.gpu
SIZES = [(1, 32), (3, 96), (7, 768), (130, 1440), (33, 2048), (257, 64)]


def rows(M, C, dtype, seed=0):
    """Rows of very different size, zero blocks and blocks of one value among them."""
    x = H.randn(M, C, dtype=torch.float32, seed=seed)
    x *= torch.exp2(torch.randint(-20, 12, (M, 1), generator=torch.Generator().manual_seed(seed)).float()).to(DEV)
    x[0, :32] = 0
    if M > 2:
        x[1], x[2, 32:64 if C > 32 else 32] = 1.0, 0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,C", SIZES)
def test_pack_and_unpack(M, C, dtype):
    """Codes and exponents as defined, bit for bit; unpacked exactly; every value within half a step of its block."""
    x = rows(M, C, dtype)
    codes, scales = act8.pack(x)
    want, wants = H.quantise(x)
    assert torch.equal(codes, want) and torch.equal(scales, wants)
    exact = H.values(codes, scales)
    for dt in (dtype, torch.float32):
        assert torch.equal(act8.unpack(codes, scales, dt).double(), exact)
    step = H.pow2(scales.to(torch.int64) - 133).repeat_interleave(32, 1)
    assert ((exact - x.double()).abs() <= step / 2).all()
    top = x.double().abs().reshape(M, -1, 32).amax(-1).repeat_interleave(32, 1)
    assert ((exact - x.double()).abs() <= top / 127).all()


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_pack_at_the_ends_of_the_range(dtype):
    """The largest and smallest values, the mantissas around the step to the next exponent, infinities and NaN."""
    f = torch.finfo(dtype)
    smallest = f.smallest_normal * f.eps
    x = torch.zeros(10, 64, dtype=dtype, device=DEV)
    x[0, 0], x[0, 1] = f.max, -f.max / 3
    x[1, 0], x[1, 1] = smallest, -3 * smallest
    x[2, :4] = torch.tensor([1.984375, 1.9921875, -1.9921875, 0.0078125], dtype=dtype)
    x[3, 0] = 1.984375
    x[4, 0], x[4, 40] = float("inf"), 1.0
    x[5, 33] = float("nan")
    x[6, 0] = -float("inf")
    x[7, :] = torch.linspace(-2, 2, 64, dtype=dtype)
    x[8, 0], x[8, 1] = f.smallest_normal, f.smallest_normal / 4
    x[9, :] = -f.max
    codes, scales = act8.pack(x)
    want, wants = H.quantise(x)
    assert torch.equal(codes, want) and torch.equal(scales, wants)
    v = act8.unpack(codes, scales, torch.float32)
    assert torch.isnan(v[4, :32]).all() and v[4, 40] == 1 and torch.isnan(v[5, 32:]).all() and not v[5, :32].any()
    assert torch.isnan(v[6, :32]).all() and torch.isfinite(v[[0, 1, 2, 3, 7, 8, 9]]).all()
    if dtype == torch.bfloat16:   # subnormal blocks are exact
        assert torch.equal(v[1].double(), x[1].double())


def glu_tol(act, g, u, ref, dtype):
    """One rounding, and the fp32 evaluation: sigmoid(z) through exp2 is off by z's own error (at most 4.5 |z| 2^-23, for
    tanh-GELU's polynomial and the factor log2 e) and 1 ulp each for exp2, reciprocal and the products. exp2 gives 0 below
    2^-126, so that sigmoid is off by up to 2^-126 there and h by |g u| 2^-126, with |g u| < 256 in these tests."""
    z = {0: g.abs(), 1: 1.6 * (g.abs() + 0.045 * g.abs() ** 3), 2: 1.702 * g.clamp(max=7.0).abs()}[act]
    return (H.half_step(dtype) + (5 * z.clamp(max=200) + 16) * 2.0 ** -23) * ref.abs() + H.tiny(dtype) + 2.0 ** -118


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,F", SIZES)
def test_glu_forward(M, F, dtype, act):
    gu = H.randn(M, 2 * F, dtype=dtype, scale=3.0)
    h, codes, scales = act8.glu_forward(gu, act=act)
    g, u = gu.double()[:, :F], gu.double()[:, F:]
    ref = H.glu(act, g, u)
    H.check(h, ref, glu_tol(act, g, u, ref, dtype))
    want, wants = H.quantise(gu)
    assert torch.equal(codes, want) and torch.equal(scales, wants)
    h2, c2, s2 = act8.glu_forward(gu, act=act, keep=False)
    assert torch.equal(h, h2) and c2 is None and s2 is None
    assert torch.equal(act8.pack(gu)[0], codes)
    wide = torch.cat([gu, gu], 1)[:, :2 * F]   # rows of a wider matrix
    assert torch.equal(act8.glu_forward(wide, act=act)[0], h)


def glu_reference(act, v, dh, wts):
    F = dh.shape[1]
    v = v.detach().requires_grad_()
    h = H.glu(act, v[:, :F], v[:, F:])
    w = torch.ones(dh.shape[0], 1, dtype=torch.float64, device=DEV) if wts is None else wts.double()[:, None]
    (dgu,) = torch.autograd.grad(h, v, dh.double() * w)
    return dgu, h.detach() * w, (dh.double() * h.detach()).sum(1), h.detach()


def grad_tol(act, v, dh, w, ref, dtype):
    """One rounding, and fp32: the derivative is a sum of two terms, each off as the GLU itself."""
    F = dh.shape[1]
    g, u = v[:, :F].abs(), v[:, F:].abs() + 1
    if act == 2:
        g, u = g.clamp(max=1e4), u.clamp(max=8)
    slope = {0: 1 + g, 1: 1 + 1.6 * g * (1 + 0.14 * g * g), 2: 1 + 1.702 * g}[act]
    z = {0: g, 1: 1.6 * (g + 0.045 * g ** 3), 2: 1.702 * g}[act].clamp(max=200)
    s = torch.sigmoid({0: 1.0, 1: 1.6, 2: 1.702}[act] * v[:, :F].clamp(max=7.0 if act == 2 else 1e9))
    tails = torch.cat([u * slope * torch.maximum(s * 4, torch.exp(-z).clamp(max=1)), g * torch.maximum(s, torch.exp(-z))], 1)
    mag = (dh.double() * w).abs().repeat(1, 2) * tails
    return H.half_step(dtype) * ref.abs() + (5 * z.repeat(1, 2) + 24) * 2.0 ** -23 * mag + H.tiny(dtype) + 2.0 ** -118


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("M,F", SIZES)
def test_glu_backward(M, F, dtype, act):
    gu, dh = H.randn(M, 2 * F, dtype=dtype, scale=3.0), H.randn(M, F, dtype=dtype, seed=1)
    wts = torch.rand(M, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    codes, scales = act8.pack(gu)
    v = H.values(codes, scales)
    for w in (wts, None):
        dgu, hw, dwts = act8.glu_backward(codes, scales, dh, act=act, wts=w)
        rg, rh, rw, h = glu_reference(act, v, dh, w)
        ww = torch.ones(M, 1, device=DEV, dtype=torch.float64) if w is None else w.double()[:, None]
        H.check(dgu, rg, grad_tol(act, v, dh, ww, rg, dtype), "dgu")
        H.check(hw, rh, glu_tol(act, v[:, :F], v[:, F:], rh, dtype), "hw")
        mags = (dh.double() * h).abs().sum(1)
        H.check(dwts, rw, (F + 5 * 200 + 24) * 2.0 ** -23 * mags + 1e-37, "dwts")
    # the same from the 16-bit rows, and with dh in fp32
    dgu, hw, dwts = act8.glu_backward(None, None, dh, act=act, wts=wts, gu=v.to(dtype))
    a = act8.glu_backward(codes, scales, dh, act=act, wts=wts)
    assert all(torch.equal(p, q) for p, q in zip((dgu, hw, dwts), a))
    if dtype == torch.bfloat16:
        b = act8.glu_backward(codes, scales, dh.float(), act=act, wts=wts)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_clamped_glu_has_no_gradient_where_the_clamp_holds():
    g = torch.tensor([6.5, 7.0, 7.5, 100.0, -100.0, 3.0, 3.0, 3.0], dtype=torch.bfloat16, device=DEV)
    u = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 7.5, -8.0, 7.0], dtype=torch.bfloat16, device=DEV)
    gu = torch.zeros(1, 64, dtype=torch.bfloat16, device=DEV)
    gu[0, :8], gu[0, 32:40] = g, u
    dh = torch.ones(1, 32, dtype=torch.bfloat16, device=DEV)
    dgu, _, _ = act8.glu_backward(None, None, dh, act=2, gu=gu)
    ref, _, _, _ = glu_reference(2, gu.double(), dh, None)
    H.check(dgu, ref, grad_tol(2, gu.double(), dh, 1.0, ref, torch.bfloat16))
    assert not dgu[0, 2:4].any() and not dgu[0, 37:39].any() and dgu[0, 1] != 0 and dgu[0, 39] != 0


@pytest.mark.parametrize("act", [0, 1, 2])
def test_large_and_non_finite_inputs(act):
    """Gates far out on both sides give the limits, not NaN; an infinity or NaN in a row stays in its element of h (and makes its
    block's gradients NaN)."""
    F = 64
    gu = H.randn(4, 2 * F, dtype=torch.bfloat16)
    gu[0, 0], gu[0, 1], gu[0, 2], gu[0, 3] = 1e30, -1e30, 1e4, -1e4
    gu[1, 5] = float("nan")
    gu[2, F + 5] = float("nan")
    h, codes, scales = act8.glu_forward(gu, act=act)
    ref = H.glu(act, gu.double()[:, :F], gu.double()[:, F:])
    assert torch.isfinite(h[0]).all() and abs(float(h[0, 1])) == 0 and abs(float(h[0, 3])) == 0
    H.check(h[:1, 4:], ref[:1, 4:], glu_tol(act, gu.double()[:1, 4:F], None, ref[:1, 4:], torch.bfloat16))
    assert torch.isnan(h[1, 5]) and torch.isnan(h[2, 5]) and int(torch.isnan(h).sum()) == 2
    dgu, hw, dw = act8.glu_backward(codes, scales, torch.ones(4, F, dtype=torch.bfloat16, device=DEV), act=act)
    assert torch.isfinite(dgu[0, 32:F]).all() and torch.isnan(dgu[1, :32]).all() and torch.isfinite(dgu[1, 32:F]).all()
    assert torch.isfinite(dgu[3]).all() and torch.isfinite(dw[3]) and torch.isnan(dw[1])
    dgu, _, _ = act8.glu_backward(None, None, torch.ones(4, F, dtype=torch.bfloat16, device=DEV), act=act, gu=gu)
    assert torch.isfinite(dgu[0]).all()


@pytest.mark.parametrize("checkpoint", [True, False])
def test_glu_gradient(checkpoint):
    F = 96
    gu = H.randn(9, 2 * F, dtype=torch.bfloat16, scale=2.0)
    dh = H.randn(9, F, dtype=torch.bfloat16, seed=1)
    leaf = gu.clone().requires_grad_()
    h = act8.glu(leaf, act=1, checkpoint=checkpoint)
    assert torch.equal(h, act8.glu(gu, act=1))
    (g,) = torch.autograd.grad(h, leaf, dh)
    v = H.values(*H.quantise(gu)) if checkpoint else gu.double()
    ref = glu_reference(1, v, dh, None)[0]
    H.check(g, ref, grad_tol(1, v, dh, 1.0, ref, torch.bfloat16))
    h = act8.glu(leaf, checkpoint=checkpoint)
    h.sum().backward()   # a broadcast gradient
    assert torch.isfinite(leaf.grad).all()


@pytest.mark.parametrize("act", [0, 1, 2])
def test_gradient_against_differences(act):
    """Central differences of the 64-bit function: their truncation error is its third derivative times step^2 / 6; with steps of
    2^-8 that is below 2^-16 times a few, against a gradient in bf16 (2^-9 of itself)."""
    F, eps = 32, 2.0 ** -8
    gu, dh = H.randn(5, 2 * F, dtype=torch.bfloat16), torch.ones(5, F, dtype=torch.bfloat16, device=DEV)
    dgu = act8.glu_backward(None, None, dh, act=act, gu=gu)[0].double()
    v = gu.double()
    up, dn = v.clone(), v.clone()
    up[:, :F] += eps
    dn[:, :F] -= eps
    dg = (H.glu(act, up[:, :F], v[:, F:]) - H.glu(act, dn[:, :F], v[:, F:])) / (2 * eps)
    up, dn = v.clone(), v.clone()
    up[:, F:] += eps
    dn[:, F:] -= eps
    du = (H.glu(act, v[:, :F], up[:, F:]) - H.glu(act, v[:, :F], dn[:, F:])) / (2 * eps)
    diff = torch.cat([dg, du], 1)
    third = 6 * (1 + v[:, F:].abs()).repeat(1, 2)
    H.check(dgu, diff, H.half_step(torch.bfloat16) * diff.abs() + third * eps ** 2 / 6 + 1e-6)


def test_captured():
    gu, dh = H.randn(70, 192, dtype=torch.float16), H.randn(70, 96, dtype=torch.float16, seed=1)
    def fn():
        h, c, s = act8.glu_forward(gu)
        return (h, c, s, act8.unpack(c, s, torch.float16), *act8.glu_backward(c, s, dh))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = fn()
    for i in range(3):
        gu.copy_(H.randn(70, 192, dtype=torch.float16, seed=5 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, fn()))


def test_no_rows():
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    c, s = act8.pack(e)
    assert c.shape == (0, 64) and s.shape == (0, 2) and act8.unpack(c, s).shape == (0, 64)
    h, c, s = act8.glu_forward(e)
    assert h.shape == (0, 32)
    assert act8.glu_backward(c, s, h)[0].shape == (0, 64)
