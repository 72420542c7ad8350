"""router.topk_scored and route_scored against 64-bit arithmetic: every score, bias, group and weight form, ties, masked experts,
scores that fp32 cannot tell apart, gradients, captured calls."""
import itertools
import math

import pytest
import torch

import mx4_helpers as M
from dense_helpers import DEV
from moelab_amd import linear, router

pytestmark = pytest.mark.gpu
LOGITS = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 8, 2, 1, 1), (5, 64, 6, 8, 3), (33, 60, 4, 1, 1), (17, 60, 5, 3, 2), (9, 256, 8, 8, 4), (7, 160, 6, 8, 3), (3, 1, 1, 1, 1),
          (4, 1024, 32, 64, 7), (6, 384, 8, 1, 1), (2, 128, 32, 4, 1), (3, 130, 7, 65 // 5, 5), (50, 16, 16, 2, 2)]


def make(T, E, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + E + T)
    return (torch.randn((T, E), generator=g, device=DEV) * 1.5).to(dtype), torch.randn(E, generator=g, device=DEV) * 0.1


def check(logits, k, **kw):
    idx, wts = router.topk_scored(logits, k, **kw)
    ri, rw = M.route(logits, k, **kw)
    assert idx.dtype == torch.int32 and wts.dtype == torch.float32
    assert torch.equal(idx.long(), ri.long())
    # one rounding of a 64-bit number
    assert ((wts.double() - rw).abs() <= 2.0 ** -23 * rw.abs() + 1e-44).all(), float((wts.double() - rw).abs().max())


@pytest.mark.parametrize("dtype", LOGITS, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score,biased,by,norm", itertools.product(["softmax", "sigmoid"], [False, True], ["max", "top2"], [True, False]))
@pytest.mark.parametrize("T,E,k,groups,top", SHAPES)
def test_choice(T, E, k, groups, top, score, biased, by, norm, dtype):
    if by == "top2" and groups > 1 and E // groups < 2:
        pytest.skip("groups of one expert have no two largest")
    logits, bias = make(T, E, dtype)
    check(logits, k, score=score, bias=bias if biased else None, groups=groups, top_groups=top, group_score=by, norm=norm, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_and_masks(score, biased):
    """Equal logits: the lowest ids; masked, NaN and infinite ones; rows with nothing left."""
    E, k = 96, 6
    bias = torch.zeros(E, device=DEV) if biased else None
    g = torch.Generator(device=DEV).manual_seed(0)
    rows = [torch.zeros(E, device=DEV), torch.randint(0, 3, (E,), generator=g, device=DEV).float(),
            torch.full((E,), -math.inf, device=DEV), torch.full((E,), math.nan, device=DEV)]
    one = torch.full((E,), -math.inf, device=DEV)
    one[77] = 1.0
    few = one.clone()
    few[[3, 50, 95]] = torch.tensor([-300.0, -200.0, 2.0], device=DEV)
    low = torch.full((E,), torch.finfo(torch.float32).min, device=DEV)
    inf = torch.randn(E, generator=g, device=DEV)
    inf[[5, 60]] = math.inf
    nan = torch.randn(E, generator=g, device=DEV)
    nan[::2] = math.nan
    zero = torch.zeros(E, device=DEV)
    zero[::2] = -0.0
    logits = torch.stack(rows + [one, few, low, inf, nan, zero])
    for groups, top, by, norm in ((1, 1, "max", True), (1, 1, "max", False), (4, 2, "max", True), (4, 2, "top2", True), (8, 1, "top2", False),
                                  (3, 3, "max", True)):
        check(logits, k, score=score, bias=bias, groups=groups, top_groups=top, group_score=by, norm=norm)


def test_bias_of_infinities():
    """A bias of -inf (or NaN) takes an expert out, +inf in, whatever its logit; the weights do not see it."""
    logits, bias = make(20, 64, torch.float32)
    bias[3], bias[10], bias[40] = -math.inf, math.nan, math.inf
    for groups, top in ((1, 1), (8, 2)):
        for score, by in itertools.product(("softmax", "sigmoid"), ("max", "top2")):
            check(logits, 5, score=score, bias=bias, groups=groups, top_groups=top, group_score=by)
    out = torch.full((64,), -math.inf, device=DEV)
    check(logits, 5, score="sigmoid", bias=out)
    idx, wts = router.topk_scored(logits, 5, score="sigmoid", bias=out)
    assert (wts == 0).all() and torch.equal(idx[0].long(), torch.arange(5, device=DEV))


def test_scores_that_fp32_cannot_tell_apart():
    """Sigmoids near 1 (logits 18 apart by 1e-3 differ in the 10th digit), with and without a bias."""
    logits = (18 + 1e-3 * torch.randperm(64, generator=torch.Generator().manual_seed(0)).float()).to(DEV).expand(4, 64).contiguous()
    assert len(torch.sigmoid(logits[0]).unique()) < 8
    for bias in (None, torch.full((64,), 0.25, device=DEV)):
        check(logits, 8, score="sigmoid", bias=bias)
        check(logits, 8, score="sigmoid", bias=bias, groups=8, top_groups=3, group_score="top2")


def gradient64(logits, k, dw, idx, **kw):
    """Autograd of the formula in 64 bits, at the experts chosen."""
    l = logits.detach().double().requires_grad_()
    p = torch.softmax(l, 1) if kw["score"] == "softmax" else torch.sigmoid(l)
    s = p.gather(1, idx.long())
    w = kw.get("scale", 1.0) * (s / s.sum(1, keepdim=True) if kw["norm"] else s)
    (dl,) = torch.autograd.grad((w * dw.double()).sum(), l)
    return dl


@pytest.mark.parametrize("dtype", LOGITS, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score,norm", itertools.product(["softmax", "sigmoid"], [True, False]))
@pytest.mark.parametrize("T,E,k,groups,top", SHAPES)
def test_gradient(T, E, k, groups, top, score, norm, dtype):
    logits, bias = make(T, E, dtype)
    for b in (None, bias):
        kw = dict(score=score, bias=b, groups=groups, top_groups=top, norm=norm, scale=1.5)
        lg = logits.clone().requires_grad_()
        idx, wts = router.topk_scored(lg, k, **kw)
        assert not idx.requires_grad
        assert torch.equal(wts.detach(), router.topk_scored(logits, k, **kw)[1])
        dw = torch.randn((T, k), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
        (dl,) = torch.autograd.grad(wts, lg, dw)
        ref = gradient64(logits, k, dw, idx, **kw)
        assert dl.dtype == dtype
        # one rounding to the logits' type after one to fp32, of 64-bit sums; differences cancel down to 2^-50 of their terms
        tol = (torch.finfo(dtype).eps / 2 * 1.01 + 2.0 ** -23) * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0) + 1e-14
        assert ((dl.double() - ref).abs() <= tol).all(), float((dl.double() - ref).abs().max())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_gradient_against_differences(score, norm):
    """Central differences of the weights in fp32 along one direction: their roundings over the step, and the third derivative (at
    most 2 k times the direction's largest entry cubed) times the step squared."""
    logits, _ = make(12, 64, torch.float32)
    logits = torch.round(logits * 64) / 64
    v = torch.randint(-1, 2, logits.shape, generator=torch.Generator().manual_seed(0)).to(DEV).float()
    dw = torch.randn((12, 6), generator=torch.Generator().manual_seed(1)).to(DEV)
    eps = 2.0 ** -9
    f = lambda l: router.topk_scored(l, 6, score=score, norm=norm)   # noqa: E731
    lg = logits.clone().requires_grad_()
    idx, wts = f(lg)
    (dl,) = torch.autograd.grad(wts, lg, dw)
    d = torch.zeros((), dtype=torch.float64, device=DEV)
    kept = 0
    for t in range(12):
        (iu, wu), (idn, wd) = f((logits + eps * v)[t:t + 1]), f((logits - eps * v)[t:t + 1])
        if torch.equal(iu, idn) and torch.equal(iu, idx[t:t + 1]):   # where the step does not change the choice
            kept += 1
            got = float(((wu - wd).double() * dw[t].double()).sum()) / (2 * eps)
            want = float((dl[t].double() * v[t].double()).sum())
            size = float(dw[t].double().abs().sum())
            assert abs(got - want) <= size * (2.0 ** -23 / eps + 12 * eps * eps) + 2.0 ** -22 * float(dl[t].abs().sum())
    assert kept >= 6


def test_masked_experts_have_no_gradient():
    E, k = 32, 4
    logits = torch.full((3, E), -math.inf, device=DEV)
    logits[1, 5], logits[1, 9] = 1.0, 2.0
    logits[2] = torch.randn(E, generator=torch.Generator().manual_seed(0)).to(DEV)
    bias = torch.zeros(E, device=DEV)
    bias[4:] = -math.inf
    for score, norm in itertools.product(("softmax", "sigmoid"), (True, False)):
        for b in (None, bias):
            lg = logits.clone().requires_grad_()
            idx, wts = router.topk_scored(lg, k, score=score, norm=norm, bias=b)
            (dl,) = torch.autograd.grad(wts, lg, torch.ones_like(wts) * torch.arange(1, k + 1, device=DEV))
            assert torch.isfinite(dl).all()
            assert (dl[0] == 0).all()
            if b is None:
                assert (dl[1, [5, 9]] != 0).any() and (dl[1, 10:] == 0).all()


def test_gradients_of_masked_experts_weights_count_for_nothing():
    """Whatever reaches the weight of an expert that was chosen at -inf, an infinity or NaN too."""
    logits = torch.tensor([[1.0, 2.0, -math.inf, -math.inf], [0.5, -math.inf, -math.inf, -math.inf]], device=DEV)
    for score, norm in itertools.product(("softmax", "sigmoid"), (True, False)):
        grads = []
        for bad in (0.0, math.inf, math.nan):
            lg = logits.clone().requires_grad_()
            idx, wts = router.topk_scored(lg, 3, score=score, norm=norm)
            dw = torch.tensor([[0.3, -0.7, bad], [0.2, bad, bad]], device=DEV)
            grads.append(torch.autograd.grad(wts, lg, dw)[0])
        assert torch.isfinite(grads[0]).all()
        assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


def test_layouts_batches_empty():
    logits, bias = make(12, 64, torch.float32)
    idx, wts = router.topk_scored(logits, 4)
    a, b = router.topk_scored(logits.t().contiguous().t(), 4)
    assert torch.equal(idx, a) and torch.equal(wts, b)
    a, b = router.topk_scored(logits.reshape(3, 4, 64), 4)
    assert torch.equal(idx, a) and torch.equal(wts, b)
    a, b = router.topk_scored(torch.empty(0, 64, device=DEV), 4)
    assert a.shape == (0, 4) and b.shape == (0, 4)
    a, b = router.topk_scored(torch.cat([logits, logits], 1)[:, 32:96], 4, bias=bias.double().float().bfloat16().float())
    ri, _ = M.route(torch.cat([logits, logits], 1)[:, 32:96], 4, bias=bias.bfloat16().float())
    assert torch.equal(a.long(), ri.long())
    lg = logits.reshape(3, 4, 64).clone().requires_grad_()
    _, w = router.topk_scored(lg, 4, score="sigmoid")
    w.sum().backward()
    assert lg.grad.shape == lg.shape
    # equal to the plain router where both apply
    i0, w0 = router.topk_norm(logits, 6)
    i1, w1 = router.topk_scored(logits, 6)
    assert torch.equal(i0, i1)
    assert ((w0 - w1).abs() <= 2.0 ** -20 * w1).all()


@pytest.mark.parametrize("T", [1, 5, 300])
def test_route_scored(T):
    """route's logits, then topk_scored on them."""
    E, d, k = 64, 512, 6
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn((T, d), generator=g, device=DEV).bfloat16()
    wr = (torch.randn((E, d), generator=g, device=DEV) * d ** -0.5).bfloat16()
    wb, bias = torch.randn(E, generator=g, device=DEV) * 0.1, torch.randn(E, generator=g, device=DEV) * 0.05
    kw = dict(score="sigmoid", bias=bias, groups=8, top_groups=3, group_score="top2", scale=2.5)
    idx, wts, logits = router.route_scored(x, wr, k, wr_bias=wb, return_logits=True, **kw)
    assert torch.equal(logits, router.route(x, wr, k, bias=wb, return_logits=True)[2])
    a, b = router.topk_scored(logits, k, **kw)
    assert torch.equal(idx, a) and torch.equal(wts, b)
    x2 = torch.cat([x, x], 1)[:, d:]
    assert torch.equal(router.route_scored(x2, wr, k, wr_bias=wb, **kw)[0], idx)
    assert router.route_scored(x[:0], wr, k, **kw)[0].shape == (0, k)


def test_trained_router():
    """Gradients reach the router's weights through the experts: linear, topk_scored, experts_mlp."""
    from moelab_amd import dense
    T, E, k, d, F = 24, 16, 3, 64, 32
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((T, d), generator=g, device=DEV).bfloat16().requires_grad_()
    wr = (torch.randn((E, d), generator=g, device=DEV) * 0.2).bfloat16().requires_grad_()
    wgu = (torch.randn((E, 2 * F, d), generator=g, device=DEV) * 0.1).bfloat16()
    wd = (torch.randn((E, d, F), generator=g, device=DEV) * 0.1).bfloat16()
    logits = linear.linear(x, wr, out_dtype=torch.float32)
    idx, wts = router.topk_scored(logits, k, score="sigmoid", groups=4, top_groups=2)
    y = dense.experts_mlp(x, idx, wts, wgu, wd, checkpoint=False)
    dy = torch.randn((T, d), generator=g, device=DEV).bfloat16()
    dx, dwr = torch.autograd.grad(y, (x, wr), dy)
    x64, wr64 = x.detach().double().requires_grad_(), wr.detach().double().requires_grad_()
    s = torch.sigmoid(x64 @ wr64.T).gather(1, idx.long())
    w = s / s.sum(1, keepdim=True)
    out = torch.zeros_like(x64)
    for j in range(k):
        gu = torch.stack([wgu[e].double() @ x64[t] for t, e in enumerate(idx[:, j].tolist())])
        h = torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]
        out = out + w[:, j:j + 1] * torch.stack([wd[e].double() @ h[t] for t, e in enumerate(idx[:, j].tolist())])
    rx, rw = torch.autograd.grad(out, (x64, wr64), dy.double())
    # norms: roundings to 16 bits of z, h and the gradients between the calls, a handful of half steps of 2^-9
    for got, ref in ((dx, rx), (dwr, rw)):
        assert float((got.double() - ref).norm()) <= 8 * 2.0 ** -8 * float(ref.norm())


def test_captured_calls():
    logits, bias = make(40, 128, torch.float32)
    lg = logits.clone().requires_grad_()
    dw = torch.randn((40, 8), generator=torch.Generator().manual_seed(1)).to(DEV)

    def step():
        idx, w = router.topk_scored(lg, 8, score="sigmoid", bias=bias, groups=8, top_groups=4, group_score="top2")
        return idx, w.detach(), torch.autograd.grad(w, lg, dw)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        with torch.no_grad():
            lg.copy_(make(40, 128, torch.float32, seed=seed + 5)[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([t.clone() for t in got], step()):
            assert torch.equal(a, b)


def test_saved_elsewhere_in_between():
    """What the backward pass needs goes to the host and back, the bias to another address."""
    logits, bias = make(20, 64, torch.float32)
    kw = dict(score="sigmoid", groups=4, top_groups=2, group_score="top2")
    dw = torch.ones(20, 6, device=DEV) * torch.arange(6, device=DEV)
    bias[7] = -math.inf
    grads = []
    for away in (False, True):
        lg = logits.clone().requires_grad_()
        b = bias.clone()
        with torch.autograd.graph.save_on_cpu() if away else torch.enable_grad():
            idx, wts = router.topk_scored(lg, 6, bias=b.bfloat16(), **kw)
        del b
        waste = torch.full((64,), -math.inf, device=DEV)
        grads.append(torch.autograd.grad(wts, lg, dw)[0])
    assert torch.equal(*grads) and grads[0].any()
