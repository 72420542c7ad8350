"""Argument checks of the routing by scores, on the host: the C entry points return their error codes before any launch (no kernel
runs here), and the Python calls refuse what the kernels cannot take."""
import ctypes

import pytest
import torch

from moelab_amd import _lib, router

ARG, DT, AL = _lib.MOE_ERR_ARG, _lib.MOE_ERR_DTYPE, _lib.MOE_ERR_ALIGN
P, BAD = 4096, 4104   # fake device pointers: never followed
GOOD = dict(E=64, k=6, score=0, groups=8, top_groups=3, group_score=1, norm=1, scale=1.0, bias=None)
BAD_SETTINGS = [dict(E=0), dict(E=1025, groups=1, top_groups=1), dict(k=0), dict(k=33, top_groups=8), dict(k=25), dict(score=2), dict(score=-1),
                dict(groups=0), dict(groups=65, E=650), dict(groups=7), dict(top_groups=0), dict(top_groups=9), dict(group_score=2),
                dict(groups=64, top_groups=10)]


def call(settings, dtype=2, T=4, logits=P, idx=P, wts=P):
    return _lib.lib().moe_topk_scored(ctypes.byref(_lib.Scored(*(GOOD | settings).values())), logits, dtype, T, idx, wts, None)


def back(settings, dtype=2, T=4, logits=P, idx=P, dwts=P, dl=P):
    return _lib.lib().moe_topk_scored_bwd(ctypes.byref(_lib.Scored(*(GOOD | settings).values())), logits, dtype, T, idx, dwts, dl, None)


def route(settings, x=P, wr=P, T=4, d=64, logits=P, idx=P, wts=P):
    return _lib.lib().moe_router_scored(ctypes.byref(_lib.Scored(*(GOOD | settings).values())), x, wr, None, T, d, logits, idx, wts, None)


@pytest.mark.parametrize("settings", BAD_SETTINGS, ids=str)
def test_settings(settings):
    assert call(settings) == back(settings) == route(settings) == ARG


def test_pointers_types_and_empty_calls():
    assert call({}, dtype=3) == back({}, dtype=3) == DT
    assert call({}, T=-1) == back({}, T=-1) == route({}, T=-1) == ARG
    assert call({}, T=2 ** 31 - 1) == back({}, T=2 ** 31 - 1) == ARG
    assert call({}, T=0, logits=None, idx=None, wts=None) == 0
    assert back({}, T=0, logits=None, idx=None, dwts=None, dl=None) == 0
    assert route({}, T=0, x=None, wr=None, logits=None, idx=None, wts=None) == 0
    for name in ("logits", "idx", "wts"):
        assert call({}, **{name: None}) == ARG
    for name in ("logits", "idx", "dwts", "dl"):
        assert back({}, **{name: None}) == ARG
    for name in ("x", "wr", "logits", "idx", "wts"):
        assert route({}, **{name: None}) == ARG
    assert route({}, x=BAD) == route({}, wr=BAD) == AL
    assert route({}, d=60) == route({}, d=0) == ARG
    assert _lib.lib().moe_topk_scored(None, P, 2, 4, P, P, None) == ARG


def test_python_refusals():
    cpu = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        router.topk_scored(cpu, 4)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        router.route_scored(cpu.bfloat16(), cpu.bfloat16(), 4)

    def settings(E=64, k=6, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", norm=True, scale=1.0):
        return router._scored(E, k, score, bias, groups, top_groups, group_score, norm, scale, cpu.device)
    desc, bias = settings(bias=torch.ones(64, dtype=torch.bfloat16), groups=8, top_groups=2, group_score="top2", score="sigmoid", scale=2)
    assert (desc.E, desc.k, desc.score, desc.groups, desc.top_groups, desc.group_score, desc.norm, desc.scale) == (64, 6, 1, 8, 2, 1, 1, 2.0)
    assert bias.dtype == torch.float32 and desc.bias == bias.data_ptr()
    for kw in (dict(score="relu"), dict(group_score="mean"), dict(E=1025), dict(E=0), dict(groups=7), dict(groups=0), dict(groups=65, E=130),
               dict(groups=8, top_groups=9), dict(groups=8, top_groups=0), dict(k=0), dict(k=33), dict(k=9, groups=8, top_groups=1),
               dict(groups=64, top_groups=8, group_score="top2"), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(bias=torch.ones(63)), dict(bias=torch.ones(64, dtype=torch.int32)), dict(bias=torch.ones(1, 64)),
               dict(bias=torch.ones(64, device="meta"))):
        with pytest.raises(ValueError):
            settings(**kw)


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    wr = torch.zeros(16, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        router.topk_scored(x.double(), 4)
    with pytest.raises(TypeError):
        router.topk_scored(x.int(), 4)
    with pytest.raises(ValueError):
        router.topk_scored(x[0, 0], 4)
    with pytest.raises(TypeError):
        router.route_scored(x.float(), wr, 4)
    with pytest.raises(ValueError):
        router.route_scored(x[:, :32], wr, 4)
    with pytest.raises(ValueError):
        router.route_scored(x, wr, 4, wr_bias=torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        router.route_scored(x, wr.cpu(), 4)
    with pytest.raises(ValueError):
        router.route_scored(x[:, :60], wr[:, :60], 4)
    with pytest.raises(NotImplementedError):
        router.route_scored(x, wr.requires_grad_(), 4)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(NotImplementedError):
        router.topk_scored(fw.make_dual(x.float(), torch.ones_like(x.float())), 4)
    lg = torch.randn(4, 64, device="cuda", requires_grad=True)
    idx, wts = router.topk_scored(lg, 4)
    (g,) = torch.autograd.grad(wts.sum(), lg, create_graph=True)
    with pytest.raises(RuntimeError):   # no second derivative
        g.sum().backward()
    idx, wts = router.topk_scored(lg, 4)
    idx.add_(1)   # what the backward pass reads
    with pytest.raises(RuntimeError, match="modified"):
        wts.sum().backward()
