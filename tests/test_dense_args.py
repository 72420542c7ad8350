"""Argument checks of the 16-bit expert operators, on the host: the C entry points return their error codes before any launch (no
kernel runs here), and the Python calls refuse what the kernels cannot take."""
import ctypes

import pytest
import torch

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import _lib, act8, dense, grouped, linear  # noqa: E402

ARG, DT, WS, AL = _lib.MOE_ERR_ARG, _lib.MOE_ERR_DTYPE, _lib.MOE_ERR_WORKSPACE, _lib.MOE_ERR_ALIGN
P, BAD = 4096, 4104   # fake device pointers: never followed
FAR = 0xB0000000 // (2 * 64) + 1


def mm(**k):
    a = dict(x=P, w=P, bias=None, off=P, rows=None, M=4, xr=4, ldx=64, E=2, N=64, K=64, dt=0, y=P, ydt=0, fill=0) | k
    return _lib.lib().moe_grouped_mm(*a.values(), None)


def dx(**k):
    a = dict(dy=P, w=P, off=P, rows=None, M=4, yr=4, ld=64, E=2, N=64, K=64, dt=0, dx=P, xdt=0, fill=0) | k
    return _lib.lib().moe_grouped_mm_dx(*a.values(), None)


def dw(**k):
    a = dict(dy=P, x=P, off=P, yi=None, xi=None, M=4, yr=4, ldy=64, xr=4, ldx=64, E=2, N=64, K=64, dt=0, dw=P, wdt=0, db=None) | k
    return _lib.lib().moe_grouped_mm_dw(*a.values(), None)


def lin(**k):
    a = dict(x=P, w=P, b=None, r=None, act=0, T=4, ldx=64, N=64, K=64, dt=0, y=P, ydt=0, z=None, ws=P, wsb=1 << 40) | k
    return _lib.lib().moe_linear(*a.values(), None)


COMMON = [(dict(dt=2), DT), (dict(dt=7), DT), (dict(E=0), ARG), (dict(E=1025), ARG), (dict(off=None), ARG), (dict(M=-1), ARG), (dict(M=2 ** 31), ARG),
          (dict(N=60), ARG), (dict(K=4), ARG), (dict(N=0), ARG), (dict(K=2 ** 21), ARG), (dict(w=BAD), AL), (dict(w=None), ARG)]


@pytest.mark.parametrize("case,rc", COMMON + [
    (dict(ydt=1), DT), (dict(ldx=56), ARG), (dict(ldx=68), ARG), (dict(ldx=2 ** 22), ARG), (dict(x=None), ARG), (dict(y=None), ARG),
    (dict(x=BAD), AL), (dict(y=BAD), AL), (dict(bias=BAD), AL), (dict(xr=3), ARG), (dict(rows=P, xr=0), ARG), (dict(rows=P, xr=FAR), ARG),
    (dict(M=0, x=None, y=None), 0)])
def test_grouped_mm(case, rc):
    assert mm(**case) == rc


@pytest.mark.parametrize("case,rc", COMMON + [
    (dict(xdt=1), DT), (dict(ld=56), ARG), (dict(dy=BAD), AL), (dict(dx=BAD), AL), (dict(dy=None), ARG), (dict(dx=None), ARG),
    (dict(yr=3), ARG), (dict(rows=P, yr=FAR), ARG), (dict(M=0), 0)])
def test_grouped_mm_dx(case, rc):
    assert dx(**case) == rc


@pytest.mark.parametrize("case,rc", [c for c in COMMON if "w" not in c[0]] + [
    (dict(wdt=1), DT), (dict(ldy=56), ARG), (dict(ldx=56), ARG), (dict(dy=BAD), AL), (dict(x=BAD), AL), (dict(dw=BAD), AL),
    (dict(dw=None), ARG), (dict(x=None), ARG), (dict(yr=3), ARG), (dict(xr=3), ARG), (dict(yi=P, yr=0), ARG),
    (dict(yi=P, xr=FAR), ARG), (dict(xi=P, yr=FAR), ARG)])
def test_grouped_mm_dw(case, rc):
    assert dw(**case) == rc


@pytest.mark.parametrize("case,rc", [
    (dict(dt=2), DT), (dict(ydt=1), DT), (dict(act=3), ARG), (dict(act=-1), ARG), (dict(T=-1), ARG), (dict(N=12), ARG), (dict(K=63), ARG),
    (dict(ldx=56), ARG), (dict(x=None), ARG), (dict(w=None), ARG), (dict(y=None), ARG), (dict(z=BAD), AL), (dict(r=BAD), AL),
    (dict(b=BAD), AL), (dict(T=0, x=None), 0)])
def test_linear(case, rc):
    assert lin(**case) == rc


def test_linear_act_bwd():
    f = _lib.lib().moe_linear_act_bwd
    def call(**k):
        a = dict(dy=P, ld=64, z=P, codes=None, scales=None, act=1, T=4, N=64, dt=0, dz=P) | k
        return f(*a.values(), None)
    for case, rc in ((dict(dt=2), DT), (dict(act=0), ARG), (dict(act=3), ARG), (dict(z=None), ARG), (dict(codes=P, scales=P), ARG),
                     (dict(z=None, codes=P), ARG), (dict(z=None, codes=P, scales=P, N=40), ARG), (dict(dz=BAD), AL), (dict(ld=60), ARG),
                     (dict(T=0, dy=None), 0)):
        assert call(**case) == rc, case


def test_act8():
    L = _lib.lib()
    assert L.moe_act8_pack(P, 64, 4, 64, 2, P, P, None) == DT
    assert L.moe_act8_pack(P, 48, 4, 48, 0, P, P, None) == ARG and L.moe_act8_pack(P, 32, 4, 64, 0, P, P, None) == ARG
    assert L.moe_act8_pack(BAD, 64, 4, 64, 0, P, P, None) == AL and L.moe_act8_pack(None, 64, 4, 64, 0, P, P, None) == ARG
    assert L.moe_act8_unpack(P, P, 4, 48, P, 0, None) == ARG and L.moe_act8_unpack(P, P, 4, 64, P, 5, None) == DT
    assert L.moe_act8_unpack(P, None, 4, 64, P, 0, None) == ARG and L.moe_act8_unpack(P, P, 4, 64, BAD, 0, None) == AL
    assert L.moe_glu_fwd(P, 128, 4, 64, 3, 0, P, P, P, None) == ARG and L.moe_glu_fwd(P, 64, 4, 64, 0, 0, P, P, P, None) == ARG
    assert L.moe_glu_fwd(P, 128, 4, 64, 0, 0, P, P, None, None) == ARG and L.moe_glu_fwd(P, 96, 4, 48, 0, 0, P, P, P, None) == ARG
    assert L.moe_glu_fwd(P, 128, 4, 64, 0, 2, P, P, P, None) == DT and L.moe_glu_fwd(P, 128, 0, 64, 0, 0, None, None, None, None) == 0
    def bwd(**k):
        a = dict(codes=P, scales=P, gu=None, ld=0, dh=P, ddt=0, wts=None, M=4, F=64, act=0, dt=0, dgu=P, hw=P, dw=P) | k
        return L.moe_glu_bwd(*a.values(), None)
    for case, rc in ((dict(dt=2), DT), (dict(ddt=1), DT), (dict(act=5), ARG), (dict(F=40), ARG), (dict(scales=None), ARG),
                     (dict(codes=None), ARG), (dict(gu=P, ld=128), ARG), (dict(codes=None, gu=P, ld=64), ARG), (dict(dh=BAD), AL),
                     (dict(dgu=None), ARG), (dict(M=0), 0)):
        assert bwd(**case) == rc, case


def _mlp(**k):
    a = dict(E=4, d=64, F=64, act=0, dtype=0, w_gate_up=P, w_down=P) | k
    return _lib.Mlp(*[a[n] if n[0] != "w" or a[n] is None else ctypes.c_void_p(a[n]) for n in a])


@pytest.mark.parametrize("m,case,rc", [
    (dict(dtype=2), {}, DT), (dict(act=4), {}, ARG), (dict(d=60), {}, ARG), (dict(F=40), {}, ARG), (dict(E=0), {}, ARG),
    (dict(E=1025), {}, ARG), (dict(w_down=None), {}, ARG), (dict(w_gate_up=BAD), {}, AL), ({}, dict(T=-1), ARG), ({}, dict(k=0), ARG),
    ({}, dict(T=FAR), ARG), ({}, dict(T=2 ** 30, k=4), ARG), ({}, dict(ydt=1), DT), ({}, dict(x=None), ARG), ({}, dict(keep=None), ARG),
    ({}, dict(codes=P), ARG), ({}, dict(ws=None), WS), ({}, dict(wsb=100), WS), ({}, dict(y=BAD), AL), ({}, dict(T=0, x=None), 0)])
def test_mlp_fwd(m, case, rc):
    a = dict(x=P, idx=P, wts=P, T=4, k=2, r=None, y=P, ydt=0, keep=P, gu=None, codes=None, scales=None, ws=P, wsb=1 << 40) | case
    assert _lib.lib().moe_mlp_fwd(_mlp(**m), *a.values(), None) == rc


@pytest.mark.parametrize("m,case,rc", [
    (dict(dtype=2), {}, DT), ({}, dict(keep=None), ARG), ({}, dict(codes=None), ARG), ({}, dict(gu=P), ARG), ({}, dict(scales=None), ARG),
    ({}, dict(dy=None), ARG), ({}, dict(ws=None), WS), ({}, dict(wsb=100), WS), ({}, dict(dx=BAD), AL), ({}, dict(T=0), ARG)])
def test_mlp_bwd(m, case, rc):
    a = dict(x=P, wts=P, dy=P, T=4, k=2, keep=P, gu=None, codes=P, scales=P, dx=P, dw=P, dgu=P, ddn=P, ws=P, wsb=1 << 40) | case
    assert _lib.lib().moe_mlp_bwd(_mlp(**m), *a.values(), None) == rc


def test_mlp_sizes():
    L = _lib.lib()
    m = _mlp()
    assert L.moe_mlp_keep_bytes(m, 4, 2) >= 3 * 8 * 4 and L.moe_mlp_keep_bytes(None, 4, 2) == 0
    assert L.moe_mlp_fwd_workspace_bytes(m, 100, 2) > L.moe_mlp_fwd_workspace_bytes(m, 50, 2) > 0
    assert L.moe_mlp_bwd_workspace_bytes(m, 100, 2) >= 200 * (64 * 4 + 2 * 64 * 2 + 64 * 2 + 64 * 2)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(2, 64, 64, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    for fn in (lambda: grouped.mm(x, w, off), lambda: grouped.mm_dx(x, w, off), lambda: grouped.mm_dw(x, x, off, 2),
               lambda: linear.linear(x, w[0]), lambda: act8.pack(x), lambda: act8.glu_forward(x), lambda: act8.unpack(x, x),
               lambda: act8.glu_backward(None, None, x, gu=x), lambda: linear.act_backward(x, x, 1),
               lambda: dense.experts_mlp(x, off[:, None], off[:, None], w, w)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            fn()


class Fake:
    """What the host checks read of a GPU tensor, without one."""

    def __init__(self, *shape, dtype=torch.bfloat16, device="cuda:0", grad=False):
        self._t = torch.empty(shape, dtype=dtype, device="meta")
        self.device, self.requires_grad, self.is_cuda, self.dtype, self.shape = torch.device(device), grad, True, dtype, self._t.shape

    def __getattr__(self, n):
        return getattr(self._t, n)

    def data_ptr(self):
        return P


BF, HF, I32 = torch.bfloat16, torch.float16, torch.int32


@pytest.mark.parametrize("call,error,words", [
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 60, 64), Fake(3, dtype=I32)), ValueError, "N = 60"),
    (lambda: grouped.mm(Fake(4, 60), Fake(2, 64, 60), Fake(3, dtype=I32)), ValueError, "K = 60"),
    (lambda: grouped.mm(Fake(4, 72), Fake(2, 64, 64), Fake(3, dtype=I32)), ValueError, "x has shape"),
    (lambda: grouped.mm(Fake(4, 64, dtype=HF), Fake(2, 64, 64), Fake(3, dtype=I32)), TypeError, "x is"),
    (lambda: grouped.mm(Fake(4, 64, dtype=torch.float32), Fake(2, 64, 64, dtype=torch.float32), Fake(3, dtype=I32)), TypeError, "w is"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(4, dtype=I32)), ValueError, "offsets"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=torch.int64)), ValueError, "offsets"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), None), ValueError, "offsets"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=I32, device="cuda:1")), ValueError, "cuda:1"),
    (lambda: grouped.mm(Fake(4, 64, device="cuda:1"), Fake(2, 64, 64), Fake(3, dtype=I32)), ValueError, "cuda:1"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=I32), bias=Fake(2, 72)), ValueError, "bias"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=I32), bias=Fake(2, 64, dtype=HF)), TypeError, "bias"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=I32), rows=Fake(4, 2, dtype=I32)), ValueError, "rows"),
    (lambda: grouped.mm(Fake(0, 64), Fake(2, 64, 64), Fake(3, dtype=I32), rows=Fake(4, dtype=I32)), ValueError, "no rows"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=I32), out_dtype=HF), TypeError, "out_dtype"),
    (lambda: grouped.mm(Fake(4, 64), Fake(2, 64, 64), Fake(3, dtype=I32), out=Fake(5, 64)), ValueError, "out"),
    (lambda: grouped.mm(Fake(4, 64, grad=True), Fake(2, 64, 64), Fake(3, dtype=I32), out=Fake(4, 64)), ValueError, "no gradient"),
    (lambda: grouped.mm(Fake(4, 64, grad=True), Fake(2, 64, 64), Fake(3, dtype=I32), rows=Fake(9, dtype=I32)), ValueError, "gradient"),
    (lambda: grouped.mm_dx(Fake(4, 72), Fake(2, 64, 64), Fake(3, dtype=I32)), ValueError, "dy has shape"),
    (lambda: grouped.mm_dw(Fake(4, 64), Fake(5, 64), Fake(3, dtype=I32), 2), ValueError, "slots"),
    (lambda: grouped.mm_dw(Fake(4, 64), Fake(4, 64), None, 2), ValueError, "offsets"),
    (lambda: grouped.mm_dw(Fake(4, 60), Fake(4, 64), Fake(3, dtype=I32), 2), ValueError, "N = 60"),
    (lambda: linear.linear(Fake(4, 64), Fake(60, 64)), ValueError, "N = 60"),
    (lambda: linear.linear(Fake(4, 72), Fake(64, 64)), ValueError, "x has shape"),
    (lambda: linear.linear(Fake(4, 64), Fake(64, 64), act=3), ValueError, "act"),
    (lambda: linear.linear(Fake(4, 64), Fake(64, 64), bias=Fake(72)), ValueError, "bias"),
    (lambda: linear.linear(Fake(4, 64), Fake(64, 64), residual=Fake(4, 72)), ValueError, "residual"),
    (lambda: linear.linear(Fake(4, 64), Fake(64, 64), residual=Fake(4, 64, dtype=torch.float32)), TypeError, "residual"),
    (lambda: linear.linear(Fake(4, 64), Fake(40, 64), act=1, checkpoint=True), ValueError, "checkpoint"),
    (lambda: linear.act_backward(Fake(4, 64), None, 1), ValueError, "either"),
    (lambda: linear.act_backward(Fake(4, 64), Fake(4, 64), 0), ValueError, "act"),
    (lambda: act8.pack(Fake(4, 40)), ValueError, "columns = 40"),
    (lambda: act8.pack(Fake(4, 64, dtype=torch.float32)), TypeError, "x is"),
    (lambda: act8.unpack(Fake(4, 64, dtype=torch.int8), Fake(4, 3, dtype=torch.uint8)), ValueError, "scales"),
    (lambda: act8.unpack(Fake(4, 64, dtype=torch.uint8), Fake(4, 2, dtype=torch.uint8)), TypeError, "codes"),
    (lambda: act8.glu_forward(Fake(4, 80)), ValueError, "F = 40"),
    (lambda: act8.glu_forward(Fake(4, 64), act=7), ValueError, "act"),
    (lambda: act8.glu_backward(None, None, Fake(4, 64)), ValueError, "either"),
    (lambda: act8.glu_backward(Fake(4, 64, dtype=torch.int8), Fake(4, 2, dtype=torch.uint8), Fake(4, 64)), ValueError, "codes"),
    (lambda: act8.glu_backward(None, None, Fake(4, 64), gu=Fake(5, 128)), ValueError, "rows"),
    (lambda: dense.experts_mlp(Fake(4, 64), Fake(4, 2, dtype=I32), Fake(4, 2), Fake(2, 100, 64), Fake(2, 64, 50)), ValueError, "F = 50"),
    (lambda: dense.experts_mlp(Fake(4, 64), Fake(4, 2, dtype=I32), Fake(4, 2), Fake(2, 64, 64), Fake(2, 64, 64)), ValueError, "w_gate_up"),
    (lambda: dense.experts_mlp(Fake(4, 64), Fake(3, 2, dtype=I32), Fake(3, 2), Fake(2, 128, 64), Fake(2, 64, 64)), ValueError, "idx"),
    (lambda: dense.experts_mlp(Fake(4, 64), Fake(4, 2, dtype=I32), Fake(4, 3), Fake(2, 128, 64), Fake(2, 64, 64)), ValueError, "wts"),
    (lambda: dense.experts_mlp(Fake(4, 64), Fake(4, 2, dtype=BF), Fake(4, 2), Fake(2, 128, 64), Fake(2, 64, 64)), TypeError, "idx"),
    (lambda: dense.experts_mlp(Fake(4, 64), Fake(4, 2, dtype=I32), Fake(4, 2), Fake(2, 128, 64, dtype=HF), Fake(2, 64, 64)), TypeError, "w_gate_up"),
    (lambda: dense.glu_mlp(Fake(4, 64), Fake(64, 64), Fake(64, 64), Fake(64, 64), act=2), ValueError, "act"),
])
def test_refusals(call, error, words, monkeypatch):
    # nothing may get as far as a result or a launch
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("reached the library"))
    monkeypatch.setattr(_lib, "dense", lambda t, dtype=None: t)
    with pytest.raises(error, match=words):
        call()
