"""Argument checks of the MXFP4 operators, on the host: the C entry points return their error codes before any launch (no kernel runs
here), and the Python calls refuse what the kernels cannot take."""
import pytest
import torch

from moelab_amd import _lib, formats, mx4

ARG, DT, WS, AL = _lib.MOE_ERR_ARG, _lib.MOE_ERR_DTYPE, _lib.MOE_ERR_WORKSPACE, _lib.MOE_ERR_ALIGN
P, BAD = 4096, 4104   # fake device pointers: never followed
ROWS = 0x7fffff00


def quant(**k):
    a = dict(x=P, ldx=64, G=1, rows=4, K=64, dt=0, c=P, s=P) | k
    return _lib.lib().moe_mx4_quantize(*a.values(), None)


def dequant(**k):
    a = dict(c=P, s=P, G=1, rows=4, K=64, out=P, dt=0) | k
    return _lib.lib().moe_mx4_dequantize(*a.values(), None)


def lin(**k):
    a = dict(x=P, ldx=64, xc=None, xs=None, wc=P, ws=P, b=None, r=None, act=0, T=4, N=64, K=64, dt=0, y=P, ydt=0, z=None, w=P, n=1 << 40) | k
    return _lib.lib().moe_mx4_linear(*a.values(), None)


def lindx(**k):
    a = dict(dz=P, ld=64, wc=P, ws=P, T=4, N=64, K=64, dt=0, dx=P, w=P, n=1 << 40) | k
    return _lib.lib().moe_mx4_linear_dx(*a.values(), None)


def linbwd(**k):
    a = dict(dy=P, ld=64, z=P, act=1, xc=P, xs=P, wc=P, ws=P, T=4, N=64, K=64, dt=0, dx=P, dw=P, db=P, w=P, n=1 << 40) | k
    return _lib.lib().moe_mx4_linear_bwd(*a.values(), None)


def grp(**k):
    a = dict(x=P, ldx=64, xc=None, xs=None, xr=4, wc=P, ws=P, b=None, off=P, rows=None, M=4, E=2, N=64, K=64, dt=0, y=P, ydt=0, fill=0, w=P,
             n=1 << 40) | k
    return _lib.lib().moe_mx4_grouped_mm(*a.values(), None)


def grpdx(**k):
    a = dict(dy=P, ld=64, wc=P, ws=P, off=P, M=4, E=2, N=64, K=64, dt=0, dx=P, xdt=0, fill=0) | k
    return _lib.lib().moe_mx4_grouped_mm_dx(*a.values(), None)


BAD_K = [(dict(K=k, ldx=1 << 21), ARG) for k in (0, 16, 48, 2 ** 20 + 32, -32)]


@pytest.mark.parametrize("case,rc", BAD_K + [
    (dict(dt=3), DT), (dict(ldx=56), ARG), (dict(ldx=68), ARG), (dict(ldx=2 ** 22), ARG), (dict(G=2, ldx=72), ARG), (dict(G=-1), ARG),
    (dict(rows=-1), ARG), (dict(rows=ROWS + 1), ARG), (dict(G=3, rows=ROWS // 2), ARG), (dict(x=None), ARG), (dict(c=None), ARG),
    (dict(s=None), ARG), (dict(x=BAD), AL), (dict(c=BAD), AL), (dict(s=BAD), AL), (dict(rows=0, x=None, c=None), 0), (dict(G=0, x=None), 0)])
def test_quantize(case, rc):
    assert quant(**case) == rc


@pytest.mark.parametrize("case,rc", [(dict(K=48), ARG), (dict(dt=3), DT), (dict(rows=-1), ARG), (dict(out=None), ARG), (dict(c=None), ARG),
                                     (dict(s=None), ARG), (dict(out=BAD), AL), (dict(c=BAD), AL), (dict(s=BAD), AL), (dict(rows=0), 0)])
def test_dequantize(case, rc):
    assert dequant(**case) == rc


COMMON = [(dict(dt=2), DT), (dict(ydt=1), DT), (dict(N=60), ARG), (dict(N=0), ARG), (dict(N=2 ** 21), ARG), (dict(wc=None), ARG), (dict(ws=None), ARG),
          (dict(y=None), ARG), (dict(x=None), ARG), (dict(xc=P), ARG), (dict(xs=P), ARG), (dict(x=None, xc=P), ARG), (dict(x=BAD), AL),
          (dict(xc=BAD, xs=P), AL), (dict(xc=P, xs=BAD), AL), (dict(wc=BAD), AL), (dict(ws=BAD), AL), (dict(y=BAD), AL), (dict(b=BAD), AL),
          (dict(w=BAD), AL), (dict(ldx=56), ARG), (dict(ldx=68), ARG)]


@pytest.mark.parametrize("case,rc", BAD_K + COMMON + [
    (dict(act=3), ARG), (dict(act=-1), ARG), (dict(T=-1), ARG), (dict(T=ROWS + 1), ARG), (dict(r=BAD), AL), (dict(z=BAD), AL),
    (dict(T=100, w=None), WS), (dict(T=100, n=100), WS), (dict(T=0, x=None, wc=None, y=None), 0)])
def test_linear(case, rc):
    assert lin(**case) == rc


@pytest.mark.parametrize("case,rc", BAD_K + COMMON + [
    (dict(E=0), ARG), (dict(E=1025), ARG), (dict(off=None), ARG), (dict(M=-1), ARG), (dict(M=ROWS + 1, xr=ROWS), ARG), (dict(xr=3), ARG),
    (dict(rows=P, xr=0), ARG), (dict(rows=P, xr=0xB0000000 // 32 + 1), ARG), (dict(M=100, xr=100, w=None), WS), (dict(M=100, xr=100, n=10), WS),
    (dict(M=0, x=None, y=None), 0)])
def test_grouped(case, rc):
    assert grp(**case) == rc


@pytest.mark.parametrize("case,rc", [(dict(K=48), ARG), (dict(N=60), ARG), (dict(ld=56), ARG), (dict(dt=2), DT), (dict(wc=None), ARG),
                                     (dict(ws=None), ARG), (dict(wc=BAD), AL), (dict(ws=BAD), AL), (dict(dx=None), ARG), (dict(dx=BAD), AL)])
def test_gradients(case, rc):
    assert lindx(**case) == rc
    assert grpdx(**case) == rc
    assert lindx(dz=None) == grpdx(dy=None) == ARG
    assert lindx(dz=BAD) == grpdx(dy=BAD) == AL
    assert lindx(T=0, dz=None) == grpdx(M=0, dy=None) == 0
    assert lindx(T=-1) == grpdx(M=-1) == grpdx(E=0) == grpdx(off=None) == ARG
    assert grpdx(xdt=1) == DT
    assert lindx(T=100, N=4096, K=4096, ld=4096, w=None) == WS


def test_sizes():
    L = _lib.lib()
    assert L.moe_mx4_scale_bytes(1, 10, 32) == 10 * 8 + 16
    assert L.moe_mx4_scale_bytes(3, 10, 288) == 3 * 2 * 10 * 8 + 16
    assert L.moe_mx4_linear_workspace_bytes(0, 64, 64) == L.moe_mx4_linear_workspace_bytes(1, 64, 64) == 0
    assert L.moe_mx4_linear_workspace_bytes(100, 64, 64) >= 100 * 32 + 100 * 8
    assert L.moe_mx4_grouped_mm_workspace_bytes(8, 1, 128, 2048, 0) == 0
    assert L.moe_mx4_grouped_mm_workspace_bytes(800, 100, 8, 2048, 1) == 0
    assert L.moe_mx4_grouped_mm_workspace_bytes(800, 100, 8, 2048, 0) >= 100 * (1024 + 64)


NOTHING = dict(dx=None, dw=None, db=None, act=0)


@pytest.mark.parametrize("case,rc", [
    (dict(dt=2), DT), (dict(act=3), ARG), (dict(act=-1), ARG), (dict(T=-1), ARG), (dict(T=ROWS + 1), ARG), (dict(N=4), ARG), (dict(K=48), ARG),
    (dict(ld=56), ARG), (dict(ld=2 ** 22), ARG), (dict(dy=None), ARG), (dict(z=None), ARG), (dict(xc=None), ARG), (dict(xs=None), ARG),
    (dict(wc=None), ARG), (dict(ws=None), ARG), (dict(w=None), WS), (dict(n=0), WS), (dict(act=0, dx=None, db=None, n=0), WS),
    (NOTHING, 0), (NOTHING | dict(T=0, dy=None, xc=None, wc=None, w=None, n=0), 0)]
    + [({n: BAD}, AL) for n in ("dy", "z", "xc", "xs", "wc", "ws", "dx", "dw", "db", "w")])
def test_linear_bwd(case, rc):
    assert linbwd(**case) == rc


def test_packed_form_on_the_cpu():
    """from_packed and to_packed are layouts only: there and back, and what an Mx4 refuses."""
    w = torch.randn(3, 8, 288, generator=torch.Generator().manual_seed(0))
    words, scales = formats.quantize_mxfp4(w)
    q = mx4.from_packed(words, scales)
    assert q.shape == (3, 8, 288) and "Mx4([3, 8, 288]" in repr(q)
    a, b = mx4.to_packed(q)
    assert torch.equal(a, words) and torch.equal(b, scales)
    one = mx4.from_packed(words[0], scales[0])
    assert one.shape == (8, 288) and torch.equal(mx4.to_packed(one)[1], scales[0])
    import copy
    import pickle
    for r in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert r.shape == q.shape and torch.equal(r.codes, q.codes) and torch.equal(r.scales, q.scales)
    with pytest.raises(AttributeError):
        q.codes = q.codes[:, :4]
    for c, s in ((q.codes[..., :-8], q.scales), (q.codes.float(), q.scales), (q.codes, q.scales[:-1]), (q.codes, q.scales.int()),
                 (q.codes.transpose(0, 1), q.scales), (q.codes[None], q.scales), (q.codes[0, 0], q.scales)):
        with pytest.raises(ValueError):
            mx4.Mx4(c, s)
    for c, s in ((words.long(), scales), (words, scales.int()), (words, scales[..., :-1]), (words[..., :-1], scales), (words[0, 0], scales[0, 0])):
        with pytest.raises(ValueError):
            mx4.from_packed(c, s)


def test_python_refusals_on_the_cpu():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16)
    q = mx4.from_packed(*formats.quantize_mxfp4(w))
    for f in (lambda: mx4.quantize(x), lambda: mx4.dequantize(q), lambda: mx4.linear(x, w), lambda: mx4.linear(x, q),
              lambda: mx4.grouped_mm(x, w[None], torch.tensor([0, 4], dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            f()


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    dev, bf, h = "cuda", torch.bfloat16, torch.float16
    x, w = torch.zeros(4, 64, dtype=bf, device=dev), torch.zeros(8, 64, dtype=bf, device=dev)
    q, qx = mx4.quantize(w), mx4.quantize(x)
    off = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    q3 = mx4.quantize(w[None])
    for kind, f in ((TypeError, lambda: mx4.quantize(x.double())), (TypeError, lambda: mx4.quantize(x.int())),
                    (ValueError, lambda: mx4.quantize(x[:, :48])), (ValueError, lambda: mx4.quantize(x[0, 0])),
                    (TypeError, lambda: mx4.dequantize(q, torch.float64)),
                    (ValueError, lambda: mx4.linear(x[:, :32], q)), (TypeError, lambda: mx4.linear(x.half(), w)),
                    (TypeError, lambda: mx4.linear(x.float(), q)), (ValueError, lambda: mx4.linear(x, q3)),
                    (ValueError, lambda: mx4.linear(x, w[None])), (TypeError, lambda: mx4.linear(x, w.float())),
                    (ValueError, lambda: mx4.linear(x, mx4.quantize(w[:4]))), (ValueError, lambda: mx4.linear(x, w[:4])),
                    (TypeError, lambda: mx4.linear(x, q, bias=torch.zeros(8, dtype=h, device=dev))),
                    (ValueError, lambda: mx4.linear(x, q, bias=torch.zeros(9, dtype=bf, device=dev))),
                    (ValueError, lambda: mx4.linear(x, q, bias=torch.zeros(8, dtype=bf))),
                    (ValueError, lambda: mx4.linear(x, q, residual=torch.zeros(4, 9, dtype=bf, device=dev))),
                    (ValueError, lambda: mx4.linear(x, q, act=3)), (TypeError, lambda: mx4.linear(x, q, out_dtype=h)),
                    (ValueError, lambda: mx4.linear(mx4.quantize(x[:, :32]), q)),
                    (ValueError, lambda: mx4.grouped_mm(x, q, off)), (ValueError, lambda: mx4.grouped_mm(x[None], q3, off)),
                    (ValueError, lambda: mx4.grouped_mm(x, q3, off.long())), (ValueError, lambda: mx4.grouped_mm(x, q3, off[:1])),
                    (ValueError, lambda: mx4.grouped_mm(x, q3, off, rows=off.long())),
                    (ValueError, lambda: mx4.grouped_mm(x[:0], q3, off, rows=off)),
                    (TypeError, lambda: mx4.grouped_mm(x, q3, off, out=torch.zeros(4, 8, dtype=h, device=dev))),
                    (ValueError, lambda: mx4.grouped_mm(x, q3, off, out=torch.zeros(5, 8, dtype=bf, device=dev))),
                    (NotImplementedError, lambda: mx4.quantize(x.clone().requires_grad_())),
                    (ValueError, lambda: mx4.linear(qx, w.clone().requires_grad_())),
                    (ValueError, lambda: mx4.grouped_mm(qx, w[None].clone().requires_grad_(), off)),
                    (ValueError, lambda: mx4.grouped_mm(x.clone().requires_grad_(), q3, off, rows=off)),
                    (ValueError, lambda: mx4.grouped_mm(x.clone().requires_grad_(), q3, off, out=torch.zeros(4, 8, dtype=bf, device=dev)))):
        with pytest.raises(kind):
            f()
    assert mx4.linear(qx, q).dtype == bf and mx4.linear(qx, q, out_dtype=h).dtype == h
    assert mx4.linear(qx, w.half()).dtype == h and mx4.linear(qx, q, bias=torch.zeros(8, dtype=h, device=dev)).dtype == h
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(NotImplementedError):
        mx4.linear(fw.make_dual(x, torch.ones_like(x)), q)
