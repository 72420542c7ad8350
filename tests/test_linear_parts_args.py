"""Argument checks of moe_linear_dx and moe_linear_dw on the host (no kernel runs), and the workspaces of products in parts."""
import pytest

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import _lib  # noqa: E402

ARG, DT, WS, AL = _lib.MOE_ERR_ARG, _lib.MOE_ERR_DTYPE, _lib.MOE_ERR_WORKSPACE, _lib.MOE_ERR_ALIGN
P, BAD = 4096, 4104   # fake device pointers: never followed


def dx(**k):
    a = dict(dz=P, w=P, T=9, ld=64, N=64, K=64, dt=0, dx=P, ws=P, wsb=1 << 40) | k
    return _lib.lib().moe_linear_dx(*a.values(), None)


def dw(**k):
    a = dict(dz=P, x=P, T=9, ldz=64, ldx=64, N=64, K=64, dt=0, dw=P, db=None, ws=P, wsb=1 << 40) | k
    return _lib.lib().moe_linear_dw(*a.values(), None)


COMMON = [(dict(dt=2), DT), (dict(dt=7), DT), (dict(T=-1), ARG), (dict(T=2 ** 31), ARG), (dict(N=60), ARG), (dict(K=4), ARG),
          (dict(N=0), ARG), (dict(K=2 ** 21), ARG), (dict(dz=None), ARG), (dict(dz=BAD), AL), (dict(ws=BAD), AL)]


@pytest.mark.parametrize("case,rc", COMMON + [(dict(ld=56), ARG), (dict(ld=68), ARG), (dict(w=None), ARG), (dict(w=BAD), AL),
                                              (dict(dx=None), ARG), (dict(dx=BAD), AL), (dict(T=0, dz=None, dx=None), 0)])
def test_dx(case, rc):
    assert dx(**case) == rc


@pytest.mark.parametrize("case,rc", COMMON + [(dict(ldz=56), ARG), (dict(ldx=56), ARG), (dict(ldx=2 ** 22), ARG), (dict(x=None), ARG),
                                              (dict(x=BAD), AL), (dict(dw=None), ARG), (dict(dw=BAD), AL), (dict(T=0, dw=None), ARG)])
def test_dw(case, rc):
    assert dw(**case) == rc


def test_workspaces():
    L = _lib.lib()
    n = L.moe_linear_workspace_bytes(64, 1032, 2056)
    assert n > 0 and n % (64 * 1032 * 4) == 0
    assert L.moe_linear(P, P, None, None, 0, 64, 2056, 1032, 2056, 0, P, 0, None, P, n - 1, None) == WS
    n = L.moe_linear_dx_workspace_bytes(64, 2056, 1032)
    assert n > 0 and dx(T=64, ld=2056, N=2056, K=1032, wsb=n - 1) == WS
    n = L.moe_linear_dw_workspace_bytes(5000, 72, 136)
    assert n > 0 and n % ((72 * 136 + 72) * 4) == 0 and dw(T=5000, ldz=72, ldx=136, N=72, K=136, wsb=n - 1) == WS
    # none where the tiles fill the machine, where there are no rows, and where a few rows take the dot products
    for f in (L.moe_linear_workspace_bytes, L.moe_linear_dx_workspace_bytes, L.moe_linear_dw_workspace_bytes):
        assert f(4096, 4096, 4096) == 0 and f(0, 64, 64) == 0
    assert all(L.moe_linear_workspace_bytes(t, 64, 4096) == 0 for t in (1, 2, 3, 4))


def test_null_workspace():
    """A size that needs one refuses NULL, whatever length is claimed."""
    assert dx(T=64, ld=2056, N=2056, K=1032, ws=None) in (ARG, WS) and dw(T=5000, ldz=72, ldx=136, N=72, K=136, ws=None) in (ARG, WS)
    assert _lib.lib().moe_linear(P, P, None, None, 0, 64, 2056, 1032, 2056, 0, P, 0, None, None, 1 << 40, None) in (ARG, WS)
