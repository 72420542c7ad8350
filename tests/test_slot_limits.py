"""Slot counts next to 2^31 are refused on the host: the kernels count slots in 32 bits, in steps past the last one, and a count
that wraps reads in front of the index lists. The largest accepted count of each entry point, worked through here as its
kernels step through it, stays below 2^31."""
import ctypes

import pytest

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import _lib  # noqa: E402

ARG = _lib.MOE_ERR_ARG
P = 4096   # a fake device pointer: never followed
SLOTS, GROUPED = 0x7fffff00, 0x78000000   # of a product; of a grouping


def calls(n):
    L = _lib.lib()
    lin = (P, P, None, None, 0, n, 64, 64, 64, 0, P, 0, None, P, 1 << 40, None)
    return {"moe_grouped_mm": lambda: L.moe_grouped_mm(P, P, None, P, None, n, n, 64, 2, 64, 64, 0, P, 0, 0, None),
            "moe_grouped_mm_dx": lambda: L.moe_grouped_mm_dx(P, P, P, None, n, n, 64, 2, 64, 64, 0, P, 0, 0, None),
            "moe_grouped_mm_dw": lambda: L.moe_grouped_mm_dw(P, P, P, None, None, n, n, 64, n, 64, 2, 64, 64, 0, P, 0, None, None),
            "moe_linear": lambda: L.moe_linear(*lin),
            "moe_linear_dx": lambda: L.moe_linear_dx(P, P, n, 64, 64, 64, 0, P, P, 1 << 40, None),
            "moe_linear_dw": lambda: L.moe_linear_dw(P, P, n, 64, 64, 64, 64, 0, P, None, P, 1 << 40, None)}


@pytest.mark.parametrize("name", list(calls(0)))
@pytest.mark.parametrize("n", [SLOTS + 1, 2 ** 31 - 64, 2 ** 31 - 1])
def test_products(name, n):
    assert calls(n)[name]() == ARG


@pytest.mark.parametrize("n", [GROUPED + 1, 2 ** 31 - 1])
def test_groupings(n):
    assert _lib.lib().moe_group(P, n, 8, P, P, P, P, P, None) == ARG


@pytest.mark.parametrize("T", [GROUPED // 64 + 1, 2 ** 25 - 1])
def test_expert_layers(T):
    L, k = _lib.lib(), 64
    m = _lib.Mlp(4, 8, 32, 0, 0, ctypes.c_void_p(P), ctypes.c_void_p(P))
    assert L.moe_mlp_fwd(m, P, P, P, T, k, None, P, 0, P, None, None, None, P, 1 << 62, None) == ARG
    assert L.moe_mlp_bwd(m, P, P, P, T, k, P, None, P, P, P, P, P, P, P, 1 << 62, None) == ARG


def test_the_largest_counts_do_not_wrap():
    # products: steps of 64 slots one past the last, each lane's slot of a step; rows rounded up to a tile
    n = SLOTS
    assert 64 * ((n + 63) // 64) + 63 < 2 ** 31 and n + 255 < 2 ** 31
    # a grouping's launches: 128 chunks of a multiple of 128 slots, four shares a chunk, sixteen waves that begin one
    for n in (GROUPED, GROUPED - 1, GROUPED - 127):
        per = (n + 127) // 128
        cs = (per + 127) // 128 * 128
        share = (cs + 255) // 256 * 64
        chunks = (n + cs - 1) // cs
        assert n + cs < 2 ** 31 and chunks * cs + 15 * share + 64 < 2 ** 31 and n + 16 * 8192 < 2 ** 31
    # in one workgroup: eight ids a thread
    assert GROUPED + 1024 * 8 < 2 ** 31
