"""The 8-bit form at the ends of the 16-bit types' ranges: finite values come back finite, within the form's bound."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import act8

pytestmark = pytest.mark.gpu


def all_finite(dtype):
    """Every finite value of a 16-bit type, each at the head of a block of its own, with smaller ones behind it."""
    v = torch.arange(-2 ** 15, 2 ** 15, device=DEV).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    return (v[:, None].double() * torch.linspace(1, -1, 32, dtype=torch.float64, device=DEV)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_every_largest_value(dtype):
    x = all_finite(dtype)
    codes, scales = act8.pack(x)
    want, wants = H.quantise(x)
    assert torch.equal(codes, want) and torch.equal(scales, wants)
    exact = H.values(codes, scales)
    assert torch.equal(act8.unpack(codes, scales, torch.float32).double(), exact)
    top = torch.finfo(dtype).max
    back = act8.unpack(codes, scales, dtype).double()
    assert torch.isfinite(back).all() and torch.equal(back, exact.clamp(-top, top))
    # half a step, which is at most 1/127.5 of the block's largest value
    gap, largest = (back - x.double()).abs(), x.double().abs().amax(1, keepdim=True)
    assert (gap <= H.pow2(scales.to(torch.int64) - 134)).all() and (gap <= largest / 127.5).all()


def test_other_values_in_fp16():
    """Codes of bf16 values: past fp16's range they are infinite, 65536 apart. (65024 and 66048 are 63.5 and 64.5 steps of
    1024, 66560 is 65: ties go to the even 64.)"""
    x = torch.zeros(1, 160, dtype=torch.bfloat16, device=DEV)
    x[0, 0], x[0, 32], x[0, 33], x[0, 64], x[0, 96], x[0, 128] = 65536, -65536, 65024, 66048, float("nan"), 66560
    v = act8.unpack(*act8.pack(x), torch.float16)[0]
    assert v[0] == 65504 and v[32] == -65504 and v[33] == 65504 and v[64] == 65504
    assert torch.isnan(v[96:128]).all() and v[128] == float("inf") and not v[129:].any()


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_a_saved_and_restored_row_is_finite(dtype):
    x = torch.full((3, 64), torch.finfo(dtype).max, dtype=dtype, device=DEV)
    x[1] *= -1
    x[2, ::2] = 0
    v = act8.unpack(*act8.pack(x), dtype)
    assert torch.isfinite(v).all() and ((v.double() - x.double()).abs() <= x.double().abs() / 127.5).all()
