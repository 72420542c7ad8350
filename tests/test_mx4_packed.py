"""The packed form and back, on the CPU: sizes without rows or matrices among them."""
import pytest
import torch

from moelab_amd import mx4


@pytest.mark.parametrize("shape", [(0, 32), (3, 0, 64), (0, 8, 288), (5, 32), (2, 3, 544)])
def test_there_and_back(shape):
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(-2 ** 31, 2 ** 31, (*shape[:-1], shape[-1] // 8), generator=g).to(torch.int32)
    scales = torch.randint(1, 255, (*shape[:-1], shape[-1] // 32), generator=g).to(torch.uint8)
    q = mx4.from_packed(codes, scales)
    assert q.shape == shape
    a, b = mx4.to_packed(q)
    assert torch.equal(a, codes) and torch.equal(b, scales)
