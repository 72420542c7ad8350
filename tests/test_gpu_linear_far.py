"""Activations of linear.linear's sums past 2^64, whose square is past fp32, on every path, and the gradients there."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV  # noqa: F401
from moelab_amd.linear import GELU, SILU, linear
from test_gpu_linear import act_of, act_tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [SILU, GELU])
@pytest.mark.parametrize("T", [3, 17, 64, 300, 1024, 2048])
def test_sums_whose_square_overflows(T, act):
    N, K, dtype = 264, 64, torch.bfloat16
    x = (H.randn(T, K, dtype=torch.float32) * 2.0 ** 40).to(dtype).requires_grad_()
    w = (H.randn(N, K, dtype=torch.float32, seed=1) * 2.0 ** 40).to(dtype)
    b, r = H.randn(N, dtype=dtype, seed=2), H.randn(T, N, dtype=dtype, seed=3)
    xv, wv = x.detach().double(), w.double()
    z = xv @ wv.T + b.double()
    assert float(z.abs().median()) > 2.0 ** 64 and float(z.abs().min()) > 2.0 ** 40
    ref = act_of(act, z) + r.double()
    tol = act_tol(act, z, (K + 8) * 2.0 ** -23 * (xv.abs() @ wv.abs().T)) + 2.0 ** -23 * (ref.abs() + r.double().abs())
    for out in (dtype, torch.float32):
        step = H.half_step(dtype) if out == dtype else 2.0 ** -23
        H.check(linear(x.detach(), w, bias=b, act=act, residual=r, out_dtype=out), ref, tol + step * ref.abs())
    dy = H.randn(T, N, dtype=dtype, seed=4)
    (dx,) = torch.autograd.grad(linear(x, w, bias=b, act=act, residual=r), x, dy)
    dz = torch.where(z > 0, dy.double(), 0.0)   # the slope is 1 or 0 to the last bit
    H.check(dx, dz @ wv, H.product_tol(dz @ wv, dz.abs() @ wv.abs(), N, dtype))
