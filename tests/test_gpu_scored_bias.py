"""router.topk_scored's bias belongs to the caller, who may change it at any time, as a bias that balances the experts is."""
import math

import pytest
import torch

from dense_helpers import DEV
from moelab_amd import router

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("norm", [True, False])
def test_bias_changed_before_the_backward_pass(score, norm, dtype):
    """The gradient is that of the call, whatever the bias holds by then: experts that were chosen at -inf stay without one, and the
    others keep theirs where the bias becomes -inf."""
    T, E, k = 33, 16, 6
    g = torch.Generator(device=DEV).manual_seed(0)
    logits = torch.randn(T, E, generator=g, device=DEV)
    bias = torch.randn(E, generator=g, device=DEV).mul_(0.1).to(dtype)
    bias[5:] = -math.inf   # one expert too few: the last choice is a dead one
    dw = torch.randn(T, k, generator=g, device=DEV)
    grads = []
    for change in (None, 0.0, -math.inf):
        lg, b = logits.clone().requires_grad_(), bias.clone()
        idx, wts = router.topk_scored(lg, k, score=score, bias=b, norm=norm)
        assert (wts[:, -1] == 0).all()
        if change is not None:
            with torch.no_grad():
                b.fill_(change)
        grads.append((idx, *torch.autograd.grad(wts, lg, dw)))
    for other in grads[1:]:
        assert all(torch.equal(p, q) for p, q in zip(grads[0], other))
    assert grads[0][1].any() and not (score == "sigmoid" and grads[0][1].gather(1, grads[0][0][:, -1:].long()).any())
