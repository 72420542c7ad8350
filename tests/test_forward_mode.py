"""Forward-mode derivatives raise in the 16-bit operators, for every argument that has a gradient, instead of being lost."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import act8, dense, grouped, linear  # noqa: E402

BF = torch.bfloat16
OPS = {
    "mm": (lambda x, w, b: grouped.mm(x, w, torch.tensor([0, 2, 4], dtype=torch.int32, device=x.device), bias=b), [(4, 64), (2, 64, 64), (2, 64)]),
    "linear": (lambda x, w, b, r: linear.linear(x, w, bias=b, act=1, residual=r), [(4, 64), (64, 64), (64,), (4, 64)]),
    "glu": (lambda gu: act8.glu(gu), [(4, 64)]),
    "experts_mlp": (lambda x, wts, gu, dn, r: dense.experts_mlp(x, torch.zeros(4, 2, dtype=torch.int32, device=x.device), wts, gu, dn, residual=r),
                    [(4, 64), (4, 2), (2, 64, 64), (2, 64, 32), (4, 64)]),
    "glu_mlp": (lambda x, g, u, dn, r: dense.glu_mlp(x, g, u, dn, residual=r), [(4, 64), (32, 64), (32, 64), (64, 32), (4, 64)]),
}
CASES = [(n, i) for n, (_, shapes) in OPS.items() for i in range(len(shapes))]


def lost(name, i, device):
    fn, shapes = OPS[name]
    args = [torch.ones(s, dtype=BF, device=device) for s in shapes]
    with fw.dual_level():
        args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fn(*args)


# on the CPU the check comes before the device's, but where an earlier product of glu_mlp meets that one
@pytest.mark.parametrize("name,i", [c for c in CASES if c not in (("glu_mlp", 2), ("glu_mlp", 3), ("glu_mlp", 4))])
def test_raises(name, i):
    lost(name, i, "cpu")


@pytest.mark.parametrize("name", list(OPS))
def test_function_transform_raises(name):
    fn, shapes = OPS[name]
    args = tuple(torch.ones(s, dtype=BF) for s in shapes)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(fn, args, args)


@pytest.mark.gpu
@pytest.mark.parametrize("name,i", CASES)
def test_raises_on_the_gpu(name, i):
    lost(name, i, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(OPS))
def test_other_tensors_of_a_level_do_not_matter(name):
    """Operands without a tangent inside a level are ordinary ones, backward pass included."""
    fn, shapes = OPS[name]
    args = [torch.ones(s, dtype=BF, device="cuda") for s in shapes]
    with fw.dual_level():
        fw.make_dual(torch.ones(2), torch.ones(2))
        leaves = [a.requires_grad_() for a in args]
        assert all(torch.isfinite(g).all() for g in torch.autograd.grad(fn(*leaves).sum(), leaves))
