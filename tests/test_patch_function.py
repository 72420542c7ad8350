"""patch_dense takes only modules whose own forward is the kernels' function: activations by their values, not their names, and
the rest of the forward by running it on random weights. Modules here are transformers' own and small ones written for the case."""
import pytest
import torch
import torch.nn.functional as nnf

import __graft_entry__

__graft_entry__.load_package()
from moelab_amd import _lib, patch  # noqa: E402
from test_patch import D, make_block  # noqa: E402


def experts(act=None):
    e = make_block("mixtral", "cpu").experts
    if act is not None:
        e.act_fn = act
    return e


def mlp(act=None):
    m = make_block("deepseek", "cpu").shared_experts
    if act is not None:
        m.act_fn = act
    return m


def activations():
    from transformers import activations as A
    return ({"silu": torch.nn.SiLU(), "silu2": A.ACT2FN["swish"]},
            {"tanh": torch.nn.GELU(approximate="tanh"), "pytorch_tanh": A.ACT2FN["gelu_pytorch_tanh"], "new": A.ACT2FN["gelu_new"],
             "fast": A.ACT2FN["gelu_fast"]},
            {"erf": torch.nn.GELU(), "gelu": A.ACT2FN["gelu"]},
            {"quick": A.ACT2FN["quick_gelu"], "hardswish": torch.nn.Hardswish(), "clipped": A.ACT2FN["gelu_10"], "relu": torch.nn.ReLU(),
             "linear": torch.nn.Identity()})


@pytest.mark.parametrize("make", [experts, mlp])
def test_activations(make):
    silu, tanh, erf, other = activations()
    for group, act in ((silu, _lib.ACT_SWIGLU), (tanh, _lib.ACT_GEGLU)):
        for fn in group.values():
            assert patch._act_of(make(fn)) == act
            patch.patch_dense(make(fn))
    for name, fn in (erf | other).items():
        m = make(fn)
        stock = m.forward
        with pytest.raises(NotImplementedError, match="activation"):
            patch.patch_dense(m)
        assert m.forward == stock and not hasattr(m, "_moelab_state"), name
    # the patches onto 4-bit weights take the exact GELU for the tanh form (4.7e-4 apart), as before, and no other function
    for fn in erf.values():
        assert patch._act_of(make(fn)) == _lib.ACT_GEGLU
    for fn in other.values():
        with pytest.raises(NotImplementedError, match="activation"):
            patch._act_of(make(fn))


def test_clamped_gates():
    """DeepSeek-V4 clamps its gates, in the experts and in the shared experts."""
    from transformers.models.deepseek_v4 import configuration_deepseek_v4 as C, modeling_deepseek_v4 as M
    cfg = C.DeepseekV4Config()
    for n, v in dict(hidden_size=64, intermediate_size=96, moe_intermediate_size=96, num_local_experts=4, n_routed_experts=4).items():
        if hasattr(cfg, n):
            setattr(cfg, n, v)
    for cls in (M.DeepseekV4Experts, M.DeepseekV4MLP):
        with pytest.raises(ValueError, match="something else"):
            patch.patch_dense(cls(cfg).to(torch.bfloat16))


def test_experts_without_weights():
    """LongCat-Flash has ids past its experts that stand for the identity."""
    from transformers.models.longcat_flash import configuration_longcat_flash as C, modeling_longcat_flash as M
    cfg = C.LongcatFlashConfig()
    for n, v in dict(hidden_size=64, expert_ffn_hidden_size=96, moe_intermediate_size=96, n_routed_experts=4).items():
        if hasattr(cfg, n):
            setattr(cfg, n, v)
    with pytest.raises(ValueError, match="something else"):
        patch.patch_dense(M.LongcatFlashExperts(cfg).to(torch.bfloat16))


class Experts(torch.nn.Module):
    """The plain layer, with one thing changed at a time."""

    def __init__(self, E=3, d=D, F=64, how="plain"):
        super().__init__()
        self.gate_up_proj = torch.nn.Parameter(torch.randn(E, 2 * F, d, dtype=torch.bfloat16))
        self.down_proj = torch.nn.Parameter(torch.randn(E, d, F, dtype=torch.bfloat16))
        self.act_fn, self.how, self.drop = torch.nn.SiLU(), how, torch.nn.Dropout(0.2 if how == "dropout" else 0.0)

    def forward(self, hidden_states, top_k_index, top_k_weights):
        how, out = self.how, torch.zeros_like(hidden_states)
        if how == "sizes":   # a forward that knows its own sizes
            hidden_states = hidden_states.reshape(-1, D)
        if how == "half":   # and one that takes 16 bits only
            assert hidden_states.dtype == torch.bfloat16
        for j in range(top_k_index.shape[1]):
            w = top_k_weights[:, j, None]
            for e in range(len(self.gate_up_proj)):
                x = hidden_states * w if how == "weighted inputs" else hidden_states
                g, u = nnf.linear(x, self.gate_up_proj[e]).chunk(2, -1)
                if how == "swapped":
                    g, u = u, g
                if how == "clamped":
                    u = u.clamp(-100.0, 100.0)
                h = self.act_fn(g) * (u + 1 if how == "plus one" else u)
                if how == "interleaved":
                    z = nnf.linear(x, self.gate_up_proj[e])
                    h = self.act_fn(z[:, ::2]) * z[:, 1::2]
                y = nnf.linear(self.drop(h), self.down_proj[e]) * (1 if how in ("weighted inputs", "unweighted") else w)
                out = out + torch.where(top_k_index[:, j, None] == e, y * (2 if how == "scaled" else 1), 0)
        return out


@pytest.mark.parametrize("how", ["plain", "sizes", "half"])
def test_takes(how):
    patch.patch_dense(Experts(how=how))


@pytest.mark.parametrize("how", ["weighted inputs", "unweighted", "swapped", "clamped", "plus one", "interleaved", "scaled", "dropout"])
def test_refuses(how):
    m = Experts(how=how).eval()
    with pytest.raises(ValueError, match="something else"):
        patch.patch_dense(m)
    assert not hasattr(m, "_moelab_state") and "forward" not in m.__dict__ and not m.training


def test_a_forward_that_cannot_be_run():
    m = Experts()
    m.__class__ = type("Odd", (Experts,), {"forward": lambda self, hidden_states: hidden_states})
    with pytest.raises(ValueError, match="could not be checked"):
        patch.patch_dense(m)


def test_the_check_leaves_the_module_alone():
    """No hook runs, no parameter or random state changes, a parametrised weight is looked through, one expert is enough."""
    m = Experts(E=1, how="plain")
    calls = []
    m.register_forward_hook(lambda *a: calls.append(a))
    m.act_fn.register_forward_hook(lambda *a: calls.append(a))
    before, rng = {n: p.clone() for n, p in m.named_parameters()}, torch.get_rng_state()
    patch.patch_dense(m)
    assert torch.equal(torch.get_rng_state(), rng) and all(torch.equal(p, before[n]) for n, p in m.named_parameters())
    assert not calls and m.training and all(p.requires_grad for p in m.parameters())

    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w
    m = Experts()
    torch.nn.utils.parametrize.register_parametrization(m, "down_proj", Twice())
    patch.patch_dense(m)


@pytest.mark.parametrize("device", ["meta", "cpu"])
def test_under_a_default_device(device):
    """The check runs on the CPU whatever device a program makes its tensors on by default (and in a model built on none)."""
    m, e, s = Experts(), experts(), mlp()
    with torch.device(device):
        patch.patch_dense(m)
        patch.patch_dense(e)
        patch.patch_dense(s)
    with torch.device("meta"):
        m = Experts(how="plain")
        patch.patch_dense(m)
        with pytest.raises(ValueError, match="something else"):
            patch.patch_dense(Experts(how="clamped"))
    assert all(p.is_meta for p in m.parameters())
