"""What a program does with a module under patch_dense besides calling it: copies, second patches, models that are refused in the
middle, hooks on and replacements of its parts. The expert layer's calls are recorded here, not run."""
import copy

import pytest
import torch

import __graft_entry__

__graft_entry__.load_package()
import dense_helpers as H  # noqa: E402
from moelab_amd import dense, patch  # noqa: E402
from test_patch import D, make_block  # noqa: E402


@pytest.fixture
def calls(monkeypatch):
    """The arguments of the expert layer's calls, which return their first one."""
    seen = []

    def record(*a, **k):
        seen.append(a)
        return a[0]
    monkeypatch.setattr(dense, "experts_mlp", record)
    monkeypatch.setattr(dense, "glu_mlp", record)
    return seen


def tokens(T=3, dtype=torch.bfloat16):
    return torch.randn(T, D, generator=torch.Generator().manual_seed(T)).to(dtype)


def slots(T=3):
    return torch.zeros(T, 2, dtype=torch.int64), torch.ones(T, 2)


def test_a_copy_uses_its_own_parameters(calls):
    block = make_block("deepseek", "cpu")
    patch.patch_model(torch.nn.ModuleList([block]), fmt="dense")
    other = copy.deepcopy(block)
    for b in (block, other):
        b.experts(tokens(), *slots())
        b.shared_experts(tokens())
        e, m = b.experts, b.shared_experts
        used = [*calls[-2][3:5], *calls[-1][1:4]]
        assert all(p is q for p, q in zip(used, [e.gate_up_proj, e.down_proj, *(getattr(m, n).weight for n in ("gate_proj", "up_proj", "down_proj"))]))
    x = tokens(dtype=torch.float32)
    other.float()
    patch.unpatch_experts(other.shared_experts)
    with torch.no_grad():
        other.shared_experts.down_proj.weight.mul_(2)
        assert torch.equal(other.shared_experts(x), 2 * make_block("deepseek", "cpu").float().shared_experts(x))
    assert hasattr(block.shared_experts, "_moelab_state")


@pytest.mark.gpu
@pytest.mark.parametrize("part", ["experts", "shared_experts"])
def test_gradients_of_a_copy(part):
    """A copy trains its own parameters, as an average or a reference model made by copying does."""
    block = make_block("deepseek", "cuda")
    patch.patch_model(torch.nn.ModuleList([block]), fmt="dense")
    other = copy.deepcopy(block)
    args = (H.randn(5, D, dtype=torch.bfloat16),) + (() if part != "experts" else
                                                     (torch.tensor([[0, 1]] * 5, device="cuda"), torch.full((5, 2), 0.5, device="cuda")))
    y = getattr(block, part)(*args)
    with torch.no_grad():
        for p in getattr(other, part).parameters():
            p.mul_(0.5)
        assert not torch.equal(getattr(other, part)(*args), y)
    getattr(other, part)(*args).sum().backward()
    assert all(p.grad is not None for p in getattr(other, part).parameters()) and all(p.grad is None for p in block.parameters())


def test_a_second_patch_keeps_the_stock_forward(calls):
    """With other settings, say: the last one holds, and undoing it gives the stock forward."""
    e = make_block("mixtral", "cpu").experts
    stock, x = e.forward, tokens()
    want = e(x, *slots())
    patch.patch_dense(e, checkpoint=True)
    patch.patch_dense(e, checkpoint=False)
    assert e._moelab_state["checkpoint"] is False
    e(x, *slots())
    assert len(calls) == 1
    patch.unpatch_experts(e)
    assert e.forward == stock and torch.equal(e(x, *slots()), want) and len(calls) == 1
    assert not any(n.startswith("_moelab") for n in e.__dict__)


@pytest.mark.gpu
def test_patches_onto_4_bits_and_back():
    """patch_experts over patch_dense and the other way round, and patch_block twice."""
    block = make_block("mixtral", "cuda")
    e, stock = block.experts, block.experts.forward
    args = (H.randn(5, D, dtype=torch.bfloat16), torch.tensor([[0, 1]] * 5, device="cuda"), torch.full((5, 2), 0.5, device="cuda"))
    with torch.no_grad():
        for first, second in ((patch.patch_dense, patch.patch_experts), (patch.patch_experts, patch.patch_dense)):
            first(e)
            second(e)
            y = e(*args)
            patch.unpatch_experts(e)
            assert e.forward == stock
            second(e)
            assert torch.equal(e(*args), y)
            patch.unpatch_experts(e)
        stock = block.forward
        patch.patch_block(block)
        patch.patch_block(block)
        patch.unpatch_block(block)
        assert block.forward == stock and not any(n.startswith("_moelab") for n in block.__dict__)


@pytest.mark.parametrize("odd", ["gpt-oss", "biased shared experts", "another activation", "fp32"])
def test_a_refused_model_is_left_as_it_was(odd):
    blocks = [make_block("deepseek", "cpu"), make_block("gpt-oss" if odd == "gpt-oss" else "deepseek", "cpu")]
    if odd == "biased shared experts":
        blocks[1].shared_experts.up_proj.bias = torch.nn.Parameter(torch.zeros(512, dtype=torch.bfloat16))
    if odd == "another activation":
        blocks[1].shared_experts.act_fn = torch.nn.GELU()
    if odd == "fp32":
        blocks[1].experts.float()
    model = torch.nn.ModuleList(blocks)
    with pytest.raises((ValueError, TypeError, NotImplementedError)):
        patch.patch_model(model, fmt="dense")
    assert not any(n.startswith("_moelab") or n == "forward" for m in model.modules() for n in m.__dict__)
    assert patch.patch_model(model[:1], fmt="dense") == 2 and patch.patch_model(model[:1], fmt="dense") == 0


def test_shared_modules_count_once():
    block = make_block("mixtral", "cpu")
    other = make_block("mixtral", "cpu")
    other.experts = block.experts
    assert patch.patch_model(torch.nn.ModuleList([block, other]), fmt="dense") == 1


class Adapter(torch.nn.Module):
    """What a finetune puts in a projection's place: the frozen product and a low-rank one beside it, with the base's weight in view."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.a = torch.nn.Parameter(torch.ones(4, base.in_features, dtype=base.weight.dtype))
        self.b = torch.nn.Parameter(torch.ones(base.out_features, 4, dtype=base.weight.dtype))

    @property
    def weight(self):
        return self.base.weight

    bias = None

    def forward(self, x):
        return self.base(x) + x @ self.a.T @ self.b.T


class Scaled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_adapters_and_subclasses_run(calls, name):
    m, x = make_block("deepseek", "cpu").shared_experts, tokens()
    patch.patch_dense(m)
    assert m(x) is x and len(calls) == 1
    stock = copy.deepcopy(m)
    patch.unpatch_experts(stock)
    p = getattr(m, name)
    setattr(m, name, Adapter(p))
    setattr(stock, name, Adapter(getattr(stock, name)))
    assert torch.equal(m(x), stock(x)) and len(calls) == 1
    sub = Scaled(p.in_features, p.out_features, bias=False, dtype=p.weight.dtype)
    sub.weight = p.weight
    setattr(m, name, sub)
    setattr(stock, name, sub)
    assert torch.equal(m(x), stock(x)) and len(calls) == 1
    patch.unpatch_experts(m)
    with pytest.raises(ValueError, match="neither"):   # and when it is there before
        patch.patch_dense(m)
    setattr(m, name, p)
    patch.patch_dense(m)
    assert m(x) is x and len(calls) == 2
    p.bias = torch.nn.Parameter(torch.ones(p.out_features, dtype=p.weight.dtype))
    m(x)
    p.bias = None
    p.forward = lambda t: torch.nn.functional.linear(t, p.weight)   # an instance's own
    m(x)
    assert len(calls) == 2


@pytest.mark.parametrize("part", ["gate_proj", "up_proj", "down_proj", "act_fn"])
def test_hooks_run(calls, part):
    m, x, seen = make_block("deepseek", "cpu").shared_experts, tokens(), []
    patch.patch_dense(m)
    for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"):
        h = getattr(getattr(m, part), register)(lambda *a: seen.append(1))
        xs = x.clone().requires_grad_()
        m(xs).sum().backward()
        assert len(seen) == 1 and not calls, register
        h.remove()
        seen.clear()
    assert m(x) is x and len(calls) == 1   # and without hooks the kernels again


def test_another_activation_runs(calls):
    for m, args in ((make_block("mixtral", "cpu").experts, (tokens(), *slots())), (make_block("deepseek", "cpu").shared_experts, (tokens(),))):
        patch.patch_dense(m)
        n = len(calls)
        assert m(*args) is args[0] and len(calls) == n + 1
        act, m.act_fn = m.act_fn, torch.nn.GELU()
        y = m(*args)
        patch.unpatch_experts(m)
        assert torch.equal(m(*args), y) and len(calls) == n + 1
        m.act_fn = act
        patch.patch_dense(m)
        h = m.act_fn.register_forward_hook(lambda *a: None)
        m(*args)
        assert len(calls) == n + 1
        h.remove()
        assert copy.deepcopy(m)(*args) is args[0] and len(calls) == n + 2


def test_activations_keep_their_bits_unless_asked():
    """Fewer bits for the backward pass are the caller's choice."""
    blocks = torch.nn.ModuleList([make_block("deepseek", "cpu")])
    for want, opt in ((False, {}), (True, {"checkpoint": True}), (False, {"checkpoint": False})):
        patch.patch_model(blocks, fmt="dense", **opt)
        for m in (blocks[0].experts, blocks[0].shared_experts):
            assert m._moelab_state["checkpoint"] is want
            patch.unpatch_experts(m)
            assert patch.patch_dense(m, **opt)._moelab_state["checkpoint"] is want
            patch.unpatch_experts(m)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["mixtral", "olmoe"])
def test_default_gradients_against_the_stock_module(kind):
    """Of the stock module in 64 bits on the same routing. In 16 bits a gradient has at most four roundings on its way (kept gate/up
    values in two factors, an operand of its last product, itself): each moves a value by an error even in +-half a step, at most
    half_step / sqrt(3) of it in the mean square, together 2 half_step / sqrt(3) = 4.5e-3 in the norm. Kept in 8 bits it is 1e-2."""
    dt = torch.bfloat16
    e = make_block(kind, "cuda").experts
    E, T, k = e.down_proj.shape[0], 200, 2
    idx = torch.rand(T, E, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").topk(k, 1)[1]
    x, wts, dy = H.randn(T, D, dtype=dt), torch.softmax(H.randn(T, k, dtype=torch.float32, seed=1), 1), H.randn(T, D, dtype=dt, seed=2)
    ref = copy.deepcopy(e).cpu().double()
    a = [x.cpu().double().requires_grad_(), wts.cpu().double().requires_grad_()]
    want = torch.autograd.grad(ref(a[0], idx.cpu(), a[1]), [*a, ref.gate_up_proj, ref.down_proj], dy.cpu().double())
    patch.patch_dense(e)
    b = [x.requires_grad_(), wts.requires_grad_()]
    got = torch.autograd.grad(e(b[0], idx, b[1]), [*b, e.gate_up_proj, e.down_proj], dy)
    for name, g, w in zip(("dx", "dwts", "dw_gate_up", "dw_down"), got, want):
        assert float((g.cpu().double() - w).norm() / w.norm()) <= 2 * H.half_step(dt) / 3 ** 0.5, name


@pytest.mark.parametrize("how", ["pickle", "torch.save"])
def test_a_saved_module_loads(calls, how):
    """Patched, with its own parameters, and its stock forward behind it."""
    import io
    import pickle
    block = make_block("deepseek", "cpu")
    patch.patch_model(torch.nn.ModuleList([block]), fmt="dense", checkpoint=True)
    for m, args in ((block.experts, (tokens(), *slots())), (block.shared_experts, (tokens(),))):
        if how == "pickle":
            other = pickle.loads(pickle.dumps(m))
        else:
            f = io.BytesIO()
            torch.save(m, f)
            f.seek(0)
            other = torch.load(f, weights_only=False)   # written two lines above
        n = len(calls)
        assert other(*args) is args[0] and len(calls) == n + 1 and other._moelab_state["checkpoint"] is True
        w = other.down_proj if m is block.experts else other.down_proj.weight
        assert any(t is w for t in calls[-1])
        patch.unpatch_experts(other)
        stock = copy.deepcopy(m)
        patch.unpatch_experts(stock)
        assert torch.equal(other(*args), stock(*args)) and len(calls) == n + 1
