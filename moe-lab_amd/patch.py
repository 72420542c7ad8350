"""Torch MoE blocks onto the gfx950 kernels: the model-patch callers of the path (reference moelab/e2e.py:29-175
`patch` and its per-family variants, moelab/universal.py:26-56), for transformers' sparse MoE blocks.

Two levels, as in the reference:

* ``patch_block`` replaces a whole sparse MoE block's forward: the router runs inside the layer call
  (experts.run_routed: moe_layer_run / moe_layer_run_shared, the router's launches also group the slots) and the
  experts and shared experts on the kernels. Families (detected from the block's modules):
    - "stacked": Qwen3-MoE, Mixtral, OLMoE (``gate.weight`` [E, d]; ``experts.gate_up_proj`` [E, 2F, d], gate rows
      first, ``experts.down_proj`` [E, d, F]; SiLU or tanh-GELU GLU): softmax, top-k, renormalised when the router
      says so (reference e2e.py:57-64);
    - "qwen2-shared": the same plus Qwen-style gated shared expert, y + sigmoid(x . w_sg) * shared(x)
      (reference e2e.py:66-68);
    - "deepseek": DeepSeek-V2 ``DeepseekV2Moe``: greedy gate = full-softmax probabilities of the top-k times
      ``routed_scaling_factor`` (reference e2e.py:129-150: the fused router for greedy gates, the stock gate for
      group-limited ones), plus the shared experts added (e2e.py:146-147). Group-limited softmax gates, and sigmoid gates
      with a bias that ranks, run on router.route_scored if the gate's own forward does what that computes (and it is in
      bf16, without hooks or a forward put in its place); any other gate stays stock;
    - "gpt-oss": ``GptOssMLP``: router with bias, top-k of the logits, softmax over them; MXFP4 experts stored
      transposed with gate and up interleaved, per-expert biases, clamped SwiGLU (reference e2e.py:153-175); the
      forward returns (y, routing weights) as the stock one does.
  A block of the first three is taken for its family by what its own forward does with random tokens, experts aside (on the CPU): the
  weights that it gives its experts, and what it adds to their result. One that does something else (sigmoid scores, shared experts
  of another form, a norm in between) keeps its own forward, and only its experts run on the kernels.
  Shared experts whose width is S times the routed experts' are split into S experts of that width and merged into
  the routed set (one expert call per layer, experts.merge_shared); other widths run as a second call.
* ``patch_experts`` (the reference's SwitchGLU-level universal patch) replaces only an experts module's per-slot
  computation: every (token, expert) slot is a row of its own with weight 1 (run_slots, the per-slot GEMV without
  its k-reduction, at T = 1), and the routing weights and the sum over a token's slots are applied afterwards,
  outside the kernels, so the model's own router and any extra terms stay as they are.

* ``patch_dense`` puts the modules that hold the 16-bit weights, an experts module or a dense GLU MLP (a shared expert),
  on the unquantised kernels (dense.experts_mlp, dense.glu_mlp): their own parameters, nothing packed, and gradients
  to the parameters, the tokens and the routing weights, for a model that is trained or not quantised yet. With
  ``patch_model(model, fmt="dense")`` every sparse MoE block's experts and shared experts; routers stay stock.

The stock forwards are kept (``_moelab_stock_forward``); ``unpatch_block`` / ``unpatch_experts`` restore them.
``load_dequantised`` writes the state's dequantised weights back into the stock modules, so stock and patched
forwards then differ by arithmetic only, not by quantisation.
"""
import copy
import functools
import math

import torch

from . import _lib, dense, router
from .experts import merge_shared, run_experts, run_layer, run_routed
from .variants import hip_mxfp4_moe, hip_q4_moe

_FMT = {"int4": hip_q4_moe, "mxfp4": hip_mxfp4_moe}


def _stacked(e):
    """Experts stored as stacked tensors gate_up [E, 2F, d] (gate rows first) and down [E, d, F], no biases."""
    return (e is not None and isinstance(getattr(e, "gate_up_proj", None), torch.Tensor)
            and isinstance(getattr(e, "down_proj", None), torch.Tensor) and getattr(e, "gate_up_proj_bias", None) is None
            and e.gate_up_proj.dim() == 3 and e.down_proj.dim() == 3
            and e.gate_up_proj.shape[1] == 2 * e.down_proj.shape[2] and e.gate_up_proj.shape[2] == e.down_proj.shape[1])


def block_kind(m):
    """The family of a transformers sparse MoE block, or None."""
    e = getattr(m, "experts", None)
    router = getattr(m, "router", None)
    if (router is not None and e is not None and isinstance(getattr(e, "gate_up_proj_bias", None), torch.Tensor)
            and isinstance(getattr(router, "bias", None), torch.Tensor)):
        return "gpt-oss"
    gate = getattr(m, "gate", None)
    if gate is None or not isinstance(getattr(gate, "weight", None), torch.Tensor) or not _stacked(e):
        return None
    if getattr(m, "shared_experts", None) is not None and hasattr(gate, "routed_scaling_factor"):
        return "deepseek"
    if getattr(m, "shared_expert", None) is not None and getattr(m, "shared_expert_gate", None) is not None:
        return "qwen2-shared"
    return "stacked"


def is_moe_block(m):
    return block_kind(m) is not None


def _act(act, z):
    """The kernels' SiLU or tanh-GELU."""
    return z * torch.sigmoid(z if act == _lib.ACT_SWIGLU else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _bare(module):
    """A copy of a small module on the CPU, without hooks."""
    c = copy.deepcopy(module).cpu()
    for m in c.modules():
        for n in _HOOKS:
            getattr(m, n).clear()
    return c


def _own_forwards(module):
    """The module, its parts' own forwards in place of those put there (which can compute with the modules that this one is a copy of)."""
    for m in module.modules():
        m.__dict__.pop("forward", None)
    return module


def _shell(module, without):
    """A module's class and another module of it, on the CPU: its settings, buffers and children, without hooks, without the children
    `without` and without its own parameters. Its forward is the class's own."""
    cls = torch.nn.utils.parametrize.type_before_parametrizations(module)
    m = cls.__new__(cls)
    torch.nn.Module.__init__(m)
    kept = {n: _bare(c) for n, c in module._modules.items() if n not in (*without, "parametrizations")}
    own = {n: v for n, v in module.__dict__.items() if n not in m.__dict__}
    m.__dict__.update({n: v for n, v in own.items() if n not in ("forward", "_moelab_stock_forward")})
    m._buffers, m._modules = dict(module._buffers), kept
    return cls, m


def _act_of(module, tol=1e-3):
    """The GLU of a module with this act_fn, which may differ from the kernels' function by tol: by default as far as the exact
    GELU does from the tanh form (4.7e-4, below what 4-bit weights do to a layer), but not as far as a function of another kind
    with a similar name (QuickGELU 2e-2, Hardswish 0.14)."""
    fn = getattr(module, "act_fn", None)
    name = type(fn).__name__.lower()
    for k, v in (("silu", _lib.ACT_SWIGLU), ("swish", _lib.ACT_SWIGLU), ("gelu", _lib.ACT_GEGLU)):
        if k in name:
            z = torch.linspace(-12, 12, 4097, dtype=torch.float64, device="cpu")
            if isinstance(fn, torch.nn.Module):
                fn = _bare(fn)
            with torch.no_grad():
                gap = float((fn(z) - _act(v, z)).abs().max())
            if gap <= tol:
                return v
            name += f", {gap:.1e} off"
            break
    raise NotImplementedError(f"activation {name}: the kernels take SiLU, tanh-GELU or gpt-oss's clamped GLU")


def _quantise(fmt, gate, up, down):
    """Dense gate/up [E, F, d], down [E, d, F] -> a packed state of the format."""
    return _FMT[fmt].prepare(gate.contiguous(), up.contiguous(), down.contiguous())


def _mlp_as_experts(mlp, F):
    """A dense GLU MLP (gate_proj/up_proj [Fs, d], down_proj [d, Fs]) as S = Fs / F experts of width F:
    (gate [S, F, d], up [S, F, d], down [S, d, F]); the GLU acts elementwise, so the S experts' sum is the MLP."""
    g, u, dn = mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight
    Fs, d = g.shape
    S = Fs // F
    return g.reshape(S, F, d), u.reshape(S, F, d), dn.reshape(d, S, F).permute(1, 0, 2)


@torch.no_grad()
def block_state(block, fmt=None):
    """The block's packed state and call settings: {"kind", "state", "k", "norm", "scale", "act", "bias",
    "stock_gate", "scored"} (stock_gate: route by itself, not inside the layer call; scored: router.route_scored's settings,
    or None: with the block's own gate). kind: block_kind's, or "own" for a block whose own forward does not route and add up as its
    kind does: it runs, and only its experts are packed."""
    kind = block_kind(block)
    if kind is None:
        raise ValueError(f"{type(block).__name__}: not a sparse MoE block this patch knows")
    cfg = {"kind": kind, "scale": 1.0, "bias": None, "stock_gate": False, "scored": None}
    if kind == "gpt-oss":
        _check_gptoss(block)
        e, r = block.experts, block.router
        gu = e.gate_up_proj                       # [E, d, 2F], columns gate, up, gate, up, ...
        s = _quantise(fmt or "mxfp4", gu[..., ::2].transpose(1, 2), gu[..., 1::2].transpose(1, 2),
                      e.down_proj.transpose(1, 2))
        s["bg"] = e.gate_up_proj_bias[:, ::2].float().contiguous()
        s["bu"] = e.gate_up_proj_bias[:, 1::2].float().contiguous()
        s["bd"] = e.down_proj_bias.float().contiguous()
        s["wr"] = r.weight.detach().to(torch.bfloat16).contiguous()
        cfg.update(state=s, k=int(r.top_k), norm=True, act=_lib.ACT_GPTOSS, bias=r.bias.detach().float().contiguous())
        return cfg
    e, gate = block.experts, block.gate
    F = e.gate_up_proj.shape[1] // 2
    fmt = fmt or "int4"
    cfg.update(act=_glu_of(e), **_routing(block, kind))
    s = _quantise(fmt, e.gate_up_proj[:, :F], e.gate_up_proj[:, F:], e.down_proj)
    s["wr"] = gate.weight.detach().to(torch.bfloat16).contiguous()
    shared = None
    if cfg["kind"] == "deepseek":
        shared = block.shared_experts
    elif cfg["kind"] == "qwen2-shared":
        shared = block.shared_expert
        s["shared_gate"] = block.shared_expert_gate.weight.detach().reshape(-1).to(torch.bfloat16).contiguous()
    if shared is not None:
        Fs = shared.gate_proj.weight.shape[0]
        if Fs % F == 0 and Fs // F + cfg["k"] <= 64:   # S experts of the routed width: merged, one call per layer
            s["shared"] = _quantise(fmt, *_mlp_as_experts(shared, F))
            s = merge_shared(s)
        else:                                          # one shared expert of its own width, a second call
            s["shared"] = _quantise(fmt, *(t.unsqueeze(0) for t in (shared.gate_proj.weight, shared.up_proj.weight,
                                                                   shared.down_proj.weight)))
    cfg["state"] = s
    return cfg


def _glu_of(experts):
    """The activation of a stacked experts module that computes the plain GLU layer: as near as _act_of takes its function for it."""
    act = _act_of(experts)
    E, d, F = experts.down_proj.shape
    _check_glu(experts, act, True, d, F, E, least=1e-2, train=False)
    return act


@torch.no_grad()
def _check_gptoss(block):
    """Raises where the block's own forward, run with experts of 32 x 32 random numbers, is not the clamped layer of the kernels with
    gate and up interleaved. (Modules that cannot be run at another size than their own are taken by their parameters.)"""
    e, T = block.experts, 8
    E, d, F = e.gate_up_proj.shape[0], e.gate_up_proj.shape[1], e.gate_up_proj.shape[2] // 2
    g = torch.Generator("cpu").manual_seed(0)

    def rand(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cpu") * scale

    def small(module, names, params):
        cls, m = _shell(module, names)
        m.__dict__.update({n: 64 if v == 2 * F and v != d else 32 for n, v in m.__dict__.items()
                           if type(v) is int and v in (d, F, 2 * F) and n != "num_experts"})
        m._parameters = {n: torch.nn.Parameter(v, requires_grad=False) for n, v in params.items()}
        return cls, m.eval()
    w, b, k = rand(E, 32, scale=0.5), rand(E), int(block.router.top_k)
    gu, gb, dn, db = rand(E, 32, 64), rand(E, 64), rand(E, 32, 32), rand(E, 32)
    try:
        with torch.device("cpu"):   # whatever the program's default device is
            cls, m = small(block, ("router", "experts"), {})
            m._modules["router"] = small(block.router, (), dict(weight=w, bias=b))[1]
            m._modules["experts"] = small(e, (), dict(gate_up_proj=gu, gate_up_proj_bias=gb, down_proj=dn, down_proj_bias=db))[1]
            x = rand(T, 32)
            got = cls.forward(m, x[None].clone())[0].reshape(T, 32)
    except Exception:
        return
    top, ids = (x @ w.T + b).topk(k, 1)
    z = torch.einsum("td,tkdf->tkf", x, gu[ids]) + gb[ids]
    gate, up = z[..., ::2].clamp(max=7.0), z[..., 1::2].clamp(-7.0, 7.0)
    h = gate * torch.sigmoid(1.702 * gate) * (up + 1)
    y = ((torch.einsum("tkf,tkfd->tkd", h, dn[ids]) + db[ids]) * torch.softmax(top, 1)[..., None]).sum(1)
    gap = float((got - y).abs().max() / y.abs().max())
    if not gap <= 1e-3:
        raise ValueError(f"{type(block).__name__} computes something else than the kernels' clamped layer with its gate and up "
                         f"interleaved (off by {gap:.1e} on random weights)")


class _Heard(torch.nn.Module):
    """Stands for a block's experts or shared experts: returns the numbers y and keeps what it is called with."""

    def __init__(self, y):
        super().__init__()
        self.y, self.calls = y, []

    def forward(self, *args, **kw):
        self.calls.append((*args, *kw.values()))
        return self.y.reshape(args[0].shape)


@torch.no_grad()
def _listen(block, kind, seed):
    """What a block's own forward does with random tokens, on the CPU in fp32: the tokens x [T, d], its router's weight [E, d], the
    weights [T, E] that it gives its experts and their number k, and whether it returns the experts' result and what its kind adds,
    of these tokens, and nothing else. Raises where it does not call its experts with tokens, ids and weights once."""
    E, d = block.experts.gate_up_proj.shape[0], block.experts.gate_up_proj.shape[2]
    g, T = torch.Generator("cpu").manual_seed(seed), 32

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cpu")
    names = [n for n in ("experts", "shared_experts", "shared_expert") if getattr(block, n, None) is not None]
    cls, m = _shell(block, names)
    for n, b in m._buffers.items():
        m._buffers[n] = b if b is None else b.detach().cpu()
    m._parameters = {n: None if p is None else torch.nn.Parameter(p.detach().cpu(), requires_grad=False)
                     for n, p in block._parameters.items()}
    heard = {n: _Heard(rand(T, d)) for n in names}
    m._modules.update(heard)
    _own_forwards(m).float().eval()
    weight, x = m.gate.weight.detach(), rand(T, d)
    spread = float((x @ weight.T).std())
    x *= 2 / spread if 0 < spread < math.inf else 1.0   # logits as far apart as a trained router's
    out = cls.forward(m, x[None].clone())
    ((tokens, idx, wts),) = heard["experts"].calls
    k = idx.shape[1]
    if (tokens.shape != x.shape or idx.shape != (T, k) or wts.shape != (T, k) or idx.is_floating_point()
            or not 0 <= int(idx.min()) <= int(idx.max()) < E):
        raise ValueError(f"experts called with {tuple(tokens.shape)}, {tuple(idx.shape)}, {tuple(wts.shape)}")
    want = heard["experts"].y
    same = torch.equal(tokens.float(), x)
    shared = {"deepseek": "shared_experts", "qwen2-shared": "shared_expert"}.get(kind)
    if shared:
        y, (call,) = heard[shared].y, heard[shared].calls
        same = same and len(call) == 1 and torch.equal(call[0].reshape(x.shape).float(), x)
        want = want + (y if kind == "deepseek" else torch.sigmoid(x @ m.shared_expert_gate.weight.T) * y)
    same = same and isinstance(out, torch.Tensor) and out.shape == (1, T, d) and bool(((out[0] - want).abs() <= 1e-4).all())
    return x, weight, torch.zeros((T, E), dtype=torch.float64, device="cpu").scatter_add(1, idx.long(), wts.double()), k, same


@torch.no_grad()
def _routing(block, kind):
    """The settings with which a block of this kind routes, by its own forward: the fused router's softmax top-k, route_scored's, the
    block's gate by itself, or (kind "own") all of the block."""
    gate = block.gate
    cfg = dict(kind=kind, norm=kind != "deepseek" and bool(getattr(gate, "norm_topk_prob", True)),
               scale=float(gate.routed_scaling_factor) if kind == "deepseek" else 1.0)
    with torch.device("cpu"):   # whatever the program's default device is
        try:
            heard = [_listen(block, kind, seed) for seed in (0, 1)]
        except Exception as e:
            raise NotImplementedError(f"{type(block).__name__} does not call its experts as the kernels take it ({type(e).__name__}: "
                                      f"{e}); patch_experts leaves all of the block but the experts as it is") from e
        cfg["k"] = heard[0][3]

        def is_it(weights):
            """Whether the block gave its experts these weights, for one set of tokens at least: two experts' scores can be equal in
            fp32."""
            for x, w, got, _, same in heard:
                try:
                    want = weights(x, w)
                    if same and got.shape == want.shape and float((got - want).abs().max()) <= 1e-4 * float(want.max()):
                        return True
                except Exception:   # another gate's result: no such experts, no such tuple
                    pass
            return False

        def softmax(norm):
            return is_it(lambda x, w: _scored_weights(x, w, cfg["k"], "softmax", None, 1, 1, "max", norm, cfg["scale"]))

        def own_gate(x, w):
            out = _own_forwards(_bare(gate)).float()(x)
            return torch.zeros((len(x), w.shape[0]), dtype=torch.float64).scatter_add(1, out[2].long(), out[1].double())
        for norm in (cfg["norm"], not cfg["norm"]):   # (kinds of one name are not all alike in it)
            if softmax(norm):
                return cfg | dict(norm=norm)
        if kind == "deepseek":
            cfg["stock_gate"], cfg["scored"] = True, _scored_settings(gate, cfg["k"])
            bias = _choice_bias(gate)
            if cfg["scored"] is not None and is_it(
                    lambda x, w: _scored_weights(x, w, cfg["k"], bias=None if bias is None else bias.cpu(), **cfg["scored"])):
                _bias_fits(cfg, gate)
                cfg["scored_for"] = _gate_settings(gate)
                return cfg
            cfg["scored"] = None
            if is_it(own_gate):
                return cfg
    return cfg | dict(kind="own", stock_gate=False)


def _choice_bias(gate):
    """The bias [E] that a sigmoid gate adds to its scores to choose by, or None."""
    b = getattr(gate, "e_score_correction_bias", None)
    return b if isinstance(b, torch.Tensor) else None


def _scored_weights(x, weight, k, score, bias, groups, top_groups, group_score, norm, scale):
    """router.topk_scored in plain 64-bit form, as weights [T, E] (0 for experts that are not chosen)."""
    logits = x.double() @ weight.double().T
    T, E = logits.shape
    p = torch.softmax(logits, 1) if score == "softmax" else torch.sigmoid(logits)
    c = p if bias is None else p + bias.double()
    top = c.reshape(T, groups, -1).topk(1 if group_score == "max" else 2, dim=2).values.sum(2)
    kept = torch.zeros_like(top).scatter(1, top.topk(top_groups, dim=1).indices, 1).bool().repeat_interleave(E // groups, 1)
    idx = torch.where(kept, c, -math.inf).topk(k, dim=1).indices
    w = p.gather(1, idx)
    w = scale * (w / w.sum(1, keepdim=True) if norm else w)
    return torch.zeros_like(p).scatter(1, idx, w)


@torch.no_grad()
def _scored_settings(gate, k):
    """topk_scored's settings for a gate that it computes, without the bias, else None: checked on the gate's own forward, on
    random tokens on the CPU. Where groups are masked, with all scores and biases negative together as well: a gate that masks the
    other groups with 0, not with -inf, then chooses an expert there, and stays stock. So a gate that is taken chooses alike whatever
    becomes of its bias; one whose bias has a negative element now stays stock as well (_bias_fits)."""
    bias = _choice_bias(gate)
    groups, top = int(getattr(gate, "num_group", 1) or 1), int(getattr(gate, "topk_group", 1) or 1)
    if bias is None:
        kw = dict(score="softmax", group_score="max", norm=False)
    else:
        kw = dict(score="sigmoid", group_score="top2", norm=bool(getattr(gate, "norm_topk_prob", True)))
    kw |= dict(groups=groups, top_groups=top, scale=float(gate.routed_scaling_factor))
    try:
        router._scored(gate.weight.shape[0], k, kw["score"], None, groups, top, kw["group_score"], kw["norm"], kw["scale"], None)
        if bias is not None and top < groups and float(bias.min()) < 0:
            return None
        g = _own_forwards(_bare(gate)).float()

        def alike(seed):
            x = torch.randn((64, g.weight.shape[1]), generator=torch.Generator("cpu").manual_seed(seed), device="cpu")
            x *= 2 / float((x @ g.weight.T).std())   # logits as far apart as a trained router's
            out = g(x)
            got = torch.zeros((64, g.weight.shape[0]), dtype=torch.float64, device="cpu").scatter(1, out[2].long(), out[1].double())
            want = _scored_weights(x, g.weight, k, bias=_choice_bias(g), **kw)
            return float((got - want).abs().max()) <= 1e-4 * float(want.max())
        if not (alike(0) or alike(1)):   # (two experts' scores can be equal in fp32)
            return None
        if bias is not None and top < groups:
            _choice_bias(g).sub_(float(bias.max()) + 1.5)
            if not (alike(0) or alike(1)):
                return None
    except Exception:   # whatever a gate of another kind makes of these tokens
        return None
    return kw


def _gate_settings(gate):
    get = gate.__dict__.get   # (a module's own lookup takes a microsecond for each that it lacks)
    return get("top_k"), get("num_group"), get("topk_group"), get("norm_topk_prob"), get("routed_scaling_factor")


def _bias_fits(cfg, gate):
    """Whether route_scored takes the gate's place with the bias as it is: not with a negative element while groups are masked. Looked
    at again only after the bias changed; while a graph is captured, or where changes leave no trace, a bias that has changed means
    the stock gate. (A change that goes unseen, through .data or between a graph's replays, does no harm: _scored_settings.)"""
    bias, kw = _choice_bias(gate), cfg["scored"]
    if bias is None or kw["top_groups"] == kw["groups"]:
        return True
    seen = None if bias.is_inference() else (bias.data_ptr(), bias._version)
    if cfg.get("bias_seen", 0) != seen or seen is None:
        if seen is None or (bias.is_cuda and torch.cuda.is_current_stream_capturing()):
            return False
        cfg["bias_fits"], cfg["bias_seen"] = float(bias.detach().min()) >= 0, seen
    return cfg["bias_fits"]


def _route_stock(block, hidden):
    """The block's own gate on the tokens: (idx int32 [T, k], wts fp32 [T, k])."""
    out = block.gate(hidden)
    wts, idx = out[1], out[2]
    return idx.to(torch.int32).contiguous(), wts.float().contiguous()


def _install(module, forward, state):
    """The patched forward and its state; a second patch keeps the stock forward of the first."""
    if not hasattr(module, "_moelab_stock_forward"):
        module._moelab_stock_forward = module.forward
    module._moelab_state = state
    module.forward = forward
    return module


def patch_block(block, fmt=None):
    """Replace a sparse MoE block's forward by the kernels (router inside the layer call). fmt: "int4" (default for
    the stacked families) or "mxfp4" (default for gpt-oss)."""
    cfg = block_state(block, fmt)
    s = cfg["state"]
    if cfg["kind"] == "own":
        def experts(hidden_states, top_k_index, top_k_weights):
            x = hidden_states.to(torch.bfloat16).contiguous()
            y = run_experts(s, x, top_k_index.to(torch.int32).contiguous(), top_k_weights.float().contiguous(), act=cfg["act"],
                            out_dtype=None if hidden_states.dtype == torch.bfloat16 else torch.float32)
            return y.to(hidden_states.dtype)
        block._moelab_cfg = cfg
        _install(block.experts, experts, s)
        return _install(block, getattr(block, "_moelab_stock_forward", block.forward), s)

    def forward(hidden_states):
        shape = hidden_states.shape
        x = hidden_states.reshape(-1, shape[-1]).to(torch.bfloat16).contiguous()
        gate = getattr(block, "gate", None)
        if (cfg["scored"] is not None and hidden_states.dtype == gate.weight.dtype == torch.bfloat16 and not _hooked(gate)
                and "forward" not in gate.__dict__ and _gate_settings(gate) == cfg["scored_for"] and _bias_fits(cfg, gate)):
            # the gate's own weight and bias, as they are now, in the settings it was checked with; in other types it computes with
            # more digits than bf16 has
            idx, wts = router.route_scored(x.detach(), gate.weight.detach(), cfg["k"], bias=_choice_bias(gate), **cfg["scored"])
            y = run_layer(s, x, idx, wts, act=cfg["act"])
        elif cfg["stock_gate"]:
            idx, wts = _route_stock(block, hidden_states.reshape(-1, shape[-1]))
            y = run_layer(s, x, idx, wts, act=cfg["act"])
        else:
            y, idx, wts = run_routed(s, x, s["wr"], cfg["k"], bias=cfg["bias"], norm=cfg["norm"], scale=cfg["scale"],
                                     act=cfg["act"])
        y = y.to(hidden_states.dtype).reshape(shape)
        if cfg["kind"] == "gpt-oss":
            return y, wts.to(hidden_states.dtype)
        return y

    block._moelab_cfg = cfg
    return _install(block, forward, s)


def unpatch_block(block):
    if block._moelab_cfg["kind"] == "own":
        unpatch_experts(block.experts)
    block.forward = block._moelab_stock_forward
    del block._moelab_stock_forward, block._moelab_state, block._moelab_cfg
    return block


def patch_experts(experts, fmt="int4"):
    """Universal patch of a stacked experts module (forward(hidden_states [T, d], top_k_index [T, k],
    top_k_weights [T, k]) -> [T, d]): the kernels compute each (token, expert) slot as a row of its own with weight
    1 (T = 1: run_slots, the per-slot GEMV without its k-reduction; T > 1: the T*k slots as rows with k = 1), and
    the routing weights and the sum over each token's k slots are applied afterwards in fp32 (reference
    universal.py:26-56: only the per-slot compute is replaced, the model keeps its routing and weighting)."""
    if not _stacked(experts):
        raise ValueError(f"{type(experts).__name__}: not a stacked experts module")
    F = experts.gate_up_proj.shape[1] // 2
    act = _glu_of(experts)
    with torch.no_grad():
        s = _quantise(fmt, experts.gate_up_proj[:, :F], experts.gate_up_proj[:, F:], experts.down_proj)

    def forward(hidden_states, top_k_index, top_k_weights):
        T, d = hidden_states.shape
        k = top_k_index.shape[-1]
        x = hidden_states.to(torch.bfloat16).contiguous()
        idx = top_k_index.to(torch.int32).contiguous()
        if T == 1:
            ones = torch.ones((1, k), dtype=torch.float32, device=x.device)
            slots = run_experts(s, x, idx, ones, act=act, path=_lib.PATH_SLOTS, nored=True, out_dtype=torch.float32)
        else:
            rows = x.repeat_interleave(k, dim=0)
            ones = torch.ones((T * k, 1), dtype=torch.float32, device=x.device)
            slots = run_experts(s, rows, idx.reshape(T * k, 1), ones, act=act, out_dtype=torch.float32)
        y = (slots.reshape(T, k, d) * top_k_weights.float().reshape(T, k, 1)).sum(1)
        return y.to(hidden_states.dtype)

    return _install(experts, forward, s)


def unpatch_experts(experts):
    experts.forward = experts._moelab_stock_forward
    del experts._moelab_stock_forward, experts._moelab_state
    return experts


_PROJ = ("gate_proj", "up_proj", "down_proj")


def _plain_linear(x):
    """Whether x multiplies by its weight and does nothing else (a subclass with a forward of its own, as of 4-bit weights or
    adapters, does)."""
    return (isinstance(x, torch.nn.Linear) and x.bias is None and "forward" not in x.__dict__
            and type(x).forward is torch.nn.Linear.forward)


def _glu_linears(m):
    """The gate, up and down weights of a dense GLU MLP without biases, or None."""
    ls = [getattr(m, n, None) for n in _PROJ]
    return [x.weight for x in ls] if all(_plain_linear(x) for x in ls) and hasattr(m, "act_fn") else None


def _hooked(x):
    return any(getattr(x, n, None) for n in _HOOKS)


def _probe(module, d, F, E, dtype, act, train=True):
    """The largest error of a module's own forward against the plain GLU layer, relative to the magnitudes that its sums add,
    on small random weights in its parameters' place (E None: a dense GLU MLP). Gates reach the hundreds, so that a clamp shows;
    routing weights are not 1, so that a weight at another place does."""
    g = torch.Generator("cpu").manual_seed(0)

    def rand(*shape):
        return torch.randn(shape, generator=g, dtype=torch.float64, device="cpu").to(dtype)
    scales = torch.tensor([0.25, 2.0, 8.0] if dtype.itemsize == 2 else [0.25, 2.0, 16.0, 128.0], device="cpu")
    x = rand(4 * len(scales), d) * scales.repeat(4)[:, None].to(dtype)
    names = ("gate_up_proj", "down_proj") if E else ("gate_proj", "up_proj", "down_proj")
    cls, m = _shell(module, names)
    if E:
        n = E if F <= 32 else 1   # at the module's own sizes its experts are one and the same
        gu, dn = rand(n, 2 * F, d).expand(E, 2 * F, d), rand(n, d, F).expand(E, d, F)
        m._parameters = {n: torch.nn.Parameter(t, requires_grad=False) for n, t in zip(names, (gu, dn))}
        k = min(2, E)
        idx = torch.stack([torch.randperm(E, generator=g, device="cpu")[:k] for _ in range(len(x))])
        wts = (torch.rand(len(x), k, generator=g, device="cpu") + 0.3).to(dtype)
        args = (x, idx, wts)
    else:
        for n, t in zip(names, (rand(F, d), rand(F, d), rand(d, F))):
            m._modules[n] = torch.nn.Linear(t.shape[1], t.shape[0], bias=False, device="meta", dtype=dtype)
            m._modules[n].weight = torch.nn.Parameter(t, requires_grad=False)
        gu = torch.cat([m.gate_proj.weight, m.up_proj.weight])[None]
        dn = m.down_proj.weight[None]
        idx, wts = torch.zeros(len(x), 1, dtype=torch.int64, device="cpu"), torch.ones(len(x), 1, device="cpu")
        args = (x,)
    got = cls.forward(m.train(train), *args)   # in training a dropout shows too
    if E:
        # ids past the experts: most forwards raise, some skip them as the kernels do, some take the last expert instead; but
        # some have experts without weights there
        try:
            past = cls.forward(m, x, torch.full_like(idx, E), wts)
        except (IndexError, RuntimeError):
            past = torch.zeros_like(x)
        if past.any() and not torch.equal(past, cls.forward(m, x, torch.full_like(idx, E - 1), wts)):
            return math.inf
    ref, mags = torch.zeros(2, len(x), d, dtype=torch.float64, device="cpu")
    for t in range(len(x)):
        for j in range(idx.shape[1]):
            e = int(idx[t, j])
            z = gu[e].double() @ x[t].double()
            h = wts[t, j].double() * _act(act, z[:F]) * z[F:]
            ref[t] += dn[e].double() @ h
            mags[t] += dn[e].double().abs() @ h.abs()
    return float(((got.double() - ref).abs() / mags).max())   # a NaN or another shape fails too


def _check_glu(module, act, stacked, d, F, E, least=0.0, train=True):
    """Raises unless the module's own forward, in training or not, is the plain GLU layer that the kernels compute (least: a difference
    that passes in every type)."""
    tried = []
    own = (module.down_proj if stacked else module.down_proj.weight).dtype
    for size in ((16, 32), (d, F)):   # some forwards know their sizes
        for dtype, tol in ((torch.float64, 1e-6), (torch.float32, 1e-4), (own, 0.05)):
            try:
                with torch.no_grad(), torch.device("cpu"):   # whatever the program's default device is
                    gap = _probe(module, *size, E if stacked else None, dtype, act, train)
            except Exception as e:   # a type or a size that this forward does not take
                tried.append(f"{type(e).__name__}: {e}")
                continue
            if gap <= max(tol, least):
                return
            raise ValueError(f"{type(module).__name__} computes something else than the plain GLU layer of the kernels (off by "
                             f"{gap:.1e} of its sums on random weights): a clamp, another gate or other routing weights")
    raise ValueError(f"{type(module).__name__}: its forward could not be checked against the kernels' GLU layer ({tried[0]})")


# patch_dense's forwards are bound to their module by a partial call: a deep copy of a patched module computes with its own
# parameters, and a saved one loads (a bound method would be looked up in the module when it loads). The kernels call none of
# the module's parts, so where one would do more than it did when the module was patched (a hook on it, an adapter or another
# module in its place), the stock forward runs.
def _experts_forward(self, hidden_states, top_k_index, top_k_weights):
    s = self._moelab_state
    if self.act_fn is not s["act_fn"] or _hooked(self.act_fn):
        return self._moelab_stock_forward(hidden_states, top_k_index, top_k_weights)
    return dense.experts_mlp(hidden_states, top_k_index, top_k_weights, self.gate_up_proj, self.down_proj, act=s["act"],
                             checkpoint=s["checkpoint"])


def _mlp_forward(self, x):
    s = self._moelab_state
    parts = [getattr(self, n) for n in _PROJ]
    if self.act_fn is not s["act_fn"] or _hooked(self.act_fn) or not all(_plain_linear(p) and not _hooked(p) for p in parts):
        return self._moelab_stock_forward(x)
    return dense.glu_mlp(x, *(p.weight for p in parts), act=s["act"], checkpoint=s["checkpoint"])


def _dense_act(module):
    """The activation of a module that patch_dense takes; raises for any other."""
    stacked, glu = _stacked(module), _glu_linears(module)
    if not stacked and glu is None:
        raise ValueError(f"{type(module).__name__}: neither a stacked experts module nor a GLU MLP without biases")
    act = _act_of(module, 1e-6)
    ws = (module.gate_up_proj, module.down_proj) if stacked else glu
    if any(w.dtype != ws[0].dtype or w.dtype not in (torch.bfloat16, torch.float16) for w in ws):
        raise TypeError(f"weights in {', '.join(sorted({str(w.dtype) for w in ws}))}: all bf16 or all fp16 expected")
    d, F = (ws[1].shape[1], ws[1].shape[2]) if stacked else (ws[0].shape[1], ws[0].shape[0])
    _lib.multiple_of(d, 8, "the hidden size")
    _lib.multiple_of(F, 32, "the intermediate size")
    _check_glu(module, act, stacked, d, F, ws[1].shape[0])
    return act


def _install_dense(module, act, checkpoint):
    return _install(module, functools.partial(_experts_forward if _stacked(module) else _mlp_forward, module),
                    {"fmt": "dense", "act": act, "act_fn": module.act_fn, "checkpoint": checkpoint})


def patch_dense(module, checkpoint=False):
    """Put a stacked experts module (forward(hidden_states [T, d], top_k_index [T, k], top_k_weights [T, k])) or a dense
    GLU MLP (gate_proj, up_proj, down_proj, act_fn) on the 16-bit kernels, forward and backward, with the module's own
    bf16 or fp16 parameters. checkpoint: activations are kept in 8 bits for the backward pass, not in 16: about half the memory,
    and gradients that are about 1% off in place of 0.3% (bf16) or 0.04% (fp16). unpatch_experts undoes it.
    A module whose forward computes anything else (clamped gates, exact GELU, QuickGELU, dropout) is refused: its forward is
    run on a few random rows and small random weights on the CPU, and compared. While a projection or the activation has
    hooks or another module in its place, the stock forward runs."""
    return _install_dense(module, _dense_act(module), checkpoint)


def _patch_model_dense(model, universal, checkpoint):
    """All parts are checked before the first is patched: a model that is refused is left as it was."""
    parts = {}
    for m in model.modules():
        if hasattr(m, "_moelab_state"):
            continue
        if universal:
            found = [m] if _stacked(m) else []
        else:
            found = [m.experts, getattr(m, "shared_expert", None), getattr(m, "shared_experts", None)] if is_moe_block(m) else []
        parts |= {id(p): p for p in found if p is not None and not hasattr(p, "_moelab_state")}
    acts = [_dense_act(p) for p in parts.values()]
    for p, act in zip(parts.values(), acts):
        _install_dense(p, act, checkpoint)
    return len(parts)


def patch_model(model, fmt=None, universal=False, checkpoint=False):
    """Patch every sparse MoE block of a model (universal: every stacked experts module instead); returns how many
    modules were patched. fmt "dense": patch_dense (with checkpoint) on each block's experts and shared experts
    (universal: on every stacked experts module); if it refuses one of them, none is patched."""
    if fmt == "dense":
        return _patch_model_dense(model, universal, checkpoint)
    n = 0
    for m in list(model.modules()):
        if hasattr(m, "_moelab_state"):
            continue
        if universal:
            if _stacked(m) and not hasattr(m, "gate_up_proj_bias"):
                patch_experts(m, fmt or "int4")
                n += 1
        elif is_moe_block(m):
            patch_block(m, fmt)
            n += 1
    return n


def _deq(s):
    mod = hip_q4_moe if s["fmt"] == "int4" else hip_mxfp4_moe
    return mod.dequant(s)


@torch.no_grad()
def load_dequantised(module):
    """Write the patched module's dequantised weights back into its stock modules (experts, shared experts), so
    stock and patched forwards see the same weights."""
    s = module._moelab_state
    if s["fmt"] == "dense":
        raise ValueError("patch_dense packs nothing: the stock modules hold the weights it runs on")
    cfg = getattr(module, "_moelab_cfg", {"kind": "experts"})
    wg, wu, wd = _deq(s)
    kind = cfg["kind"]
    if kind == "experts":
        e = module
    else:
        e = module.experts
    if kind == "gpt-oss":
        gu = e.gate_up_proj
        gu[..., ::2].copy_(wg.transpose(1, 2).to(gu.dtype))
        gu[..., 1::2].copy_(wu.transpose(1, 2).to(gu.dtype))
        e.down_proj.copy_(wd.transpose(1, 2).to(e.down_proj.dtype))
        return
    E = e.gate_up_proj.shape[0]
    e.gate_up_proj.copy_(torch.cat([wg[:E], wu[:E]], dim=1).to(e.gate_up_proj.dtype))
    e.down_proj.copy_(wd[:E].to(e.down_proj.dtype))
    shared = module.shared_experts if kind == "deepseek" else (module.shared_expert if kind == "qwen2-shared" else None)
    if shared is None:
        return
    if "n_shared" in s:   # merged: experts E .. E + S - 1
        sg, su, sd = wg[E:], wu[E:], wd[E:]
    else:
        sg, su, sd = _deq(s["shared"])
    S, F, d = sg.shape
    shared.gate_proj.weight.copy_(sg.reshape(S * F, d).to(shared.gate_proj.weight.dtype))
    shared.up_proj.weight.copy_(su.reshape(S * F, d).to(shared.up_proj.weight.dtype))
    shared.down_proj.weight.copy_(sd.permute(1, 0, 2).reshape(d, S * F).to(shared.down_proj.weight.dtype))
