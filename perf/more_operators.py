"""Routing by scores and groups, and MXFP4: what is timed, the operators' plain forms, and what they must return.

Four operators, each a case's "op":
    route    router logits -> the k experts of each token and their weights: softmax or sigmoid scores, a bias that only
             ranks, groups of experts of which the best few are kept, weights renormalised or not; with train the gradient
             of the logits too
    quant    rows of numbers to MXFP4 (an E2M1 code each, an E8M0 exponent per 32 neighbours), returned as the values that
             the form stands for
    linear   one product of MXFP4 operands, x quantised in the call, with bias, activation and residual; with train its
             gradients (straight through the roundings), the weights then 16-bit ones that are quantised in the call too
    grouped  the same by expert with ragged sizes, x's rows read through the slot list; with train the gradients of x and
             the bias (the weights are frozen codes)

Sizes are the model shapes of the package's shapes.py, or generic ones. Activations are normal with channels of different
size, weights are codes and exponents as a checkpoint holds them, routing takes the k largest of random logits per token,
skew "zipf" adds a Zipf(1.1) popularity to them.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NONE, SILU, GELU = 0, 1, 2   # activations of linear


def _route(name, T, E, k, *, x="fp32", score="sigmoid", bias=True, groups=1, top_groups=1, by="max", norm=True, scale=1.0,
           train=False):
    c = dict(op="route", T=T, E=E, k=k, x=x, score=score, bias=bias, groups=groups, top_groups=top_groups, by=by, norm=norm,
             scale=scale, train=train)
    return c if name is None else dict(c, name=name)


def _quant(name, M, K, *, x="bf16"):
    c = dict(op="quant", M=M, K=K, x=x)
    return c if name is None else dict(c, name=name)


def _linear(name, T, N, K, *, x="bf16", bias=False, act=NONE, residual=False, train=False):
    c = dict(op="linear", T=T, N=N, K=K, x=x, bias=bias, act=act, residual=residual, train=train)
    return c if name is None else dict(c, name=name)


def _grouped(name, E, N, K, T, k, *, x="bf16", rows=True, bias=False, train=False, skew="uniform"):
    c = dict(op="grouped", E=E, N=N, K=K, T=T, k=k, x=x, rows=rows, bias=bias, train=train, skew=skew)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one token's router in a decode step: 256 experts in 8 groups, of which 4 count
        _route("route decode T1", 1, 256, 8, groups=8, top_groups=4, by="top2", scale=2.5),
        # the same router on a prefill chunk
        _route("route prefill T4096", 4096, 256, 8, groups=8, top_groups=4, by="top2", scale=2.5),
        # a training batch through a softmax router that is limited to 3 of 8 groups, an odd number of tokens, and its gradient
        _route("route train T8191", 8191, 64, 6, x="bf16", score="softmax", bias=False, groups=8, top_groups=3, norm=False,
               train=True),
        # a few tokens' activations before a product
        _quant("quant T5", 5, 2880),
        # a projection's weights when a model is quantised, and fp32 masters of a smaller one
        _quant("quant weights", 14336, 4096),
        _quant("quant fp32 masters", 5760, 2880, x="fp32"),
        # one token through a wide projection
        _linear("linear decode T1", 1, 14336, 4096, act=SILU),
        # a ragged prompt through a shared expert's down projection, everything in the epilogue
        _linear("linear prompt T237 fp16", 237, 2048, 2816, x="fp16", bias=True, act=GELU, residual=True),
        # a training step of a square projection
        _linear("linear train T4096", 4096, 4096, 4096, bias=True, act=SILU, residual=True, train=True),
        # one token's gate/up on 8 of 128 experts: a decode step
        _grouped("gate_up decode T1", 128, 1536, 2048, 1, 8),
        # gate/up of a prefill chunk, skewed experts
        _grouped("gate_up prefill T4096", 128, 1536, 2048, 4096, 8, skew="zipf"),
        # a finetune over frozen experts: forward, dx and the biases' gradients, an odd number of tokens
        _grouped("gate_up finetune T1111", 32, 5760, 2880, 1111, 4, rows=False, bias=True, train=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


#: Bounds on a drawn case: the largest listed one does 412e9 operations (linear train) and moves 1.4e9 bytes (finetune).
MAX_FLOPS, MAX_BYTES = 400e9, 1.3e9


def draw(rng):
    while True:
        op = rng.choice(["route", "route", "quant", "linear", "linear", "grouped", "grouped"])
        if op == "route":
            groups = rng.choice([1, 1, 2, 4, 8, 16])
            E = groups * rng.randint(2, max(2, min(512 // groups, 64)))
            live = rng.randint(1, groups)
            score, train = rng.choice(["softmax", "sigmoid"]), rng.random() < 0.4
            c = _route(None, _log(rng, 1, 8192), E, rng.randint(1, min(16, live * (E // groups))),
                       x=rng.choice(["fp32", "bf16", "fp16"]), score=score, bias=rng.random() < 0.5, groups=groups,
                       top_groups=live, by=rng.choice(["max", "top2"]), norm=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                       train=train)
        elif op == "quant":
            c = _quant(None, _log(rng, 1, 16384), 32 * _log(rng, 1, 256), x=rng.choice(["bf16", "fp16", "fp32"]))
        elif op == "linear":
            c = _linear(None, _log(rng, 1, 8192), 8 * _log(rng, 8, 1792), 32 * _log(rng, 2, 256), x=rng.choice(["bf16", "fp16"]),
                        bias=rng.random() < 0.5, act=rng.randint(0, 2), residual=rng.random() < 0.5, train=rng.random() < 0.4)
        else:
            c = _grouped(None, rng.choice([1, 3, 8, 16, 32, 60, 64, 128]), 8 * _log(rng, 8, 720), 32 * _log(rng, 2, 128),
                         _log(rng, 1, 4096), 1, x=rng.choice(["bf16", "fp16"]), bias=rng.random() < 0.4,
                         train=rng.random() < 0.3, skew=rng.choice(["uniform", "zipf"]))
            c["k"] = rng.randint(1, min(8, c["E"]))
            c["rows"] = not c["train"] and rng.random() < 0.7
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


# ------------------------------------------------------------------------------------------------------- inputs
def _ids(c, seed):
    """Expert ids [T, k]: the k largest of random logits."""
    r = np.random.default_rng(7919 * (seed + 1))
    lg = r.gumbel(size=(c["T"], c["E"]))
    if c["skew"] == "zipf":
        lg += r.permutation(np.log(np.arange(1, c["E"] + 1)) * -1.1)
    return np.argpartition(-lg, c["k"] - 1, axis=1)[:, :c["k"]].astype(np.int32)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(dtype)


def _activations(g, M, K, dtype):
    """Rows and channels of different size, as hidden states have them."""
    x = torch.randn((M, K), generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn((M, 1), generator=g, device=DEV))
    x *= torch.exp(0.7 * torch.randn((1, K), generator=g, device=DEV))
    return x.to(dtype)


def _codes(g, E, N, K):
    """Random weights as a checkpoint holds them: E2M1 codes, two to a byte, the low half first, [E, N, K / 2], and E8M0
    exponents [E, N, K / 32]; their size is about 1 / sqrt(K)."""
    codes = torch.randint(0, 256, (E, N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    e = 127 - 1 - int(round(math.log2(K) / 2))
    scales = torch.randint(e - 1, e + 1, (E, N, K // 32), generator=g, device=DEV, dtype=torch.uint8)
    return codes, scales


def prepare(case, seed):
    c, g, dt = case, _gen(seed), DT[case["x"]]
    s = {"c": c}
    if c["op"] == "route":
        s["logits"] = _normal(g, (c["T"], c["E"]), dt, 1.5)
        s["bias"] = _normal(g, (c["E"],), torch.float32, 0.05) if c["bias"] else None
        s["dw"] = _normal(g, (c["T"], c["k"]), torch.float32) if c["train"] else None
        s["leaves"] = [s["logits"]]
    elif c["op"] == "quant":
        s["x"] = _activations(g, c["M"], c["K"], dt)
        s["leaves"] = []
    elif c["op"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        s["x"] = _activations(g, T, K, dt)
        s["b"] = _normal(g, (N,), dt, 0.1) if c["bias"] else None
        s["r"] = _normal(g, (T, N), dt) if c["residual"] else None
        s["dy"] = _normal(g, (T, N), dt) if c["train"] else None
        if c["train"]:
            s["w"] = _normal(g, (N, K), dt, K ** -0.5)
            s["leaves"] = [s[n] for n in ("x", "w", "b") if s[n] is not None]
        else:
            s["codes"], s["scales"] = (t[0] for t in _codes(g, 1, N, K))
            s["leaves"] = []
    else:
        E, N, K, T, k = (c[n] for n in ("E", "N", "K", "T", "k"))
        ids = _ids(c, seed).reshape(-1)
        order = np.argsort(ids, kind="stable").astype(np.int32)
        counts = np.bincount(ids, minlength=E)
        s["counts"] = counts.tolist()   # the plain form's ranges; the kernels read the offsets
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).to(DEV)
        s["rows"] = torch.from_numpy(order // k).to(DEV) if c["rows"] else None
        s["x"] = _activations(g, T if c["rows"] else T * k, K, dt)
        s["codes"], s["scales"] = _codes(g, E, N, K)
        s["b"] = _normal(g, (E, N), dt, 0.1) if c["bias"] else None
        s["dy"] = _normal(g, (T * k, N), dt) if c["train"] else None
        s["leaves"] = [s[n] for n in ("x", "b") if s[n] is not None]
    if c.get("train"):
        for t in s["leaves"]:
            t.requires_grad_()
    if own and "codes" in s:   # the weights as a program that multiplies by them keeps them: laid out once
        s["w4"] = _package()[1].from_packed(s["codes"].view(torch.int32), s["scales"])
    return s


# --------------------------------------------------------------------------------------------------- plain forms
def _pow2(e):
    """2^e in fp32 for -126 <= e <= 127, from its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """fp32 [M, K] -> the fp32 values that its MXFP4 form stands for."""
    b = x.reshape(-1, 32)
    a = b.abs().amax(1, keepdim=True)
    e = ((a.view(torch.int32) >> 23) - 127 - 2).clamp(-126, 125)   # floor(log2 of the largest) - 2
    v = b * _pow2(-e)
    m = v.abs()
    # spacing of E2M1: 1/2 below 2, 1 below 4, 2 above; ties go to the even code
    q = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), 2 * torch.round(m / 2)))
    q = torch.copysign(q.clamp(max=6.0), v) * _pow2(e)
    return torch.where(a < 2.0 ** -124, torch.zeros_like(q), q).reshape(x.shape)


def _values(codes, scales):
    """fp32 values [..., K] of codes [..., K / 2] and exponents [..., K / 32]."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV)
    table = torch.cat([table, -table])
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1)
    return (v.reshape(*scales.shape, 32) * _pow2(scales.int() - 127)[..., None]).reshape(*codes.shape[:-1], -1)


def _gelu_parts(z):
    t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return t, math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)


def _plain_route(s):
    """In 64 bits: experts next to each other at the border of the choice differ by less than 32 bits keep."""
    c = s["c"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    l = s["logits"].detach().double()
    if c["score"] == "softmax":
        p = torch.exp(l - l.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-l))
    rank = l if s["bias"] is None else p + s["bias"].double()
    if G > 1:
        v = (p if s["bias"] is None and c["by"] == "top2" else rank).reshape(T, G, E // G).sort(2, descending=True)[0]
        v = v[:, :, 0] if c["by"] == "max" else v[:, :, 0] + v[:, :, 1]
        kept = v.sort(dim=1, descending=True, stable=True)[1][:, :c["top_groups"]]
        live = torch.zeros((T, G), dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        rank = torch.where(live.repeat_interleave(E // G, 1), rank, -math.inf)
    idx = rank.sort(dim=1, descending=True, stable=True)[1][:, :k]
    chosen = p.gather(1, idx)
    total = chosen.sum(1, keepdim=True) if c["norm"] else torch.ones_like(chosen[:, :1])
    w = c["scale"] * chosen / total
    out = (idx.to(torch.int32), w.float())
    if not c["train"]:
        return out
    dw = s["dw"].double()
    ds = c["scale"] * dw / total
    if c["norm"]:
        ds = ds - (ds * chosen).sum(1, keepdim=True) / total
    if c["score"] == "softmax":
        dl = -p * (ds * chosen).sum(1, keepdim=True)
        dl = dl.scatter_add(1, idx, chosen * ds)
    else:
        dl = torch.zeros_like(p).scatter(1, idx, ds * chosen * (1 - chosen))
    return *out, dl.to(s["logits"].dtype)


def _plain_quant(s):
    return (_quantised(s["x"].float()).to(s["x"].dtype),)


def _plain_linear(s):
    c, dt = s["c"], s["x"].dtype
    x = _quantised(s["x"].detach().float())
    w = _quantised(s["w"].detach().float()) if c["train"] else _values(s["codes"], s["scales"])
    z = x @ w.T
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    sg = 1 / (1 + torch.exp(-z)) if c["act"] == SILU else None
    t, tz = _gelu_parts(z) if c["act"] == GELU else (None, None)
    y = z * sg if c["act"] == SILU else 0.5 * z * (1 + t) if c["act"] == GELU else z
    if s["r"] is not None:
        y = y + s["r"].float()
    if not c["train"]:
        return (y.to(dt),)
    dz = s["dy"].float()
    if c["act"] == SILU:
        dz = dz * (sg + z * sg * (1 - sg))
    elif c["act"] == GELU:
        dz = dz * (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * tz)
    out = [y, dz @ w, dz.T @ x] + ([dz.sum(0)] if s["b"] is not None else [])
    return tuple(t.to(dt) for t in out)


def _plain_grouped(s):
    c, dt = s["c"], s["x"].dtype
    x = _quantised(s["x"].detach().float())
    x = x if s["rows"] is None else x[s["rows"].long()]
    dys = s["dy"].float().split(s["counts"]) if c["train"] else [None] * c["E"]
    y, dx, db = [], [], []
    for e, (a, dy) in enumerate(zip(x.split(s["counts"]), dys)):
        if len(a):
            w = _values(s["codes"][e], s["scales"][e])
            y.append(a @ w.T if s["b"] is None else a @ w.T + s["b"][e].detach().float())
            if c["train"]:
                dx.append(dy @ w)
        if c["train"]:
            db.append(dy.sum(0))
    out = [torch.cat(y)]
    if c["train"]:
        out += [torch.cat(dx)] + ([torch.stack(db)] if s["b"] is not None else [])
    return tuple(t.to(dt) for t in out)


# ------------------------------------------------------------------------------------------------- the operators
@functools.lru_cache(maxsize=None)
def _package():
    import importlib

    import __graft_entry__
    __graft_entry__.load_package()
    return [importlib.import_module("moelab_amd." + n) for n in ("router", "mx4")]


def _own(s):
    router, mx4 = _package()
    c = s["c"]
    if c["op"] == "route":
        idx, y = router.topk_scored(s["logits"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                                    top_groups=c["top_groups"], group_score=c["by"], norm=c["norm"], scale=c["scale"])
        if not c["train"]:
            return idx, y
        return idx, y.detach(), *torch.autograd.grad(y, s["leaves"], s["dw"])
    if c["op"] == "quant":
        return (mx4.dequantize(mx4.quantize(s["x"]), s["x"].dtype),)
    if c["op"] == "linear":
        y = mx4.linear(s["x"], s["w"] if c["train"] else s["w4"], bias=s["b"], act=c["act"], residual=s["r"])
    else:
        y = mx4.grouped_mm(s["x"], s["w4"], s["offsets"], bias=s["b"], rows=s["rows"])
    if not c["train"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"]))


PLAIN = {"route": _plain_route, "quant": _plain_quant, "linear": _plain_linear, "grouped": _plain_grouped}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["c"]["op"]](state)


# ----------------------------------------------------------------------------------------------------- the floor
def work(case):
    """Bytes that must move and operations that must be done: inputs once, outputs once; an MXFP4 operand is 17 bytes per 32
    values; experts without a row are not read."""
    c = case
    size = 4 if c["x"] == "fp32" else 2
    if c["op"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        nbytes = T * E * size + T * k * 8 + (4 * E if c["bias"] else 0)
        flops = 20.0 * T * E
        if c["train"]:   # + the weights' gradients, dlogits
            nbytes += T * k * 4 + T * E * size
    elif c["op"] == "quant":   # x -> the values
        nbytes, flops = c["M"] * c["K"] * 2.0 * size, 10.0 * c["M"] * c["K"]
    elif c["op"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        nbytes = 2.0 * (T * K + T * N * (1 + c["residual"]) + c["bias"] * N) + N * K * (2.0 if c["train"] else 17 / 32)
        flops = 2.0 * T * N * K
        if c["train"]:
            nbytes += 2.0 * (T * N + T * K + N * K + c["bias"] * N)
            flops *= 3
    else:
        E, N, K, T, k = (c[n] for n in ("E", "N", "K", "T", "k"))
        M, live = T * k, len(np.unique(_ids(c, 0)))
        nbytes = 2.0 * ((T if c["rows"] else M) * K + M * N + c["bias"] * live * N) + live * N * K * 17 / 32
        flops = 2.0 * M * N * K
        if c["train"]:   # + dy, dx and the biases' gradients
            nbytes += 2.0 * (M * N + M * K + c["bias"] * E * N)
            flops *= 2
    return {"bytes": float(nbytes), "flops": float(flops)}


# --------------------------------------------------------------------------------------------------- in 64 bits
def _nearest(x):
    """The MXFP4 values of x [M, K], by comparing with the borders between neighbouring values, in 64 bits."""
    b = x.detach().double().reshape(-1, 32)
    top = b.abs().max(1, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(torch.where(top == 0, torch.ones_like(top), top))) - 2)
    unit = torch.where(unit * 8 <= top, unit * 2, torch.where(unit * 4 > top, unit / 2, unit))   # should log2 have rounded
    r = b.abs() / unit
    # from the lower value to the next one at this border: on it the even code of the two wins
    up = ((r > 0.25).double() * 0.5 + (r >= 0.75).double() * 0.5 + (r > 1.25).double() * 0.5 + (r >= 1.75).double() * 0.5
          + (r > 2.5).double() + (r >= 3.5).double() + (r > 5.0).double() * 2)
    v = torch.sign(b) * up * unit
    return torch.where(top < 2.0 ** -124, torch.zeros_like(v), v).reshape(x.shape)


def _exact_values(codes, scales):
    lo, hi = (codes & 15).to(torch.int64), (codes >> 4).to(torch.int64)
    q = torch.stack([lo, hi], -1).flatten(-2)
    m = (q & 7).double()
    big = (2 + (q & 1)) * torch.exp2(torch.div(q & 7, 2, rounding_mode="floor").double() - 2)   # (1 + m / 2) 2^(e - 1)
    v = torch.where(m < 2, m / 2, big) * torch.where(q > 7, -1.0, 1.0)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _exact_act(act, z):
    """act(z) and its slope."""
    if act == NONE:
        return z, torch.ones_like(z)
    if act == SILU:
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    a, b = math.sqrt(2 / math.pi), 0.044715   # tanh form: z sigmoid(2 a (z + b z^3))
    s = torch.sigmoid(2 * a * (z + b * z ** 3))
    return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * b * z * z)


def _exact_route(s, c):
    T, E, G = c["T"], c["E"], c["groups"]
    n = E // G
    l = s["logits"].detach().double()
    p = torch.softmax(l, 1) if c["score"] == "softmax" else torch.sigmoid(l)
    key = l if s["bias"] is None else p + s["bias"].double()
    ids = torch.arange(E, device=DEV)
    dead = torch.zeros((T, E), dtype=torch.bool, device=DEV)
    if G > 1:
        val = key if c["by"] == "max" or s["bias"] is not None else p
        parts = val.reshape(T, G, n)
        first, at = parts.max(2)
        if c["by"] == "top2":
            first = first + parts.scatter(2, at.unsqueeze(2), -math.inf).max(2).values
        # a group is out if as many as top_groups others come before it
        before = (first.unsqueeze(1) > first.unsqueeze(2)) | ((first.unsqueeze(1) == first.unsqueeze(2))
                                                            & (torch.arange(G, device=DEV) < torch.arange(G, device=DEV)[:, None]))
        dead = (before.sum(2) >= c["top_groups"])[:, ids // n]
    left, picks = ~dead, []
    for _ in range(c["k"]):
        best = torch.where(left, key, -math.inf).max(1, keepdim=True).values
        pick = torch.where(left & (key == best), ids, E).min(1).values
        picks.append(pick)
        left = left & (ids != pick[:, None])
    idx = torch.stack(picks, 1)
    hit = torch.zeros_like(p).scatter(1, idx, 1.0)
    total = (p * hit).sum(1, keepdim=True) if c["norm"] else torch.ones_like(p[:, :1])
    out = (idx.to(torch.int32), (c["scale"] * p / total).gather(1, idx))
    if not c["train"]:
        return out
    g = torch.zeros_like(p).scatter(1, idx, s["dw"].double()) * c["scale"] / total   # by the scores, the total held
    if c["norm"]:
        g = (g - (g * p).sum(1, keepdim=True) / total) * hit
    dl = p * (g - (g * p).sum(1, keepdim=True)) if c["score"] == "softmax" else g * p * (1 - p)
    return *out, dl


@torch.no_grad()
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "route":
        return _exact_route(s, c)
    if c["op"] == "quant":
        return (_nearest(s["x"]),)
    x = _nearest(s["x"])
    if c["op"] == "linear":
        w = _nearest(s["w"]) if c["train"] else _exact_values(s["codes"], s["scales"])
        z = torch.mm(x, w.t()) + (0.0 if s["b"] is None else s["b"].double())
        y, slope = _exact_act(c["act"], z)
        y = y if s["r"] is None else y + s["r"].double()
        if not c["train"]:
            return (y,)
        dz = s["dy"].double() * slope
        return (y, torch.mm(dz, w), torch.mm(dz.t(), x)) + ((dz.sum(0),) if s["b"] is not None else ())
    x = x if s["rows"] is None else x[s["rows"].long()]
    y = torch.empty((len(x), c["N"]), dtype=torch.float64, device=DEV)
    dx, db = torch.empty_like(x), torch.zeros((c["E"], c["N"]), dtype=torch.float64, device=DEV)
    lo = 0
    for e, n in enumerate(s["counts"]):
        r = slice(lo, lo + n)
        lo += n
        if n:
            w = _exact_values(s["codes"][e], s["scales"][e])
            y[r] = torch.mm(x[r], w.t())
            if s["b"] is not None:
                y[r] += s["b"][e].double()
            if c["train"]:
                dx[r] = torch.mm(s["dy"][r].double(), w)
                db[e] = s["dy"][r].double().sum(0)
    if not c["train"]:
        return (y,)
    return (y, dx) + ((db,) if s["b"] is not None else ())
