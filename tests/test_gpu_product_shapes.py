"""The 16-bit products on every tile shape that their rules choose, and dense products split over their sums (linear.linear and
its gradients), element by element against 64-bit products: sums that end inside a part and inside a step, more rounds of
tiles than workgroups with a rest that is cut into pieces, uneven groups, operands of another stride, streams, graphs."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import _lib, grouped, linear
from test_gpu_grouped import reference as grouped_reference
from test_gpu_grouped import verify
from test_gpu_linear import act_of, make, reference

pytestmark = pytest.mark.gpu

# (T, N, K): few output tiles and long sums for the forward product, for dx, for dw; parts of one size and a shorter last one
SPLIT = [(5, 72, 4104), (9, 4104, 72), (5000, 72, 136), (64, 1032, 2056), (130, 520, 3080), (4999, 264, 520), (700, 264, 4104),
         (300, 2056, 1032), (12000, 520, 264)]


def _parts(T, N, K):
    L = _lib.lib()
    return [bool(f(T, N, K)) for f in (L.moe_linear_workspace_bytes, L.moe_linear_dx_workspace_bytes, L.moe_linear_dw_workspace_bytes)]


def test_the_sizes_are_split():
    seen = [_parts(*s) for s in SPLIT]
    assert all(any(p) for p in seen) and all(sum(p[i] for p in seen) >= 3 for i in range(3)), seen


@pytest.mark.parametrize("act", [linear.NONE, linear.SILU, linear.GELU])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K", SPLIT)
def test_split_forward(T, N, K, dtype, act):
    for bias, residual in ((True, True), (False, False)):
        x, w, b, r = make(T, N, K, dtype, bias, residual)
        z, mags, y, tol = reference(x, w, b, r, act)
        got = linear.linear(x, w, bias=b, act=act, residual=r)
        H.check(got, y, tol + H.half_step(dtype) * y.abs() + H.tiny(dtype))
        assert torch.equal(linear.linear(x, w, bias=b, act=act, residual=r), got)
        H.check(linear.linear(x, w, bias=b, act=act, residual=r, out_dtype=torch.float32), y, tol + 2.0 ** -23 * y.abs())
        _, kept = linear._forward(x, w, b, act, r, None, True)
        H.check(kept, z, H.product_tol(z, mags, K, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K", SPLIT)
def test_split_gradients(T, N, K, dtype):
    x, w, b, _ = make(T, N, K, dtype)
    dy = H.randn(T, N, dtype=dtype, seed=4)
    wide_x, wide_dy = torch.cat([x, x], 1)[:, K:], torch.cat([dy, dy], 1)[:, :N]
    out = []
    for xi, di in ((x, dy), (wide_x, dy), (x, wide_dy)):
        leaves = [t.clone().requires_grad_() if t.is_contiguous() else t.detach().requires_grad_() for t in (xi, w, b)]
        out.append(torch.autograd.grad(linear.linear(leaves[0], leaves[1], bias=leaves[2]), leaves, di))
    dx, dw, db = out[0]
    assert all(torch.equal(p, q) for o in out[1:] for p, q in zip(out[0], o))
    x, w, dy = x.double(), w.double(), dy.double()
    for got, ref, mags, R in ((dx, dy @ w, dy.abs() @ w.abs(), N), (dw, dy.T @ x, dy.abs().T @ x.abs(), T),
                              (db, dy.sum(0), dy.abs().sum(0), T)):
        H.check(got, ref, H.product_tol(ref, mags, R, dtype))


def test_split_keeps_infinities_in_their_rows():
    T, N, K = 64, 1032, 2056
    x, w, _, _ = make(T, N, K, torch.bfloat16, False, False)
    want = linear.linear(x, w)
    x[7, 2050], x[40, 3] = float("inf"), float("nan")
    got = linear.linear(x, w)
    rest = [t for t in range(T) if t not in (7, 40)]
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[40]).all() and not torch.isfinite(got[7]).any()


def test_split_on_streams_and_in_graphs():
    """Calls at once on several streams have workspaces of their own; a graph of a step replays with new inputs."""
    T, N, K = 130, 520, 3080
    xs = [H.randn(T, K, dtype=torch.bfloat16, seed=i) for i in range(4)]
    w, dy = H.randn(N, K, dtype=torch.bfloat16, scale=K ** -0.5), H.randn(T, N, dtype=torch.bfloat16, seed=9)

    def fn(x):
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = linear.linear(*leaves, act=linear.SILU)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = [fn(x) for x in xs]
    streams, got = [torch.cuda.Stream() for _ in xs], []
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(fn(x))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for a, b in zip(got, want) for p, q in zip(a, b))
    x = xs[0].clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            out = fn(x)
        graphs.append((graph, out))
    for i in range(4):
        x.copy_(xs[i])
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i])) and torch.equal(fn(x)[0], want[i][0])


# (slots per expert, N, K): for each rule of the forward product and dx, and each of dw's two shapes: up to 32 slots on average;
# few tiles; 128 and 256 rows; averages in 129 .. 192; long groups; more tiles than workgroups and a rest
GROUPS = [
    ([3, 60, 0, 33, 20, 1, 40, 31], 328, 520),
    ([90, 128, 129, 40, 100, 33, 65, 1], 520, 264),
    ([70, 250, 33, 128, 1, 190, 100, 127, 60, 129, 90, 65], 3336, 136),
    ([140, 150, 131, 190, 129, 170, 256, 133, 140, 64, 150, 160], 3336, 136),
    ([140, 150, 131, 190, 129, 170, 256, 133, 140, 64, 150, 160], 136, 5640),
    ([400, 513, 31, 700], 4104, 72),
    ([1300, 1025, 900, 1100, 1027, 1200], 1544, 1800),
]


@pytest.mark.parametrize("lists", [False, True], ids=["slots", "lists"])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K", GROUPS, ids=[f"{len(c)}x{sum(c)}-{n}-{k}" for c, n, k in GROUPS])
def test_grouped_shapes(counts, N, K, dtype, lists):
    E, M = len(counts), sum(counts)
    rows = torch.randint(0, 97, (M,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).int() if lists else None
    T = 97 if lists else M
    x, w = H.randn(T, K, dtype=dtype), H.randn(E, N, K, dtype=dtype, scale=K ** -0.5, seed=1)
    dy = H.randn(T, N, dtype=dtype, seed=3)
    off = H.offsets_of(counts)
    ref, mag = grouped_reference(counts, x, w, None, dy, rows)
    got = {"y": grouped.mm(x, w, off, rows=rows), "dx": grouped.mm_dx(dy, w, off, rows=rows)}
    got["dw"], got["db"] = grouped.mm_dw(dy, x, off, E, dy_rows=rows, x_rows=rows, bias=True)
    verify(counts, got, ref, mag, dtype)
    assert torch.equal(grouped.mm(x, w, off, rows=rows), got["y"]) and torch.equal(grouped.mm_dx(dy, w, off, rows=rows), got["dx"])


@pytest.mark.parametrize("K", [64, 4104])
def test_guard_rows_around_results(K):
    """Results written into the middle of a larger buffer: no byte around them changes, with pieces and whole rounds."""
    for counts in ([40] * 5, [300, 0, 129]):
        E, M, N = len(counts), sum(counts), 1032
        x, w = H.randn(M, K, dtype=torch.bfloat16), H.randn(E, N, K, dtype=torch.bfloat16, seed=1)
        off = H.offsets_of(counts)
        for fn, shape in ((lambda o: grouped.mm(x, w, off, out=o), (M, N)),
                          (lambda o: grouped.mm_dw(grouped.mm(x, w, off), x, off, E, out=o), (E, N, K))):
            n = torch.Size(shape).numel()
            buf = torch.full((n + 8192,), 7.0, dtype=torch.bfloat16, device=DEV)
            fn(buf[4096:4096 + n].view(shape))
            assert (buf[:4096] == 7).all() and (buf[4096 + n:] == 7).all()
