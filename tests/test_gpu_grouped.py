"""Grouped 16-bit products (grouped.mm, mm_dx, mm_dw) against 64-bit products, element by element: ragged groups, empty ones,
one slot, sizes off every tile, rows through index lists, strides, slots behind the last group, other streams, captured
calls, matrices past 32-bit offsets, and gradients."""
import pytest
import torch

import dense_helpers as H
from dense_helpers import DEV, TYPES
from moelab_amd import grouped

pytestmark = pytest.mark.gpu

# (slots per expert, N, K): one slot; few; sizes that end inside every tile and every step; many experts, most of them empty;
# the tiles of 64, 128 and 256 rows and their part tiles; one large group
CASES = [
    ([1], 8, 8),
    ([0, 1, 0], 64, 64),
    ([2, 3, 0, 1, 1], 72, 136),
    ([5], 264, 72),
    ([0] * 70 + [1] + [0] * 70 + [2, 1], 40, 520),
    ([17, 0, 33, 64, 1, 65], 200, 328),
    ([100, 30, 129, 0, 255], 136, 200),
    ([300, 513, 0, 31], 520, 264),
    ([40] * 60, 1032, 72),
    ([700], 2056, 136),
    ([1500, 20], 4104, 64),
]
IDS = [f"{len(c)}x{sum(c)}-{n}-{k}" for c, n, k in CASES]


def reference(counts, x, w, b, dy, rows=None):
    """y, dx, dw, db and the magnitudes that their error bounds need, in 64 bits."""
    x, w, dy = x.double(), w.double(), dy.double()
    if rows is not None:
        x, dy = x[rows.long()], dy[rows.long()]
    E, N, K = w.shape
    M = sum(counts)
    ref = {n: torch.zeros(s, dtype=torch.float64, device=DEV) for n, s in
           (("y", (M, N)), ("dx", (M, K)), ("dw", (E, N, K)), ("db", (E, N)))}
    mag = {n: torch.zeros_like(t) for n, t in ref.items()}
    for e, r in H.ranges(counts):
        for out, f in ((ref, lambda t: t), (mag, torch.abs)):
            out["y"][r] = f(x[r]) @ f(w[e]).T + (0 if b is None else f(b[e].double()))
            out["dx"][r] = f(dy[r]) @ f(w[e])
            out["dw"][e] = f(dy[r]).T @ f(x[r])
            out["db"][e] = f(dy[r]).sum(0)
    return ref, mag


def verify(counts, got, ref, mag, dtype):
    N, K = ref["dw"].shape[1:]
    for n, R in (("y", K), ("dx", N), ("dw", max(counts)), ("db", max(counts))):
        if n in got:
            H.check(got[n], ref[n], H.product_tol(ref[n], mag[n], R, dtype if got[n].dtype == dtype else torch.float32), n)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K", CASES, ids=IDS)
def test_products(counts, N, K, dtype):
    E, M = len(counts), sum(counts)
    x, w = H.randn(M, K, dtype=dtype), H.randn(E, N, K, dtype=dtype, scale=K ** -0.5, seed=1)
    b, dy = H.randn(E, N, dtype=dtype, seed=2), H.randn(M, N, dtype=dtype, seed=3)
    off = H.offsets_of(counts)
    ref, mag = reference(counts, x, w, b, dy)
    got = {"y": grouped.mm(x, w, off, bias=b), "dx": grouped.mm_dx(dy, w, off)}
    got["dw"], got["db"] = grouped.mm_dw(dy, x, off, E, bias=True)
    verify(counts, got, ref, mag, dtype)
    assert torch.equal(grouped.mm_dw(dy, x, off, E), got["dw"])


@pytest.mark.parametrize("counts,N,K", CASES, ids=IDS)
def test_products_to_fp32(counts, N, K):
    E, M = len(counts), sum(counts)
    x, w, dy = (H.randn(*s, dtype=torch.bfloat16, seed=i) for i, s in enumerate(((M, K), (E, N, K), (M, N))))
    off = H.offsets_of(counts)
    ref, mag = reference(counts, x, w, None, dy)
    f32 = dict(out_dtype=torch.float32)
    got = {"y": grouped.mm(x, w, off, **f32), "dx": grouped.mm_dx(dy, w, off, **f32), "dw": grouped.mm_dw(dy, x, off, E, **f32)}
    assert all(t.dtype == torch.float32 for t in got.values())
    verify(counts, got, ref, mag, torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K", CASES[2:], ids=IDS[2:])
def test_rows_through_lists(counts, N, K, dtype):
    """Repeated rows, every operand that can be indexed, and one operand indexed while the other is not."""
    E, M = len(counts), sum(counts)
    T = max(1, M // 3)
    g = torch.Generator().manual_seed(M)
    rows = torch.randint(0, T, (M,), generator=g).to(torch.int32).to(DEV)
    x, w = H.randn(T, K, dtype=dtype), H.randn(E, N, K, dtype=dtype, scale=K ** -0.5, seed=1)
    dy = H.randn(T, N, dtype=dtype, seed=3)
    off = H.offsets_of(counts)
    ref, mag = reference(counts, x, w, None, dy, rows)
    got = {"y": grouped.mm(x, w, off, rows=rows), "dx": grouped.mm_dx(dy, w, off, rows=rows)}
    got["dw"], got["db"] = grouped.mm_dw(dy, x, off, E, dy_rows=rows, x_rows=rows, bias=True)
    verify(counts, got, ref, mag, dtype)
    xs, ds = x[rows.long()], dy[rows.long()]
    for a, ar, b, br in ((dy, rows, xs, None), (ds, None, x, rows), (ds, None, xs, None)):
        assert torch.equal(grouped.mm_dw(a, b, off, E, dy_rows=ar, x_rows=br), got["dw"])
    assert torch.equal(grouped.mm(xs, w, off), got["y"]) and torch.equal(grouped.mm_dx(ds, w, off), got["dx"])


@pytest.mark.parametrize("counts", [[3, 2], [70, 90, 40], [600, 300]], ids=["few", "some", "many"])
def test_rows_outside_read_as_zeros(counts):
    """An index outside x, on either side: a row of zeros, and nothing read."""
    E, M, T, N, K = len(counts), sum(counts), 5, 64, 72
    x, w, dy = (H.randn(*s, dtype=torch.bfloat16, seed=i) for i, s in enumerate(((T, K), (E, N, K), (T, N))))
    rows = (torch.arange(M, device=DEV) % (T + 3) - 1).to(torch.int32)   # -1, 0 .. T - 1, T, T + 1
    rows[0], rows[-1] = -2 ** 31, 2 ** 31 - 1
    bad = (rows < 0) | (rows >= T)
    safe = torch.where(bad, 0, rows).long()
    off = H.offsets_of(counts)
    xs, ds = torch.where(bad[:, None], 0, x[safe]), torch.where(bad[:, None], 0, dy[safe])
    ref, mag = reference(counts, xs, w, None, ds)
    got = {"y": grouped.mm(x, w, off, rows=rows), "dx": grouped.mm_dx(dy, w, off, rows=rows),
           "dw": grouped.mm_dw(dy, x, off, E, dy_rows=rows, x_rows=rows)}
    verify(counts, got, ref, mag, torch.bfloat16)


@pytest.mark.parametrize("counts,tail", [([1, 0, 2], 3), ([40, 9], 70), ([300, 20], 600), ([0, 0], 5), ([0] * 8, 300)])
def test_slots_behind_the_last_group(counts, tail):
    """Zeros in a new result; left as they are in out=. The rows there may hold anything."""
    E, M, N, K = len(counts), sum(counts), 136, 72
    x, w, dy = (H.randn(*s, dtype=torch.bfloat16, seed=i) for i, s in enumerate(((M + tail, K), (E, N, K), (M + tail, N))))
    x[M:], dy[M:] = float("nan"), float("inf")
    off = H.offsets_of(counts)
    ref, mag = reference(counts, x[:M], w, None, dy[:M])
    for fn, arg, cols, name in ((grouped.mm, x, N, "y"), (grouped.mm_dx, dy, K, "dx")):
        for dt in (torch.bfloat16, torch.float32):
            y = fn(arg, w, off, out_dtype=dt)
            assert not y[M:].any()
            verify(counts, {name: y[:M]}, ref, mag, torch.bfloat16)
            out = torch.full((M + tail, cols), 7.0, dtype=dt, device=DEV)
            assert fn(arg, w, off, out=out) is out
            assert (out[M:] == 7).all() and torch.equal(out[:M], y[:M])
    dw, db = grouped.mm_dw(dy, x, off, E, bias=True)
    verify(counts, {"dw": dw, "db": db}, ref, mag, torch.bfloat16)


@pytest.mark.parametrize("n", [3, 90, 700])
def test_infinities_stay_in_their_rows(n):
    """An inf or NaN in one slot's row, or in one expert's weights, reaches no other slot and no other expert."""
    N, K = 72, 136
    x, w = H.randn(2 * n, K, dtype=torch.bfloat16), H.randn(2, N, K, dtype=torch.bfloat16, seed=1)
    off = H.offsets_of([n, n])
    clean = grouped.mm(x, w, off)
    x2, w2 = x.clone(), w.clone()
    x2[1, 5] = float("inf")
    x2[n - 1, K - 1] = float("nan")   # the last row of a part tile, the last value of a part step
    y = grouped.mm(x2, w, off)
    others = [i for i in range(2 * n) if i not in (1, n - 1)]
    assert torch.equal(y[others], clean[others]) and not torch.isfinite(y[1]).any() and torch.isnan(y[n - 1]).all()
    w2[1, N - 1, K - 1] = float("nan")
    y = grouped.mm(x, w2, off)
    assert torch.equal(y[:n], clean[:n]) and torch.equal(y[n:, :-1], clean[n:, :-1]) and torch.isnan(y[n:, -1]).all()
    dw = grouped.mm_dw(clean, x2, off, 2)
    assert torch.isfinite(dw[1]).all()


def test_strided_and_unaligned_operands():
    """A slice of a wider matrix is read in place; layouts that 16-byte pieces cannot read are copied; all give the same."""
    counts, N, K = [65, 3, 40], 72, 136
    M = sum(counts)
    off = H.offsets_of(counts)
    wide = H.randn(M, 2 * K + 16, dtype=torch.float16)
    w, dy = H.randn(3, N, K, dtype=torch.float16, seed=1), H.randn(M, N, dtype=torch.float16, seed=2)
    for x in (wide[:, 8:8 + K], wide[:, 3:3 + K], wide[:, :2 * K:2], wide[:, :K].T.contiguous().T):
        c = x.contiguous()
        assert torch.equal(grouped.mm(x, w, off), grouped.mm(c, w, off))
        assert torch.equal(grouped.mm_dw(dy, x, off, 3), grouped.mm_dw(dy, c, off, 3))
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(grouped.mm(wide[:, :K], wt, off), grouped.mm(wide[:, :K], w, off))
    ds = H.randn(M, 1, dtype=torch.float16).expand(M, N)
    assert torch.equal(grouped.mm_dx(ds, w, off), grouped.mm_dx(ds.contiguous(), w, off))


def test_bad_offsets_stay_inside():
    """Offsets past the slots or descending: nothing outside the matrices is read or written (guard rows stay), and groups
    whose offsets are sound come out right."""
    N, K, M = 64, 64, 40
    x, w = H.randn(M, K, dtype=torch.bfloat16), H.randn(4, N, K, dtype=torch.bfloat16, seed=1)
    off = torch.tensor([0, 10, 4, 2 ** 31 - 1, -5], dtype=torch.int32, device=DEV)
    guard = torch.full((M + 64, N), 3.0, dtype=torch.bfloat16, device=DEV)
    grouped.mm(x, w, off, out=guard[:M])
    assert (guard[M:] == 3).all()
    ref, mags = x[:4].double() @ w[0].double().T, x[:4].double().abs() @ w[0].double().abs().T
    H.check(guard[:4], ref, H.product_tol(ref, mags, K, torch.bfloat16))
    dw = grouped.mm_dw(H.randn(M, N, dtype=torch.bfloat16), x, off, 4)
    assert torch.isfinite(dw).all() and not dw[3].any()


def test_gradients():
    """mm's gradients are mm_dx and mm_dw of the incoming one; only those that are asked for come back; a broadcast incoming
    gradient; a second use of the same leaf adds up."""
    counts, N, K = [33, 0, 70, 2], 72, 136
    x, w, b = H.randn(105, K, dtype=torch.bfloat16), H.randn(4, N, K, dtype=torch.bfloat16, seed=1), H.randn(4, N, dtype=torch.bfloat16, seed=2)
    off = H.offsets_of(counts)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = grouped.mm(leaves[0], leaves[1], off, bias=leaves[2])
    assert torch.equal(y, grouped.mm(x, w, off, bias=b))
    dy = H.randn(105, N, dtype=torch.bfloat16, seed=3)
    got = torch.autograd.grad(y, leaves, dy)
    want = (grouped.mm_dx(dy, w, off), *grouped.mm_dw(dy, x, off, 4, bias=True))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    y = grouped.mm(x, leaves[1], off)
    y.sum().backward()
    ones = torch.ones_like(dy)
    assert leaves[0].grad is None and torch.equal(leaves[1].grad, grouped.mm_dw(ones, x, off, 4))
    y = grouped.mm(x, leaves[1], off, out_dtype=torch.float32)
    (g,) = torch.autograd.grad(y, leaves[1], dy.float())
    assert torch.equal(g, want[1])
    rows = torch.arange(105, device=DEV, dtype=torch.int32)
    (g,) = torch.autograd.grad(grouped.mm(x, leaves[1], off, rows=rows), leaves[1], dy)
    assert torch.equal(g, want[1])


def test_gradient_against_differences():
    """The product is linear in x and in w, so a difference of two results (fp32) is the gradient's product with the step but
    for the sums' roundings."""
    counts, N, K = [20, 45], 64, 72
    off = H.offsets_of(counts)
    x, w = H.randn(65, K, dtype=torch.bfloat16), H.randn(2, N, K, dtype=torch.bfloat16, seed=1)
    dy = H.randn(65, N, dtype=torch.bfloat16, seed=2)
    f = lambda x, w: grouped.mm(x, w, off, out_dtype=torch.float32).double()   # noqa: E731
    mags = float((f(x.abs(), w.abs()) * dy.double().abs()).sum())
    for i in range(2):
        args = [x, w]
        step = torch.zeros_like(args[i])
        step.view(-1)[::7] = 0.5
        up, dn = list(args), list(args)
        up[i], dn[i] = (args[i].double() + step.double()).to(torch.bfloat16), args[i]
        d = up[i].double() - dn[i].double()      # the step that bf16 leaves
        diff = float(((f(*up) - f(*dn)) * dy.double()).sum())
        grad = (grouped.mm_dx(dy, w, off, out_dtype=torch.float32) if i == 0 else
                grouped.mm_dw(dy, x, off, 2, out_dtype=torch.float32)).double()
        bound = 4 * (K + N + 65 + 8) * 2.0 ** -23 * (mags + float((grad.abs() * d.abs()).sum()))
        assert abs(diff - float((grad * d).sum())) <= bound, (i, diff, bound)


def test_calls_repeat_bit_for_bit_and_on_other_streams():
    counts, N, K = [100, 37, 300, 0, 5], 264, 200
    M = sum(counts)
    x, w, dy = (H.randn(*s, dtype=torch.float16, seed=i) for i, s in enumerate(((M, K), (5, N, K), (M, N))))
    off = H.offsets_of(counts)
    fns = (lambda: grouped.mm(x, w, off), lambda: grouped.mm_dx(dy, w, off), lambda: grouped.mm_dw(dy, x, off, 5))
    want = [f() for f in fns]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in fns]
    got = []
    for _ in range(3):
        for f, s in zip(fns, streams):
            with torch.cuda.stream(s):
                got.append(f())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))


@pytest.mark.parametrize("counts,N,K", [([1, 0, 1], 64, 200), ([100, 3, 61], 136, 72), ([700, 90], 520, 136)])
def test_captured_calls(counts, N, K):
    """Forward and backward products in a graph, replayed with new inputs and with eager calls between."""
    M, E = sum(counts), len(counts)
    x, w, dy = (H.randn(*s, dtype=torch.bfloat16, seed=i) for i, s in enumerate(((M, K), (E, N, K), (M, N))))
    off = H.offsets_of(counts)
    fn = lambda: (grouped.mm(x, w, off), grouped.mm_dx(dy, w, off), *grouped.mm_dw(dy, x, off, E, bias=True))   # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = fn()
    for i in range(3):
        x.copy_(H.randn(M, K, dtype=torch.bfloat16, seed=10 + i))
        off.copy_(H.offsets_of(counts[1:] + counts[:1]) if i == 1 else H.offsets_of(counts))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, fn()))


def test_no_slots():
    w = H.randn(3, 64, 72, dtype=torch.bfloat16)
    off = torch.zeros(4, dtype=torch.int32, device=DEV)
    x, dy = torch.empty(0, 72, dtype=torch.bfloat16, device=DEV), torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    assert grouped.mm(x, w, off).shape == (0, 64) and grouped.mm_dx(dy, w, off).shape == (0, 72)
    dw, db = grouped.mm_dw(dy, x, off, 3, bias=True)
    assert not dw.any() and not db.any() and dw.shape == w.shape


def _sampled(got, x, w, rows, dtype=torch.bfloat16):
    ref = x[rows].double() @ w.double().T
    mags = x[rows].double().abs() @ w.double().abs().T
    H.check(got[rows], ref, H.product_tol(ref, mags, x.shape[1], dtype))


def test_past_32_bit_offsets():
    """x of 4.9 GB (slots past 2^31 elements), read in place, and through a list where 32 bits do not reach (gathered first)."""
    M, K, N = 600_000, 4096, 8
    x = torch.empty(M, K, dtype=torch.bfloat16, device=DEV)
    for i in range(0, M, 100_000):
        x[i:i + 100_000] = H.randn(100_000, K, dtype=torch.bfloat16, seed=i)
    w = H.randn(2, N, K, dtype=torch.bfloat16, scale=K ** -0.5)
    n0 = M - 1000
    y = grouped.mm(x, w, H.offsets_of([n0, 1000]))
    far = torch.tensor([0, 262143, 262144, 524288, n0 - 1], device=DEV)
    _sampled(y, x, w[0], far)
    _sampled(y, x, w[1], torch.tensor([n0, M - 1], device=DEV))
    dw = grouped.mm_dw(y, x, H.offsets_of([n0, 1000]), 2)
    ref = y[n0:].double().T @ x[n0:].double()
    mags = y[n0:].double().abs().T @ x[n0:].double().abs()
    H.check(dw[1], ref, H.product_tol(ref, mags, 1000, torch.bfloat16))
    rows = torch.tensor([M - 1, 3, 524289, -1, M], dtype=torch.int32, device=DEV)
    y = grouped.mm(x, w, H.offsets_of([5, 0]), rows=rows)
    ref = x[rows[:3].long()].double() @ w[0].double().T
    H.check(y[:3], ref, H.product_tol(ref, x[rows[:3].long()].double().abs() @ w[0].double().abs().T, K, torch.bfloat16))
    assert not y[3:].any()


def test_weights_past_32_bit_offsets():
    E, N, K = 20, 16384, 8192   # 5.4 GB
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device=DEV)
    for e in range(E):
        w[e] = H.randn(N, K, dtype=torch.bfloat16, scale=K ** -0.5, seed=e)
    for counts in ([0] * (E - 1) + [2], [0] * (E - 2) + [90, 20]):
        M = sum(counts)
        x, dy = H.randn(M, K, dtype=torch.bfloat16), H.randn(M, N, dtype=torch.bfloat16, seed=1)
        off = H.offsets_of(counts)
        y, dx = grouped.mm(x, w, off), grouped.mm_dx(dy, w, off)
        for e, r in H.ranges(counts):
            if r.start < r.stop:
                _sampled(y[r], x[r], w[e], torch.tensor([0, r.stop - r.start - 1], device=DEV))
                ref, mags = dy[r].double() @ w[e].double(), dy[r].double().abs() @ w[e].double().abs()
                H.check(dx[r], ref, H.product_tol(ref, mags, N, torch.bfloat16))
