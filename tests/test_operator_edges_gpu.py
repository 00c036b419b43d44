"""GPU: calls of the batched operators at the borders of their kernels' ranges - odd strides beside NaN, results in place,
captured graphs of every form, two streams at once, very many models, sizes where the form changes.  Tolerances are those
of test_dense_gpu.py and test_muon_gpu.py."""
import pytest
import torch

from mplc import dense, muon
from test_dense_gpu import check_backward, check_forward, live_rows, reference_forward
from test_muon_gpu import TYPES, close, rand, reference_step

pytestmark = pytest.mark.gpu


def framed(shape, t, seed, left, right):
    """Random matrices as views into rows whose other columns are NaN: (the rows, the view)."""
    G, m, n = shape
    rows = torch.full((G, m, left + n + right), float("nan"), dtype=t, device="cuda")
    view = rows[:, :, left:left + n]
    view.copy_(rand(shape, t, seed))
    return rows, view


# no short side of 4: the general form; 4 and 5: the first of the narrow one; 64, 65, 128, 129: where its width changes
LONG = [(5000, 1), (5000, 2), (5001, 3), (5001, 4), (5003, 5), (1, 5003), (2, 5001), (3, 5000), (4, 5003), (5, 7001),
        (1001, 64), (64, 1003), (1003, 65), (65, 1001), (701, 128), (128, 703), (703, 129), (129, 701)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("size", LONG, ids=lambda s: "x".join(map(str, s)))
def test_long_matrices_beside_nan_and_in_place(size, dtype):
    t = TYPES[dtype]
    rows, g = framed((3,) + size, t, sum(size), 3, 2)
    keep = g.clone()
    out = muon.orthogonalize(g)
    for i in range(3):
        close(out[i], keep[i])
    assert torch.equal(g, keep)
    muon.orthogonalize(g, out=g)
    assert torch.equal(g, out) and rows[:, :, :3].isnan().all() and rows[:, :, -2:].isnan().all()


@pytest.mark.parametrize("size", [(2, 5001, 3), (2, 3, 5002), (2, 5001, 70), (2, 70, 5001), (2, 301, 203), (2, 203, 301), (2, 61, 35)])
def test_steps_beside_nan(size):
    (wr, w), (mr, m) = framed(size, torch.float32, 1, 1, 3), framed(size, torch.float32, 2, 5, 1)
    _, g = framed(size, torch.bfloat16, 3, 1, 2)
    rw, rm, tol = reference_step(w, g, m, 0.02, 0.95, True, 0.1, 1.5)
    muon.muon_step(w, g, m, lr=0.02, weight_decay=0.1, scale=1.5)
    assert ((m.double() - rm).abs() <= 2.0 ** -23 * (rm.abs() + 4)).all()
    for i in range(size[0]):
        err = float(torch.linalg.vector_norm(w[i].double() - rw[i]))
        assert err <= tol[i] + 2.0 ** -22 * float(torch.linalg.vector_norm(rw[i]))
    assert wr[:, :, 0].isnan().all() and wr[:, :, -3:].isnan().all()
    assert mr[:, :, :5].isnan().all() and mr[:, :, -1].isnan().all()


@pytest.mark.parametrize("size", [(20, 12), (900, 20), (20, 900), (150, 140)])
def test_extreme_scales(size):
    """The same matrix times a power of two, values near the ends of fp32's range included, gives the same bits."""
    g = rand((2,) + size, seed=9).clamp(-4, 4)
    g = torch.where(g.abs() < 2.0 ** -10, 2.0 ** -10, g)
    want = muon.orthogonalize(g)
    for e in (-110, 120):
        assert torch.equal(muon.orthogonalize(g * 2.0 ** e), want)
    mixed = g.clone()  # one value far above the rest, at the end: what was summed before is scaled down
    mixed[:, -1, -1] = 2.0 ** 40
    out = muon.orthogonalize(mixed)
    for i in range(2):
        close(out[i], mixed[i])


@pytest.mark.parametrize("size", [(3000, 9, 5), (700, 700, 5), (700, 5, 700)])
def test_very_many_models(size):
    g = rand(size, seed=4)
    out = muon.orthogonalize(g)
    for i in (0, 1, 255, 256, size[0] - 1):
        close(out[i], g[i])
    w = rand((size[0], 40, 5), seed=5)
    x = rand((size[0], 3, 40), seed=6)
    _, pre = check_forward(x, w, act="silu")
    check_backward(rand((size[0], 3, 5), seed=7), x, w, pre, "silu")


# one workgroup per matrix with much LDS; narrow, of both directions; general
@pytest.mark.parametrize("size", [(2, 300, 60), (2, 2000, 48), (2, 100, 1500), (2, 400, 300)])
def test_every_form_replays(size):
    w, m, g = rand(size, seed=1), rand(size, seed=2), rand(size, seed=3)
    start = (w.clone(), m.clone())
    graph = torch.cuda.CUDAGraph()
    muon.muon_step(w.clone(), g, m.clone(), lr=0.05)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        muon.muon_step(w, g, m, lr=0.05)
        o = muon.orthogonalize(g)
    we, me = (t.clone() for t in start)
    for k in range(3):
        g.copy_(rand(size, seed=30 + k))
        graph.replay()
        torch.cuda.synchronize()
        muon.muon_step(we, g, me, lr=0.05)
        assert torch.equal(w, we) and torch.equal(m, me) and torch.equal(o, muon.orthogonalize(g))


def test_two_streams_at_once():
    """Two calls of one shape, with workspaces, in flight together."""
    gs = [rand((2, 900, 300), seed=i) for i in range(2)]
    xs = [rand((2, 40, 5000), torch.bfloat16, 10 + i) for i in range(2)]
    w = rand((2, 5000, 70), torch.bfloat16, 3, 0.02)
    want = [(muon.orthogonalize(g), dense.dense_forward(x, w, activation="gelu")) for g, x in zip(gs, xs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = (muon.orthogonalize(gs[i]), dense.dense_forward(xs[i], w, activation="gelu"))
    torch.cuda.synchronize()
    for a, c in zip(want, got):
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_plans_follow_values_not_objects():
    """Coefficients in a tensor that changes between two calls."""
    g = rand((1, 40, 200), seed=1)
    coef = torch.tensor([1.5, -0.5, 0.0])
    close(muon.orthogonalize(g, steps=3, coefficients=coef)[0], g[0], 3, (1.5, -0.5, 0.0))
    coef.copy_(torch.tensor([1.875, -1.25, 0.375]))
    close(muon.orthogonalize(g, steps=3, coefficients=coef)[0], g[0], 3, (1.875, -1.25, 0.375))
    for steps in (2.5, "5", None):
        with pytest.raises((TypeError, ValueError)):
            muon.orthogonalize(g, steps=steps)


# the largest tile and its short-sum form with operands that no 16-byte load takes, split sums of few columns, an input that
# ends inside a tile
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("size,left", [((1, 600, 512, 520), 1), ((3, 300, 64, 512), 3), ((2, 20, 4000, 3), 1), ((2, 20, 4000, 2), 0),
                                       ((1, 9, 6000, 1), 1), ((4, 257, 40, 8), 8), ((1, 512, 512, 512), 8)])
def test_products_beside_nan(size, left, dtype):
    G, B, K, N = size
    t = TYPES[dtype]
    _, x = framed((G, B, K), t, 1, left, 2)
    rows, w = framed((G, K, N), t, 2, left, 1)
    w.mul_(K ** -0.5)
    _, r = framed((G, B, N), t, 3, left, 1)
    outs, out = framed((G, B, N), t, 4, left, 1)
    b = rand((G, N), t, 5)
    pre = torch.empty(G, B, N, device="cuda")
    dense.dense_forward(x, w, b, residual=r, activation="gelu", preact=pre, out=out)
    z, y, ez, ey = reference_forward(x, w, b, r, "gelu", None)
    assert ((out.double() - y).abs() <= ey).all() and ((pre.double() - z).abs() <= ez).all()
    assert outs[:, :, :left].isnan().all() and outs[:, :, -1].isnan().all()
    dxs, dx = framed((G, B, K), t, 6, left, 1)
    check_backward(rand((G, B, N), t, 7), x, w, pre, "gelu", dx=dx)
    assert dxs[:, :, :left].isnan().all() and dxs[:, :, -1].isnan().all()


@pytest.mark.parametrize("rows", [1, 8])
def test_few_rows_of_idle_and_many_models(rows):
    """No model has a row, every model has one, and more models than workgroups fit at a time."""
    t = torch.float16
    x, w = rand((70, rows, 300), t, 1), rand((70, 300, 259), t, 2, 0.05)
    for n in (0, 1, -4, 99):
        counts = torch.full((70,), n, dtype=torch.int32, device="cuda")
        out, pre = check_forward(torch.where(live_rows(70, rows, counts), x, float("nan")), w, act="silu", counts=counts)
        if n <= 0:
            assert (out == 7).all() and (pre == 9).all()


def test_long_batch_of_one_column():
    """More blocks of rows than a grid's second axis has places."""
    B = 65536 * 64 + 5
    x, w = rand((1, B, 1), seed=1), rand((1, 1, 1), seed=2)
    dout, pre = rand((1, B, 1), seed=3), torch.empty(1, B, 1, device="cuda")
    dense.dense_forward(x, w, activation="relu", preact=pre)
    dx, dw, db = dense.dense_backward(dout, x, w, preact=pre, activation="relu")
    d = torch.where(x.double() * w.double() > 0, dout.double(), 0.0)
    assert torch.equal(dx, torch.where(pre > 0, dout, 0.0) * w)
    # db: sums of 64 values, joined in order; dw: the bound of any order
    for got, terms, roundings in ((dw, x.double() * d, B + 4), (db, d, B // 64 + 68)):
        assert abs(float(got) - float(terms.sum())) <= roundings * 2.0 ** -23 * float(terms.abs().sum())


def padded(x):
    """x behind a row that ends in NaN, in rows of whole 16-byte chunks plus a NaN."""
    G, m, n = x.shape
    rows = torch.full((G, m, (n + 15) // 8 * 8), float("nan"), dtype=x.dtype, device="cuda")
    rows[:, :, :n] = x
    return rows[:, :, :n]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("K,N", [(1001, 1003), (1001, 1000), (1008, 1003)])
def test_large_products_of_cut_rows(K, N, dtype):
    """Large tiles at odd borders: ragged batches with NaN behind the counts, operands shared by the models or repeated for
    each, aligned rows with NaN behind their last column, a base that is not aligned."""
    t = TYPES[dtype]
    G, B = 3, 2500
    counts = torch.tensor([2500, 0, 2311], dtype=torch.int32, device="cuda")
    live = live_rows(G, B, counts)
    x, w, b = rand((G, B, K), t, 1), rand((G, K, N), t, 2, K ** -0.5), rand((G, N), t, 3)
    dout = torch.where(live, rand((G, B, N), t, 4), float("nan"))
    ragged = torch.where(live, x, float("nan"))
    _, pre = check_forward(ragged, w, b, act="silu", counts=counts)
    check_backward(dout, ragged, w, torch.where(live, pre, float("inf")), "silu", counts)
    check_backward(dout, ragged, w, None, "none", counts)
    dout = rand((G, B, N), t, 5)
    one = w[:1].expand(G, K, N)
    check_forward(x[:1].expand(G, B, K), one)
    check_backward(dout, x[:1].expand(G, B, K), one, None, "none")
    check_forward(x[0], w)
    check_backward(dout, x[0], w, None, "none", counts=counts)
    check_forward(padded(x), padded(w))
    check_backward(padded(dout), padded(x), padded(w), None, "none")
    _, odd = framed((G, K, N), t, 6, 1, 7 - N % 8 if N % 8 else 7)
    check_forward(x, odd)
    for need in (("dx",), ("dw",)):
        got = dense.dense_backward(dout, x, w, need=need)
        full = dense.dense_backward(dout, x, w)
        assert all(torch.equal(a, c) for a, c in zip(got, full) if a is not None)
