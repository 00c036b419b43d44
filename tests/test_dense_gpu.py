"""GPU: the batched dense layer (mplc.dense, csrc/dense.hip) against its formulas in 64 bits.

Tolerances, per element, fixed before the first run: a sum of R products in fp32 is off by at most (R + 4) 2^-23 times
the sum of the products' magnitudes (each addition rounds by half a step of at most the sum so far; twice that covers any
order and truncation), an activation or its slope by 2^-20 of its argument, a rounding to type t by eps(t) / 2."""
import math

import pytest
import torch

from mplc import dense

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def act64(name, z):
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps  # a subnormal result's whole step


def rand(shape, t, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(t).cuda()


def live_rows(G, B, counts):
    if counts is None:
        return torch.ones(G, B, 1, dtype=torch.bool, device="cuda")
    return (torch.arange(B, device="cuda")[None, :, None] < counts[:, None, None])


def reference_forward(x, w, b, r, act, counts):
    """(z, y, bound of z, bound of y) in 64 bits; x [1 or G, B, K]."""
    G, B, K = w.shape[0], x.shape[1], w.shape[1]
    xd, wd = x.double().expand(G, B, K), w.double()
    z = torch.matmul(xd, wd)
    mag = torch.matmul(xd.abs(), wd.abs())
    if b is not None:
        z, mag = z + b.double()[:, None], mag + b.double().abs()[:, None]
    dz = (K + 4) * 2.0 ** -23 * mag
    y, _ = act64(act, z)
    dy = 1.13 * dz + 2.0 ** -20 * z.abs()
    if r is not None:
        y = y + r.double()
        dy = dy + 2.0 ** -23 * (y.abs() + r.double().abs())
    t = w.dtype
    return z, y, dz + 2.0 ** -24 * z.abs(), dy + half(t) * (y.abs() + dy) + tiny(t)


def check_forward(x, w, b=None, r=None, act="none", counts=None):
    G, B, N = w.shape[0], x.shape[-2], w.shape[2]
    out = torch.full((G, B, N), 7.0, dtype=w.dtype, device="cuda")
    pre = torch.full((G, B, N), 9.0, device="cuda")
    x3 = x if x.dim() == 3 else x[None]
    live = live_rows(G, B, counts)
    z, y, ez, ey = reference_forward(torch.nan_to_num(x3), w, b, None if r is None else torch.nan_to_num(r), act, counts)
    got = dense.dense_forward(x, w, b, residual=r, activation=act, counts=counts, preact=pre, out=out)
    assert got is out
    assert ((out.double() - y).abs() <= ey)[live.expand_as(out)].all()
    assert ((pre.double() - z).abs() <= ez)[live.expand_as(out)].all()
    assert (out[~live.expand_as(out)] == 7).all() and (pre[~live.expand_as(pre)] == 9).all()
    return out, pre


def check_backward(dout, x, w, pre, act, counts=None, dx=None):
    G, B, K = w.shape[0], x.shape[-2], w.shape[1]
    t = w.dtype
    x3 = x if x.dim() == 3 else x[None]
    live = live_rows(G, B, counts)
    xd = torch.where(live, x3.double().expand(G, B, K), 0.0)
    _, slope = act64(act, pre.double()) if act != "none" else (None, torch.ones_like(dout, dtype=torch.float64))
    d = torch.where(live, dout.double() * slope, 0.0)
    ed = torch.where(live, dout.double().abs() * 2.0 ** -20 * (1 + (pre.double().abs() if act != "none" else 0)), 0.0)
    if act == "none":
        ed = torch.zeros_like(ed)
    er = ed + (half(t) * (d.abs() + ed) + tiny(t) * live if act != "none" else 0)  # as an operand of the products
    wt = w.double().transpose(1, 2).contiguous()
    N = w.shape[2]
    rx = torch.matmul(d, wt)
    ex = torch.matmul(er, wt.abs()) + (N + 4) * 2.0 ** -23 * torch.matmul(d.abs() + er, wt.abs())
    if x3.shape[0] == 1 and G != 1 or x.dim() == 2:
        # one sum over (model, out)
        ex = torch.matmul(er, wt.abs()).sum(0, keepdim=True) + (G * N + 4) * 2.0 ** -23 * torch.matmul(
            d.abs() + er, wt.abs()).sum(0, keepdim=True)
        rx = rx.sum(0, keepdim=True)
        live_x = torch.ones(1, B, 1, dtype=torch.bool, device="cuda")
    else:
        live_x = live
    xt = xd.transpose(1, 2).contiguous()
    rw = torch.matmul(xt, d)
    ew = torch.matmul(xt.abs(), er) + (B + 4) * 2.0 ** -23 * torch.matmul(xt.abs(), d.abs() + er)
    rb, eb = d.sum(1), ed.sum(1) + (B + 4) * 2.0 ** -23 * (d.abs() + ed).sum(1)
    gx, gw, gb = dense.dense_backward(dout, x, w, preact=pre if act != "none" else None, activation=act, counts=counts,
                                      dx=dx)
    assert gx.shape == x.shape and gw.shape == w.shape and gb.shape == (G, N)
    gx3 = gx if gx.dim() == 3 else gx[None]
    for name, got, ref, err in (("dx", gx3, rx, ex), ("dw", gw, rw, ew), ("db", gb, rb, eb)):
        err = err + half(t) * (ref.abs() + err) + tiny(t)
        bad = (got.double() - ref).abs() > err
        if name == "dx":
            bad &= live_x.expand_as(bad)
        assert not bad.any(), (name, int(bad.sum()), float((got.double() - ref).abs().max()))
    return gx, gw, gb


SIZES = [(1, 1, 1, 1), (3, 1, 5, 7), (2, 33, 65, 129), (5, 51, 300, 10), (1, 128, 64, 128), (2, 130, 257, 131),
         (4, 7, 9, 300), (1, 200, 1000, 72)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes_forward_and_backward(size, dtype):
    G, B, K, N = size
    t = TYPES[dtype]
    act = ["none", "relu", "gelu", "silu"][(G + B + N) % 4]
    x, w, b = rand((G, B, K), t, 1), rand((G, K, N), t, 2, K ** -0.5), rand((G, N), t, 3)
    r = rand((G, B, N), t, 4) if N % 2 else None
    _, pre = check_forward(x, w, b, r, act)
    check_backward(rand((G, B, N), t, 5), x, w, pre, act)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_activations_and_plain_products(act, dtype):
    t = TYPES[dtype]
    x, w = rand((2, 40, 70), t, 1, 3.0), rand((2, 70, 50), t, 2)
    _, pre = check_forward(x, w, act=act)
    check_backward(rand((2, 40, 50), t, 3), x, w, pre, act)


@pytest.mark.parametrize("G,B,K,N", [(3, 2, 9216, 128), (2, 3, 5000, 33), (1, 5, 4099, 257), (1, 40, 3000, 24)])
def test_long_sums_are_split(G, B, K, N):
    for t in (torch.float32, torch.bfloat16):
        x, w = rand((G, B, K), t, 1), rand((G, K, N), t, 2, K ** -0.5)
        _, pre = check_forward(x, w, rand((G, N), t, 3), rand((G, B, N), t, 4), "silu")
        check_backward(rand((G, B, N), t, 5), x, w, pre, "silu")


@pytest.mark.parametrize("rows", [1, 2, 3, 8])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_few_rows_of_odd_weights(rows, dtype):
    t = TYPES[dtype]
    for K, N in ((7, 129), (1001, 333), (4100, 131)):
        counts = torch.tensor([rows, 0, rows - 1], dtype=torch.int32, device="cuda")
        check_forward(rand((3, rows, K), t, 1), rand((3, K, N), t, 2, K ** -0.5), rand((3, N), t, 3), rand((3, rows, N), t, 4),
                      "gelu", counts)
        check_forward(rand((rows, K), t, 5), rand((3, K, N), t, 2, K ** -0.5), act="none")


def test_long_batch():
    x, w = rand((1, 3000, 40), torch.float16, 1), rand((1, 40, 24), torch.float16, 2)
    _, pre = check_forward(x, w, act="gelu")
    check_backward(rand((1, 3000, 24), torch.float16, 3, 0.1), x, w, pre, "gelu")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shared", [False, True])
def test_ragged_counts_leave_the_rest_alone(dtype, shared):
    t = TYPES[dtype]
    G, B, K, N = 6, 70, 33, 45
    counts = torch.tensor([70, 0, 1, 64, 65, 200], dtype=torch.int32, device="cuda")
    live = live_rows(G, B, counts)
    x = rand((1 if shared else G, B, K), t, 1)
    r, dout = rand((G, B, N), t, 4), rand((G, B, N), t, 5)
    if not shared:  # what stands behind a count is never read
        x = torch.where(live, x, float("nan"))
    r, dout = torch.where(live, r, float("nan")), torch.where(live, dout, float("inf"))
    w, b = rand((G, K, N), t, 2, 0.2), rand((G, N), t, 3)
    _, pre = check_forward(x, w, b, r, "gelu", counts)
    pre = torch.where(live, pre, float("nan"))
    dx = torch.full_like(x, 5.0)
    gx, gw, gb = check_backward(dout, x, w, pre, "gelu", counts, dx=dx)
    assert gx is dx and (gw[1] == 0).all() and (gb[1] == 0).all()
    if not shared:
        assert (dx[~live.expand_as(dx)] == 5).all()
        auto = dense.dense_forward(x, w, counts=counts)
        assert (auto[~live.expand_as(auto)] == 0).all()
        gx, _, _ = dense.dense_backward(dout, x, w, counts=counts)
        assert (gx[~live.expand_as(gx)] == 0).all()


def test_negative_counts_and_idle_batches():
    t = torch.float32
    x, w = rand((3, 9, 20), t, 1), rand((3, 20, 30), t, 2)
    counts = torch.tensor([-5, 0, -1], dtype=torch.int32, device="cuda")
    out, _ = check_forward(x, w, counts=counts)
    _, gw, gb = check_backward(rand((3, 9, 30), t, 3), x, w, None, "none", counts)
    assert (out == 7).all() and (gw == 0).all() and (gb == 0).all()


def test_empty_batches():
    for t in TYPES.values():
        w = rand((2, 4, 5), t, 1)
        x = torch.empty(2, 0, 4, dtype=t, device="cuda")
        assert dense.dense_forward(x, w).shape == (2, 0, 5)
        gx, gw, gb = dense.dense_backward(torch.empty(2, 0, 5, dtype=t, device="cuda"), x, w)
        assert gx.shape == x.shape and (gw == 0).all() and (gb == 0).all()
        none = torch.empty(0, 4, 5, dtype=t, device="cuda")
        assert dense.dense_forward(torch.empty(0, 3, 4, dtype=t, device="cuda"), none).shape == (0, 3, 5)
        gx, _, _ = dense.dense_backward(torch.empty(0, 3, 5, dtype=t, device="cuda"), rand((3, 4), t, 2), none)
        assert gx.shape == (3, 4) and (gx == 0).all()


def test_shared_input_of_one_and_many_models():
    for t in TYPES.values():
        for G in (1, 9):
            x, w, b = rand((37, 50), t, 1), rand((G, 50, 66), t, 2, 0.2), rand((G, 66), t, 3)
            _, pre = check_forward(x, w, b, act="silu")
            check_backward(rand((G, 37, 66), t, 4), x, w, pre, "silu")
    # an expanded view is G inputs that happen to coincide: dx per model
    x, w = rand((1, 8, 16), torch.float32, 1).expand(3, 8, 16), rand((3, 16, 4), torch.float32, 2)
    check_forward(x, w)
    gx, _, _ = dense.dense_backward(rand((3, 8, 4), torch.float32, 3), x, w)
    assert gx.shape == (3, 8, 16)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_strided_views_and_odd_alignment(dtype):
    t = TYPES[dtype]
    G, B, K, N = 3, 21, 35, 27
    rows = rand((G, 3 * K * N + 11), t, 1, 0.2)  # models' parameter rows: w at an odd place, the bias behind it
    w = rows[:, 5:5 + K * N].view(G, K, N)
    b = rows[:, 5 + K * N:5 + K * N + N]
    x = rand((G, B, 2 * K + 3), t, 2)[:, :, 1:1 + K]
    r = rand((B, G, N + 1), t, 3)[:, :, 1:].transpose(0, 1)  # models beside one another
    out = torch.full((B, G, N + 1), 3.0, dtype=t, device="cuda")
    pre = torch.full((G, B, N + 2), 3.0, device="cuda")
    got = dense.dense_forward(x, w, b, residual=r, activation="gelu", preact=pre[:, :, 1:-1],
                              out=out[:, :, :-1].transpose(0, 1))
    z, y, ez, ey = reference_forward(x, w, b, r, "gelu", None)
    assert ((got.double() - y).abs() <= ey).all() and ((pre[:, :, 1:-1].double() - z).abs() <= ez).all()
    assert (out[:, :, -1] == 3).all() and (pre[:, :, 0] == 3).all() and (pre[:, :, -1] == 3).all()
    grads = torch.zeros_like(rows)
    dw = grads[:, 5:5 + K * N].view(G, K, N)
    db = grads[:, 5 + K * N:5 + K * N + N]
    dout = rand((G, B, N), t, 4)
    want = check_backward(dout, x, w, pre[:, :, 1:-1], "gelu")
    got = dense.dense_backward(dout, x, w, preact=pre[:, :, 1:-1], activation="gelu", dw=dw, db=db)
    for a, c in zip(want, got):
        assert torch.equal(a, c)
    assert (grads[:, :5] == 0).all() and (grads[:, 5 + K * N + N:] == 0).all()


def test_places_past_32_bits():
    buf = torch.empty(3 * (1 << 31) // 2 + (1 << 20), dtype=torch.bfloat16, device="cuda")
    w = buf.as_strided((2, 48, 40), (1 << 31, 1 << 24, 1))  # rows 16 M apart, models 2 G apart
    w.copy_(rand((2, 48, 40), torch.bfloat16, 1))
    x = rand((2, 5, 48), torch.bfloat16, 2)
    _, pre = check_forward(x, w, act="relu")
    check_backward(rand((2, 5, 40), torch.bfloat16, 3), x, w, pre, "relu")


def test_infinities_and_nan_stay_in_their_rows():
    for t in TYPES.values():
        x, w = rand((1, 70, 40), t, 1), rand((1, 40, 60), t, 2)
        clean = dense.dense_forward(x, w, activation="gelu")
        y = x.clone()
        y[0, 3, 5], y[0, 66, 0] = float("nan"), float("inf")
        got = dense.dense_forward(y, w, activation="gelu")
        keep = torch.ones(70, dtype=torch.bool, device="cuda")
        keep[3] = keep[66] = False
        assert torch.equal(got[0, keep], clean[0, keep]) and got[0, 3].isnan().all()
        assert not got[0, 66].isnan().any()  # gelu(-inf) = 0, gelu(inf) = inf
        for act in ("relu", "silu"):
            assert dense.dense_forward(y, w, activation=act)[0, 3].isnan().all()


def test_gradients_agree_with_differences():
    """The directional derivative of sum(out * dout) by central differences of the 64-bit formula: its own error is
    h^2 / 6 of the third derivative, below 1e-6 of the terms' magnitude here; the kernel's fp32 gradients add 1e-5."""
    G, B, K, N = 2, 11, 23, 19
    for act in ("gelu", "silu"):
        x, w, b = rand((G, B, K), torch.float32, 1), rand((G, K, N), torch.float32, 2, 0.3), rand((G, N), torch.float32, 3)
        r, dout = rand((G, B, N), torch.float32, 4), rand((G, B, N), torch.float32, 5)
        _, pre = check_forward(x, w, b, r, act)
        dx, dw, db = dense.dense_backward(dout, x, w, preact=pre, activation=act)
        vx, vw, vb = (rand(s, torch.float32, 10 + i).double() for i, s in enumerate([(G, B, K), (G, K, N), (G, N)]))

        def f(h):
            z = torch.matmul(x.double() + h * vx, w.double() + h * vw) + (b.double() + h * vb)[:, None]
            return (act64(act, z)[0] * dout.double()).sum()
        h = 1e-4
        num = (f(h) - f(-h)) / (2 * h)
        terms = [(dx.double() * vx), (dw.double() * vw), (db.double() * vb)]
        ana, size = sum(t.sum() for t in terms), sum(t.abs().sum() for t in terms)
        assert abs(num - ana) <= 1.1e-5 * size


def test_need_selects_the_gradients():
    x, w, d = rand((2, 6, 8), torch.float32, 1), rand((2, 8, 10), torch.float32, 2), rand((2, 6, 10), torch.float32, 3)
    full = dense.dense_backward(d, x, w)
    for need in (("dx",), ("dw",), ("db",), ("dw", "db"), ()):
        got = dense.dense_backward(d, x, w, need=need)
        for name, a, c in zip(("dx", "dw", "db"), got, full):
            assert (a is None) == (name not in need) and (a is None or torch.equal(a, c))


def test_other_stream_and_replayed_graph():
    G, B, K, N = 3, 20, 2500, 30  # split sums: the graph holds its own workspace
    x, w, b = rand((G, B, K), torch.bfloat16, 1), rand((G, K, N), torch.bfloat16, 2, 0.02), rand((G, N), torch.bfloat16, 3)
    dout, pre = rand((G, B, N), torch.bfloat16, 4), torch.empty(G, B, N, device="cuda")

    def step():
        out = dense.dense_forward(x, w, b, activation="silu", preact=pre)
        return (out,) + dense.dense_backward(dout, x, w, preact=pre, activation="silu")
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        x.copy_(rand((G, B, K), torch.bfloat16, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        eager = step()
        assert all(torch.equal(a, c) for a, c in zip(replayed, eager))


def test_results_repeat_bit_for_bit():
    x, w, d = rand((2, 300, 700), torch.float16, 1), rand((2, 700, 90), torch.float16, 2), rand((2, 300, 90), torch.float16, 3)
    a = (dense.dense_forward(x, w),) + dense.dense_backward(d, x, w)
    for _ in range(3):
        c = (dense.dense_forward(x, w),) + dense.dense_backward(d, x, w)
        assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_refusals():
    x, w = rand((2, 6, 8), torch.float32, 1), rand((2, 8, 10), torch.float32, 2)
    d, pre = rand((2, 6, 10), torch.float32, 3), torch.zeros(2, 6, 10, device="cuda")
    bad = [
        lambda: dense.dense_forward(x.cpu(), w), lambda: dense.dense_forward(x, w.double()),
        lambda: dense.dense_forward(x.bfloat16(), w), lambda: dense.dense_forward(x[:, :, :7], w),
        lambda: dense.dense_forward(x, w, activation="tanh"), lambda: dense.dense_forward(x, w[0]),
        lambda: dense.dense_forward(x, w.transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: dense.dense_forward(x, w, bias=torch.zeros(10, device="cuda")),
        lambda: dense.dense_forward(x, w, counts=torch.tensor([1, 2], device="cuda")),
        lambda: dense.dense_forward(x, w, out=torch.zeros(1, 6, 10, device="cuda").expand(2, 6, 10)),
        lambda: dense.dense_forward(x, w, preact=torch.zeros(2, 6, 10, dtype=torch.bfloat16, device="cuda")),
        lambda: dense.dense_forward(x, w, residual=d, out=d),
        lambda: dense.dense_backward(d, x, w, activation="gelu"),
        lambda: dense.dense_backward(d[:, :5], x, w),
        lambda: dense.dense_backward(d, x, w, dx=x), lambda: dense.dense_backward(d, x, w, need=("dz",)),
        lambda: dense.dense_backward(d, x, w, preact=pre.half(), activation="relu"),
    ]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
