"""GPU: the batched operators at the ends of what they accept - the longest matrices, inputs that no model reaches, the
tails of the activations, results as the exact parts of one buffer."""
import math

import pytest
import torch

from mplc import dense, muon
from test_dense_gpu import TYPES, check_backward, check_forward, half, live_rows, rand, tiny

pytestmark = pytest.mark.gpu


def test_longest_row():
    """A 1 x L matrix whose last chunk of columns ends less than a chunk below 2^31.  k = 1: O(u) = u / |u| times the number
    that five steps make of 1.  A sum of squares is fp32, each partial sum at most 3 * 2^16 additions long (4194304 columns,
    16 a matrix instruction, 4 waves, 3 instructions each): off by less than 3 * 2^16 * 2^-24 = 1.2 %.  Such errors of both
    phases' sums change the result by at most 2 % (the recurrence with sums off by 1.2 % up or down); its rounding is 2^-9.  X = u / |u| is held
    in two fp16 numbers at a scale of 2^14, whose last place is 2^-24: off by at most half of that, 2^-39 of |u|, which shows
    where u itself is below 2^-24 or so of |u|; X Q1 Q2 multiplies that by less than 1."""
    L = 2147400000
    u = torch.empty(1, L, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    square = 0.0
    for i in range(0, L, 1 << 28):
        part = u[0, i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=g, dtype=torch.bfloat16))
        square += float(part.double().square_().sum())
    out = torch.zeros_like(u)
    assert muon.orthogonalize(u, out=out) is out
    s = 1.0
    a, b, c = muon.COEFFICIENTS
    for _ in range(5):
        s = s * (a + s * s * (b + s * s * c))
    for i in (0, 1 << 30, 511 * 4194304 - 5, 511 * 4194304, L - (1 << 21), L - 1):
        part = slice(i, min(L, i + (1 << 20)))
        want = u[0, part].double() * (s / square ** 0.5)
        assert ((out[0, part].double() - want).abs() <= (0.02 + 2.0 ** -9) * want.abs() + 2.0 ** -39).all(), i
    # every column is written: no zero but where |u| is below 2^-39 of |U|, as above
    for i in range(0, L, 1 << 28):
        part = slice(i, min(L, i + (1 << 28)))
        assert not ((out[0, part] == 0) & (u[0, part].abs() > square ** 0.5 * 2.0 ** -39)).any(), i


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("B,K,N", [(70, 33, 45), (40, 64, 128), (5, 40, 9000), (300, 264, 520)])
def test_shared_rows_that_no_model_reaches(B, K, N, dtype):
    """One model behind its count, and no model at all: such rows of a given dx get 0, as with several models."""
    t = TYPES[dtype]
    x, w = rand((B, K), t, 1), rand((1, K, N), t, 2, 0.2)
    for n in (B - 3, 0):
        counts = torch.tensor([n], dtype=torch.int32, device="cuda")
        dout = rand((1, B, N), t, 3)
        dout[:, n:] = float("nan")
        for act in ("none", "silu"):
            pre = rand((1, B, N), torch.float32, 4)
            dx = torch.full_like(x, 5.0)
            gx, _, _ = check_backward(dout, x, w, pre, act, counts, dx=dx)
            assert gx is dx and (dx[n:] == 0).all()
    for shape in ((B, K), (1, B, K)):
        dx = torch.full(shape, 5.0, dtype=t, device="cuda")
        none = torch.empty(0, K, N, dtype=t, device="cuda")
        gx, _, _ = dense.dense_backward(torch.empty(0, B, N, dtype=t, device="cuda"), x.view(shape), none, dx=dx)
        assert gx is dx and (dx == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("N", [20000, 20001])
def test_gelu_keeps_its_digits_in_the_tail(N, dtype):
    """z = 1 * w, exactly.  gelu: the documented relative error, 2^-19 in fp32 and 2^-16 for 16-bit results, and the rounding.
    Its slope cdf + z density (db of one row, with dout = 1): for z <= -2 twice that (the two terms cancel by a factor of 1.6
    at most), elsewhere 2^-20 as well.  Results below 2^-120 may be off by that."""
    t = TYPES[dtype]
    z = torch.linspace(-16.0, 8.0, N, dtype=torch.float64).to(t).cuda()
    rel = 2.0 ** -19 if dtype == "fp32" else 2.0 ** -16
    zd = z.double()
    cdf = 0.5 * torch.erfc(-zd / math.sqrt(2))
    one = torch.ones(1, 1, 1, dtype=t, device="cuda")
    pre = torch.empty(1, 1, N, device="cuda")
    y = dense.dense_forward(one, z.view(1, 1, N), activation="gelu", preact=pre)[0, 0]
    assert torch.equal(pre[0, 0].double(), zd)
    want = zd * cdf
    err = rel * want.abs()
    assert ((y.double() - want).abs() <= err + half(t) * (want.abs() + err) + tiny(t) + 2.0 ** -120).all()
    _, _, db = dense.dense_backward(torch.ones(1, 1, N, dtype=t, device="cuda"), one, z.view(1, 1, N), preact=pre, activation="gelu")
    want = cdf + zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    err = 2 * rel * want.abs() + torch.where(zd <= -2, 0.0, 2.0 ** -20)
    assert ((db[0].double() - want).abs() <= err + half(t) * (want.abs() + err) + tiny(t) + 2.0 ** -120).all()


def test_tensors_that_require_grad():
    """No result without its graph: refused in grad mode, computed under no_grad; what a call overwrites is seen by a graph
    that has saved it."""
    x, w, d, pre = rand((2, 6, 8), torch.float32, 1), rand((2, 8, 10), torch.float32, 2), rand((2, 6, 10), torch.float32, 3), torch.empty(2, 6, 10, device="cuda")
    want = dense.dense_forward(x, w, preact=pre)
    m = torch.zeros_like(w)
    calls = [lambda t: dense.dense_forward(t(x), w), lambda t: dense.dense_forward(x, t(w)), lambda t: dense.dense_forward(x, w, residual=t(d)),
             lambda t: dense.dense_forward(x, w, out=t(d)), lambda t: dense.dense_backward(d, x, t(w)),
             lambda t: dense.dense_backward(t(d), x, w), lambda t: dense.dense_backward(d, x, w, preact=t(pre), activation="silu"),
             lambda t: muon.orthogonalize(t(w)), lambda t: muon.orthogonalize(t(w[0])), lambda t: muon.muon_step(t(w), w.clone(), m, lr=0.1),
             lambda t: muon.muon_step(w.clone(), t(w), m, lr=0.1)]

    def leaf(t):
        return t.detach().clone().requires_grad_()
    for f in calls:
        with pytest.raises(ValueError, match="requires grad"):
            f(leaf)
        with torch.no_grad():
            f(leaf)
    with torch.no_grad():
        assert torch.equal(dense.dense_forward(leaf(x), leaf(w)), want)
    a = torch.ones(2, 8, 10, device="cuda", requires_grad=True)
    for write in (lambda v: dense.dense_backward(d, x, w, need=("dw",), dw=v), lambda v: muon.muon_step(v, w.clone(), m, lr=0.1),
                  lambda v: muon.muon_step(w.clone(), w.clone(), v, lr=0.1), lambda v: muon.orthogonalize(v, out=v),
                  lambda v: muon.orthogonalize(w[0], out=v[0])):
        v = w.clone()
        loss = (a * v).sum()
        write(v)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        assert torch.equal(dense.dense_forward(x, w, out=torch.empty(2, 6, 10, device="cuda")), want)


@pytest.mark.parametrize("G", [1, 2])
def test_results_into_columns_of_one_buffer(G):
    """Two layers' results side by side, the second's input and residual in the same rows."""
    x, w, v = rand((G, 9, 20), torch.float32, 1), rand((G, 20, 12), torch.float32, 2), rand((G, 12, 12), torch.float32, 3)
    buf = torch.full((G, 9, 40), 3.0, device="cuda")
    a, b, r = buf[:, :, :12], buf[:, :, 12:24], buf[:, :, 25:37]
    want = dense.dense_forward(x, w)
    want2 = dense.dense_forward(want, v, residual=r.clone(), activation="silu")
    dense.dense_forward(x, w, out=a)
    dense.dense_forward(a, v, residual=r, activation="silu", out=b)
    assert torch.equal(a, want) and torch.equal(b, want2) and (buf[:, :, 24:] == 3).all()
    g = rand((G, 8, 30), torch.float32, 4)
    o = muon.orthogonalize(g[:, :, :14].contiguous())
    muon.orthogonalize(g[:, :, :14], out=g[:, :, 14:28])
    assert torch.equal(g[:, :, 14:28], o)


@pytest.mark.parametrize("rows", [1, 2, 3, 8])
@pytest.mark.parametrize("G,K,N", [(3, 4100, 401), (1, 32771, 131), (200, 171, 130), (9, 4099, 129)])
def test_few_rows_of_large_fp32_weights(G, K, N, rows):
    """Weights of 4 M elements and more in cut rows: sums split and whole, one to many models, idle ones, rows behind the
    counts that hold NaN, and an input shared by all."""
    t = torch.float32
    counts = torch.tensor([rows, 0, rows - 1, 99, -3][:G] + [rows] * max(0, G - 5), dtype=torch.int32, device="cuda")
    x, w = rand((G, rows, K), t, 1), rand((G, K, N), t, 2, K ** -0.5)
    x = torch.where(live_rows(G, rows, counts), x, float("nan"))
    check_forward(x, w, rand((G, N), t, 3), rand((G, rows, N), t, 4), "gelu", counts)
    check_forward(rand((rows, K), t, 5), w, act="none")


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("B,K,N,pad", [(40, 33, 45, 0), (130, 64, 128, 0), (130, 60, 128, 4), (5, 40, 9000, 0), (300, 520, 264, 0),
                                       (700, 1030, 96, 0), (2048, 2304, 512, 0)])
def test_shared_gradient_beside_models_that_are_not_finite(B, K, N, pad, dtype):
    """A shared input's dx sums each row over the models that have it: a model that has no row there, idle or behind its
    count, adds nothing, be its weights infinite or NaN.  Rows that such a model has are not finite."""
    t = TYPES[dtype]
    counts = torch.tensor([B - 2, 0, B, 1, -3, B // 2, 2 * B], dtype=torch.int32, device="cuda")
    G = len(counts)
    live = live_rows(G, B, counts)
    x = rand((B, K + pad), t, 1)[:, :K]
    w = rand((G, K, N + pad), t, 2, 0.2)[:, :, :N]
    dout, pre = rand((G, B, N), t, 3), rand((G, B, N), torch.float32, 4)
    dout, pre = torch.where(live, dout, float("nan")), torch.where(live, pre, float("inf"))
    for act in ("none", "gelu"):
        want, _, _ = check_backward(dout, x, w, pre, act, counts)
        bad = w.clone()
        bad[1], bad[4] = float("nan"), float("inf")
        dx = torch.full((B, K), 5.0, dtype=t, device="cuda")
        got, _, _ = dense.dense_backward(dout, x, bad, preact=pre, activation=act, counts=counts, need=("dx",), dx=dx)
        assert got is dx and torch.equal(got, want)
        bad[3], bad[5, :, 0] = float("inf"), float("nan")
        got, _, _ = dense.dense_backward(dout, x, bad, preact=pre, activation=act, counts=counts, need=("dx",))
        assert torch.equal(got[B // 2:], want[B // 2:]) and got[:B // 2].isnan().all()


def test_step_sizes_that_are_not_finite_in_fp32():
    """Refused before anything is written."""
    w, g, m = rand((2, 6, 8), torch.float32, 1), rand((2, 6, 8), torch.float32, 2), rand((2, 6, 8), torch.float32, 3)
    keep = w.clone(), m.clone()
    nan, big = float("nan"), 1e39
    for kw in (dict(lr=big), dict(lr=nan), dict(lr=-big), dict(lr=0.0, scale=big), dict(lr=1e30, scale=1e30), dict(lr=0.1, beta=big),
               dict(lr=0.1, beta=nan), dict(lr=0.1, weight_decay=big), dict(lr=0.0, weight_decay=float("inf")),
               dict(lr=1e30, weight_decay=1e30)):
        with pytest.raises(ValueError, match="finite"):
            muon.muon_step(w, g, m, **kw)
    assert torch.equal(w, keep[0]) and torch.equal(m, keep[1])
