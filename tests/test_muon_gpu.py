"""GPU: the orthogonalised update and the Muon step (mplc.muon, csrc/muon.hip) against their formulas in 64 bits.

Tolerance, in the Frobenius norm, fixed before the first run: a step's matrices are held and summed to 2^-21 of their size;
an error e of the Gram matrix enters X with |b| + 2 |c| < 9, so a step perturbs X_t by at most 2^-21 (9 + 3) |X_t| < 2^-17
|X_t| (a phase of three steps from one Gram matrix: the same, twice), and each later step multiplies a perturbation by at
most the largest slope of a s + b s^3 + c s^5, which is a.  Then the rounding to the result's type."""
import math

import pytest
import torch

from mplc import muon

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
COEF = muon.COEFFICIENTS


def rand(shape, t=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(t).cuda()


def exact(u, steps=5, coef=COEF):
    """(O(u), tolerance) in 64 bits for one matrix."""
    a, b, c = coef
    x = u.double()
    n = torch.linalg.vector_norm(x)
    if n == 0:
        return x, 0.0
    x = x / n
    tol = 0.0
    for _ in range(steps):
        tol = a * (tol + 2.0 ** -17 * float(torch.linalg.vector_norm(x)))
        if x.shape[0] <= x.shape[1]:
            A = x @ x.t().contiguous()
            x = a * x + (b * A + c * (A @ A)) @ x
        else:
            A = x.t().contiguous() @ x
            x = a * x + x @ (b * A + c * (A @ A))
    return x, tol


def close(got, u, steps=5, coef=COEF):
    ref, tol = exact(u, steps, coef)
    eps = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    err = float(torch.linalg.vector_norm(got.double() - ref))
    tol += eps * (float(torch.linalg.vector_norm(ref)) + tol) + torch.finfo(got.dtype).tiny * math.sqrt(got.numel())
    assert err <= tol, (err, tol)


SIZES = [(1, 1), (1, 9), (9, 1), (3, 5), (32, 9), (10, 128), (128, 10), (64, 64), (65, 63), (65, 200), (288, 32),
         (130, 130), (128, 1000), (777, 150), (300, 290), (2000, 128), (2000, 40), (40, 2000)]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes(size):
    g = rand((3,) + size, seed=sum(size))
    out = muon.orthogonalize(g)
    for i in range(3):
        close(out[i], g[i])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [(33, 70), (256, 512), (1000, 64)])
def test_16_bit_updates(dtype, size):
    g = rand((2,) + size, TYPES[dtype], 1)
    out = muon.orthogonalize(g)
    assert out.dtype == TYPES[dtype]
    for i in range(2):
        close(out[i], g[i])


@pytest.mark.parametrize("spectrum", ["power", "steep", "low rank"])
def test_decaying_spectra(spectrum):
    k, L = 96, 700
    s = {"power": 1.0 / torch.arange(1, k + 1), "steep": 0.9 ** torch.arange(k).float(),
         "low rank": torch.cat([torch.ones(5), torch.zeros(k - 5)])}[spectrum].double()
    u = torch.linalg.qr(rand((k, k)).double().cpu())[0]
    v = torch.linalg.qr(rand((L, k), seed=1).double().cpu())[0]
    g = ((u * s) @ v.t()).float().cuda()
    for m in (g, g.t().contiguous()):
        close(muon.orthogonalize(m), m)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_steps_and_coefficients(steps):
    for shape in ((60, 60), (40, 200)):
        g = rand(shape, seed=steps)
        close(muon.orthogonalize(g, steps=steps), g, steps)
        cubic = (1.5, -0.5, 0.0)
        close(muon.orthogonalize(g, steps=steps, coefficients=cubic), g, steps, cubic)


def test_many_steps_orthogonalize():
    g = rand((50, 200))
    o = muon.orthogonalize(g, steps=16, coefficients=(1.5, -0.5, 0.0)).double()
    assert (o @ o.t().contiguous() - torch.eye(50, device="cuda")).abs().max() < 1e-4


def test_scale_does_not_matter():
    g = rand((2, 30, 90))
    want = muon.orthogonalize(g)
    for s in (2.0 ** -100, 2.0 ** 60):
        assert torch.equal(muon.orthogonalize(g * s), want)


def test_zero_and_not_finite_matrices():
    for shape in ((6, 70, 40), (6, 9, 5), (6, 200, 130)):
        g = rand(shape, seed=3)
        g[1] = 0
        g[2, 3, 4], g[4, 0, 0] = float("nan"), float("inf")
        out = muon.orthogonalize(g)
        assert (out[1] == 0).all() and out[2].isnan().all() and out[4].isnan().all()
        for i in (0, 3, 5):
            close(out[i], g[i])


def test_strided_views_and_in_place():
    G, m, n = 3, 31, 45
    rows = rand((G, m * n + 13))
    keep = rows.clone()
    v = rows[:, 7:7 + m * n].view(G, m, n)
    want = muon.orthogonalize(v)
    out = torch.full((G, m, n + 3), 2.0, device="cuda")
    got = muon.orthogonalize(v, out=out[:, :, 1:-2])
    assert torch.equal(got, want) and (out[:, :, 0] == 2).all() and (out[:, :, -2:] == 2).all()
    assert torch.equal(rows, keep)
    muon.orthogonalize(v, out=v)
    assert torch.equal(v, want) and torch.equal(rows[:, :7], keep[:, :7]) and torch.equal(rows[:, 7 + m * n:], keep[:, 7 + m * n:])


def reference_step(w, g, m, lr, beta, nesterov, wd, scale):
    """(w, m, tolerance of w per matrix) in 64 bits."""
    mom = beta * m.double() + g.double()
    u = g.double() + beta * mom if nesterov else mom
    out, tol = [], []
    for i in range(w.shape[0]):
        o, t = exact(u[i])
        # u itself is rounded to fp32 twice; its relative error 2^-22 grows as any perturbation of X_0 does
        out.append((1 - lr * wd) * w[i].double() - lr * scale * o)
        tol.append(lr * scale * 2 * t)
    return torch.stack(out), mom, tol


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("size", [(5, 128, 10), (2, 100, 260), (3, 9, 32), (2, 1152, 128)])
def test_step(size, nesterov, dtype):
    w, m, g = rand(size, seed=1), rand(size, seed=2), rand(size, TYPES[dtype], 3)
    scale = math.sqrt(max(1.0, size[2] / size[1]))
    rw, rm, tol = reference_step(w, g, m, 0.02, 0.95, nesterov, 0.1, scale)
    assert muon.muon_step(w, g, m, lr=0.02, nesterov=nesterov, weight_decay=0.1) is w
    assert ((m.double() - rm).abs() <= 2.0 ** -23 * (rm.abs() + 4)).all()
    for i in range(size[0]):
        err = float(torch.linalg.vector_norm(w[i].double() - rw[i]))
        assert err <= tol[i] + 2.0 ** -22 * float(torch.linalg.vector_norm(rw[i]))


def test_step_on_parameter_rows_leaves_the_rest():
    G, K, N = 4, 60, 33
    rows, grads, moms = rand((G, K * N + 20), seed=1), rand((G, K * N + 20), seed=2), rand((G, K * N + 20), seed=3)
    keep = [t.clone() for t in (rows, grads, moms)]
    views = [t[:, 9:9 + K * N].view(G, K, N) for t in (rows, grads, moms)]
    rw, rm, tol = reference_step(views[0], views[1], views[2], 0.1, 0.9, True, 0.0, 3.0)
    muon.muon_step(*views, lr=0.1, beta=0.9, scale=3.0)
    for i in range(G):
        assert float(torch.linalg.vector_norm(views[0][i].double() - rw[i])) <= tol[i] + 2.0 ** -22 * float(
            torch.linalg.vector_norm(rw[i]))
    assert torch.equal(grads, keep[1])
    for t, k in zip((rows, moms), (keep[0], keep[2])):
        assert torch.equal(t[:, :9], k[:, :9]) and torch.equal(t[:, 9 + K * N:], k[:, 9 + K * N:])


def test_zero_update_only_decays():
    w, m, g = rand((2, 20, 30), seed=1), torch.zeros(2, 20, 30, device="cuda"), torch.zeros(2, 20, 30, device="cuda")
    want = w * float(torch.tensor(1 - 0.5 * 0.1, dtype=torch.float32))
    muon.muon_step(w, g, m, lr=0.5, weight_decay=0.1)
    assert torch.equal(w, want) and (m == 0).all()


def test_other_stream_and_replayed_graph():
    w, m, g = rand((3, 150, 700), seed=1), rand((3, 150, 700), seed=2), rand((3, 150, 700), seed=3)
    start = (w.clone(), m.clone())

    def step():
        muon.muon_step(w, g, m, lr=0.05)
        return muon.orthogonalize(g)
    want = [t.clone() for t in (step(), w, m)]
    w.copy_(start[0]), m.copy_(start[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, (o, w, m)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    w.copy_(start[0]), m.copy_(start[1])
    we, me = w.clone(), m.clone()
    for k in range(3):
        g.copy_(rand((3, 150, 700), seed=30 + k))
        graph.replay()
        torch.cuda.synchronize()
        muon.muon_step(we, g, me, lr=0.05)
        assert torch.equal(w, we) and torch.equal(m, me) and torch.equal(o, muon.orthogonalize(g))


def test_refusals():
    g = rand((2, 6, 8))
    bad = [
        lambda: muon.orthogonalize(g.cpu()), lambda: muon.orthogonalize(g.double()), lambda: muon.orthogonalize(g[0, 0]),
        lambda: muon.orthogonalize(g[:, :0]), lambda: muon.orthogonalize(g, steps=0), lambda: muon.orthogonalize(g, steps=17),
        lambda: muon.orthogonalize(g, coefficients=(4.0, -4.0, 3.0)), lambda: muon.orthogonalize(g, coefficients=(1.5, -0.5)),
        lambda: muon.orthogonalize(g, coefficients=(float("nan"), 0.0, 0.0)),
        lambda: muon.orthogonalize(g.transpose(1, 2)), lambda: muon.orthogonalize(g, out=torch.empty_like(g, dtype=torch.half)),
        lambda: muon.orthogonalize(g, out=g.flatten()[8:88].view(2, 5, 8)),
        lambda: muon.muon_step(g.clone(), g, g.half(), lr=0.1), lambda: muon.muon_step(g.clone(), g, g, lr=0.1),
        lambda: muon.muon_step(g, g.clone(), g, lr=0.1), lambda: muon.muon_step(g.clone(), g, g.clone(), lr=float("inf")),
        lambda: muon.muon_step(g[:1].clone().expand(2, 6, 8), g, g.clone(), lr=0.1),
    ]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
    none = torch.empty(0, 3, 4, device="cuda")
    assert muon.orthogonalize(none).shape == (0, 3, 4)


@pytest.mark.parametrize("size", [(128, 10), (60, 40), (1500, 100), (100, 1500), (300, 200), (200, 600)])
def test_batch_invariant_results(size):
    """The same bits alone, in a small and in a large batch."""
    g = rand((40,) + size, seed=5)
    want = muon.orthogonalize(g, batch_invariant=True)
    for n in (1, 7):
        assert torch.equal(muon.orthogonalize(g[:n], batch_invariant=True), want[:n])
    close(want[3], g[3])
    w, m = rand((40,) + size, seed=6), rand((40,) + size, seed=7)
    w1, m1 = w[:1].clone(), m[:1].clone()
    muon.muon_step(w, g, m, lr=0.1, batch_invariant=True)
    muon.muon_step(w1, g[:1], m1, lr=0.1, batch_invariant=True)
    assert torch.equal(w1, w[:1]) and torch.equal(m1, m[:1])
