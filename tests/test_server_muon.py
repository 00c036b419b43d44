"""The server's Muon optimizer (mplc.muon.ServerMuon) in the engine's FedAvg rounds: its settings (CPU), one round against
the formula in 64 bits, independence of the batch, and a chain of the batched operators (GPU)."""
import numpy as np
import pytest

from mplc import muon


def scenario(**kw):
    from mplc.dataset import ArrayDataset, digits_as_mnist
    from mplc.scenario import Scenario
    x, y = digits_as_mnist()
    ds = ArrayDataset(x[:900], y[:900], x[900:1200], y[900:1200])
    kw = dict(dict(minibatch_count=1, gradient_updates_per_pass_count=4, epoch_count=1, is_early_stopping=False), **kw)
    return Scenario(4, [0.2, 0.3, 0.3, 0.2], dataset=ds, **kw)


def test_settings():
    s = muon.ServerMuon("muon")
    assert s.params == muon.ServerMuon.DEFAULTS and s.describe()["name"] == "muon"
    assert muon.ServerMuon({"name": "muon", "lr": 0.1, "steps": 3}).params["lr"] == 0.1
    for bad in ("adam", {"lr": 0.1}, {"name": "muon", "momentum": 0.9}, {"name": "muon", "lr": 0}, {"name": "muon", "beta": 1.0},
                {"name": "muon", "steps": 0}, {"name": "muon", "lr": float("nan")}):
        with pytest.raises(ValueError):
            muon.ServerMuon(bad)
    layers = ((0, (3, 3, 1, 32)), (288, (32,)), (320, (9216, 128)))
    assert muon.ServerMuon.matrices(layers) == [(0, 9, 32), (320, 9216, 128)]


def test_scenario_checks_and_fingerprint():
    plain, other = scenario().provision(), scenario(server_optimizer={"name": "muon", "lr": 0.05}).provision()
    assert "server_optimizer" not in plain.coalition_values_fingerprint()
    assert "0.05" in other.coalition_values_fingerprint()
    with pytest.raises(ValueError):
        scenario(server_optimizer="sgd")
    with pytest.raises(NotImplementedError):
        scenario(server_optimizer="muon", multi_partner_learning_approach="seqavg")


def engine(**kw):
    from mplc.engine import CoalitionEngine
    return CoalitionEngine.for_scenario(scenario(**kw).provision(), memory_budget_bytes=4 << 30, eval_budget_bytes=1 << 30)


def exact(u):
    a, b, c = muon.COEFFICIENTS
    x = u / np.linalg.norm(u)
    for _ in range(5):
        if x.shape[0] <= x.shape[1]:
            A = x @ x.T
            x = a * x + (b * A + c * (A @ A)) @ x
        else:
            A = x.T @ x
            x = a * x + x @ (b * A + c * (A @ A))
    return x


@pytest.mark.gpu
def test_one_round_is_the_formula():
    """A round's difference (before - average) comes from the same training with and without the server optimizer; the
    first step's direction is the orthogonalised difference itself (momentum 0).  Tolerance: 2^-9 of the step in the
    Frobenius norm (the difference of two fp32 models carries about 2^-24 |W| / |difference| < 2^-14 of error, and
    small singular values grow by up to a^5 = 485 beside directions of that size) and fp32's rounding of the weights."""
    import torch
    from mplc import _native, cnn
    coal, lr, wd = (0, 2, 3), 0.03, 0.1
    eng = engine()
    average = eng.evaluate([coal], return_details=True, return_models=True)["models"][0]
    init = torch.empty((1, cnn.STRIDE), device="cuda")
    key = torch.from_numpy(np.array([cnn.init_key(eng.seed, sum(1 << p for p in coal))], dtype=np.uint64).view(np.int64)).cuda()
    eng.model_impl.init_params(init, key, _native.stream_handle())
    before = cnn.keras_weights(init[0].cpu().numpy())
    moved = engine(server_optimizer={"name": "muon", "lr": lr, "weight_decay": wd}).evaluate(
        [coal], return_details=True, return_models=True)["models"][0]
    for w0, avg, got in zip(before, average, moved):
        if w0.ndim == 1:
            assert np.array_equal(avg, got)
            continue
        cols = w0.shape[-1]
        w, d = w0.reshape(-1, cols).astype(np.float64), (w0 - avg).reshape(-1, cols).astype(np.float64)
        step = lr * muon.update_scale(*w.shape) * exact(d)
        want = (1 - lr * wd) * w - step
        err = np.linalg.norm(got.reshape(-1, cols) - want)
        assert err <= 2.0 ** -9 * np.linalg.norm(step) + 2.0 ** -22 * np.linalg.norm(want), (w0.shape, err)


@pytest.mark.gpu
def test_values_do_not_depend_on_the_batch():
    spec = {"name": "muon", "lr": 0.02}
    kw = dict(server_optimizer=spec, minibatch_count=2, epoch_count=2)
    coals = [(0, 1), (0, 1, 2, 3), (2,), (1, 3), (0, 2, 3)]
    a = engine(**kw).evaluate(coals, return_details=True, return_models=True)["models"]
    for i in (0, 1, 4):
        b = engine(**kw).evaluate([coals[i]], return_details=True, return_models=True)["models"][0]
        assert all(np.array_equal(p, q) for p, q in zip(a[i], b))
    single = engine(minibatch_count=2, epoch_count=2).evaluate([(2,)], return_details=True, return_models=True)["models"][0]
    assert all(np.array_equal(p, q) for p, q in zip(a[2], single))  # a singleton has no server


@pytest.mark.gpu
def test_cifar_rounds_run_with_it():
    from mplc.dataset import Cifar10
    from mplc.engine import CoalitionEngine
    from mplc.scenario import Scenario
    ds = Cifar10(synthetic=True, signal=1.0)
    ds.shorten_dataset_proportion(0.01)
    sc = Scenario(2, [0.5, 0.5], dataset=ds, minibatch_count=2, gradient_updates_per_pass_count=2, epoch_count=1,
                  is_early_stopping=False, server_optimizer="muon").provision()
    eng = CoalitionEngine.for_scenario(sc, memory_budget_bytes=4 << 30, eval_budget_bytes=1 << 30)
    m = eng.evaluate([(0, 1)], return_details=True, return_models=True)["models"][0]
    assert all(np.isfinite(w).all() for w in m)


@pytest.mark.gpu
def test_operators_train_a_lockstep_batch():
    """Two dense layers of 5 models in their parameter rows: forward, backward, Muon steps, FedAvg - captured into a graph
    and replayed, equal to the eager run; the gradients of the chain against the 64-bit formula.  Tolerance of the
    chain's gradients: each of the 4 products sums at most 64 terms in fp32, 64 * 4 * 2^-23 of the terms' magnitude,
    taken in the Frobenius norm with the norms of the factors."""
    import torch
    from mplc import dense
    from mplc.fedavg import fedavg_aggregate
    G, B, K, H, N = 5, 33, 48, 64, 10
    gen = torch.Generator().manual_seed(0)
    sizes = (K * H, H, H * N, N)
    offs = np.concatenate([[0], np.cumsum(sizes)])
    rows = (torch.randn(G, int(offs[-1]) + 6, generator=gen) * 0.1).cuda()
    x, d = torch.randn(G, B, K, generator=gen).cuda(), torch.randn(G, B, N, generator=gen).cuda()
    counts = torch.tensor([33, 1, 20, 0, 33], dtype=torch.int32, device="cuda")

    def views(r):
        p = [r[:, offs[i]:offs[i + 1]] for i in range(4)]
        return p[0].view(G, K, H), p[1], p[2].view(G, H, N), p[3]
    grads, mom = torch.zeros_like(rows), torch.zeros_like(rows)

    def step(rows, grads, mom):
        w1, b1, w2, b2 = views(rows)
        g1, c1, g2, c2 = views(grads)
        z1 = torch.zeros(G, B, H, device="cuda")
        h = dense.dense_forward(x, w1, b1, activation="gelu", counts=counts, preact=z1)
        y = dense.dense_forward(h, w2, b2, counts=counts)
        dh, _, _ = dense.dense_backward(d, h, w2, counts=counts, dw=g2, db=c2)
        dense.dense_backward(dh, x, w1, preact=z1, activation="gelu", counts=counts, need=("dw", "db"), dw=g1, db=c1)
        m1, _, m2, _ = views(mom)
        muon.muon_step(w1, g1, m1, lr=0.02)
        muon.muon_step(w2, g2, m2, lr=0.02)
        return y

    start = rows.clone()
    y = step(rows, grads, mom)
    w1, b1, w2, b2 = (t.double() for t in views(start))
    live = torch.arange(B, device="cuda")[None, :, None] < counts[:, None, None]
    z = torch.matmul(x.double(), w1) + b1[:, None]
    cdf = 0.5 * torch.erfc(-z / 2 ** 0.5)
    h = z * cdf * live
    dd = d.double() * live
    dz = torch.matmul(dd, w2.transpose(1, 2).contiguous()) * (cdf + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5) * live
    want = [torch.matmul(x.double().transpose(1, 2).contiguous(), dz), dz.sum(1),
            torch.matmul(h.transpose(1, 2).contiguous(), dd), dd.sum(1)]
    tol = 64 * 4 * 2.0 ** -23
    for got, ref, f in zip(views(grads), want, (x, d, h, d)):
        scale = float(torch.linalg.vector_norm(f.double())) * float(torch.linalg.vector_norm(dd if ref is want[2] or ref is want[3] else dz))
        assert float(torch.linalg.vector_norm(got.double() - ref)) <= tol * scale
    assert (y[3] == 0).all() and torch.equal(rows[3, :K * H], start[3, :K * H])  # an idle model's update is zero
    rows2, grads2, mom2 = start.clone(), torch.zeros_like(grads), torch.zeros_like(mom)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(rows2, grads2, mom2)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows2, rows) and torch.equal(mom2, mom)
        step(rows, grads, mom)
    avg = fedavg_aggregate(rows, [[0, 1, 2], [3, 4]], [[1, 1, 1], [2, 2]], scheme="uniform")
    assert torch.isfinite(avg).all()
