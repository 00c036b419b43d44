"""GPU: the server's Muon optimizer as a lockstep batch carries it on - its rounds enqueue without waiting for the device."""
import pytest

from test_server_muon import engine

pytestmark = pytest.mark.gpu


def test_a_round_does_not_wait_for_the_device():
    """Two lockstep batches on two streams are enqueued by one thread: an upload from pageable memory in one's round would
    hold back the other's."""
    import torch
    eng = engine(server_optimizer="muon")
    st = eng.trainer.prepare([(0, 1), (2,), (1, 2, 3)], 1)
    st.aggregate()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        st.aggregate()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()
    for ci, rows in ((0, (0, 1)), (2, (3, 4, 5))):
        for r in rows:
            assert torch.equal(st.params[r], st.glob[ci])


def test_rounds_are_the_recurrence_through_stops_and_compaction():
    """Four rounds of hand-filled replicas against m = beta m + (before - average), u = difference + beta m, w = (1 - lr wd)
    before - lr scale O(u) in 64 bits, each round from the device's own models; the middle coalition stops after the second,
    which splits the runs; a batch compacted there continues with the same bits.  Tolerances: of w as for one round (2^-9 of
    the step in the Frobenius norm and fp32's rounding of the weights); of m two roundings of its terms a round."""
    import numpy as np
    import torch
    from mplc import cnn, muon
    from mplc.fedavg import aggregation_weights
    from test_server_muon import exact
    lr, beta, wd = 0.05, 0.8, 0.1
    eng = engine(server_optimizer={"name": "muon", "lr": lr, "beta": beta, "weight_decay": wd})
    coals = [(0, 1), (2,), (1, 2, 3), (0, 3), (0, 2)]
    whole, small = (eng.trainer.prepare(coals, 1) for _ in range(2))
    live = list(range(len(coals)))
    place = {ci: ci for ci in live}  # coalition -> its row in `small`
    mats = muon.ServerMuon.matrices(cnn.KERAS_LAYERS)
    mom = {ci: [np.zeros((r, c)) for _, r, c in mats] for ci in live}
    size = {ci: [np.zeros((r, c)) for _, r, c in mats] for ci in live}

    def fill(st, ci, row, n):
        """The round's partner models: the coalition's model and a change that only the round, the coalition and the member set."""
        for k in range(st.coal_first[row + 1] - st.coal_first[row]):
            gen = torch.Generator().manual_seed(1000 * n + 10 * ci + k)
            st.params[st.coal_first[row] + k] = st.glob[row] + 0.01 * torch.randn(cnn.STRIDE, generator=gen).cuda()

    for n in range(4):
        if n == 2:  # coalition 2 stops: (0, 1) before it, (0, 3) and (0, 2) behind it
            for st in (whole, small):
                st.stop([2])
            live = [ci for ci in live if ci != 2]
            stood = whole.glob[2].clone(), whole.server_m[2].clone()
            small = eng.trainer._compact(small, live)
            place = {ci: i for i, ci in enumerate(live)}
        before = whole.glob.clone()
        for ci in live:
            fill(whole, ci, ci, n)
            fill(small, ci, place[ci], n)
        for st in (whole, small):
            st.aggregate()
        for ci in live:
            if len(coals[ci]) == 1:
                continue
            for t in ("glob", "server_m"):
                assert torch.equal(getattr(whole, t)[ci], getattr(small, t)[place[ci]]), (n, ci, t)
            rows = whole.params[whole.coal_first[ci]:whole.coal_first[ci + 1]]
            assert all(torch.equal(r, whole.glob[ci]) for r in rows)
            w, scale = aggregation_weights([eng.partner_sizes[p] for p in coals[ci]], eng.aggregation)
            members = []
            for k in range(len(coals[ci])):
                gen = torch.Generator().manual_seed(1000 * n + 10 * ci + k)
                members.append((before[ci] + 0.01 * torch.randn(cnn.STRIDE, generator=gen).cuda()).cpu().numpy())
            avg = (sum(m.astype(np.float64) * v for m, v in zip(members, w)) / scale).astype(np.float32)
            b, got, m_got = (t[ci].cpu().numpy() for t in (before, whole.glob, whole.server_m))
            for off, shape in cnn.KERAS_LAYERS:
                if len(shape) == 1:
                    assert np.array_equal(got[off:off + shape[0]], avg[off:off + shape[0]])
            for i, (off, r, c) in enumerate(mats):
                b64, a64, g64, m64 = (v[off:off + r * c].reshape(r, c).astype(np.float64) for v in (b, avg, got, m_got))
                d = (b64 - a64).astype(np.float32).astype(np.float64)
                mom[ci][i] = beta * mom[ci][i] + d
                size[ci][i] = beta * size[ci][i] + np.abs(d)
                assert (np.abs(m64 - mom[ci][i]) <= (n + 1) * 2.0 ** -22 * size[ci][i] + 2.0 ** -30).all(), (n, ci, i)
                step = lr * muon.update_scale(r, c) * exact(d + beta * mom[ci][i])
                want = (1 - lr * wd) * b64 - step
                err = np.linalg.norm(g64 - want)
                assert err <= 2.0 ** -9 * np.linalg.norm(step) + 2.0 ** -22 * np.linalg.norm(want), (n, ci, i, err)
    assert torch.equal(whole.glob[2], stood[0]) and torch.equal(whole.server_m[2], stood[1])


def test_two_streams_give_the_values_of_one():
    """CIFAR10's default of two lockstep batches at once: momenta, workspaces and averages of one do not meet the other's."""
    import itertools
    import numpy as np
    from mplc.dataset import Cifar10
    from mplc.engine import CoalitionEngine
    from mplc.scenario import Scenario
    ds = Cifar10(synthetic=True, n_train=3000, n_test=500, signal=0.3)
    sc = Scenario(6, [0.1, 0.15, 0.15, 0.2, 0.2, 0.2], dataset=ds, epoch_count=1, minibatch_count=3, is_early_stopping=False,
                  server_optimizer="muon").provision()
    eng = CoalitionEngine.for_scenario(sc)
    coals = [c for k in range(1, 7) for c in itertools.combinations(range(6), k)][:40]
    eng.concurrent_batches = 1
    one = eng.evaluate(coals)
    eng.concurrent_batches = 2
    assert eng._concurrent_ok(coals, eng.epoch_count, eng.is_early_stopping, None, False)
    assert np.array_equal(one, eng.evaluate(coals))
    assert len(np.unique(one)) > 5


def test_early_stopping_with_and_without_compaction():
    """Coalitions that stop at different epochs: the same values, epochs and traces whether the batch is kept whole or
    compacted whenever a replica is idle."""
    from itertools import combinations
    import numpy as np
    from mplc.dataset import ArrayDataset, digits_as_mnist
    from mplc.engine import CoalitionEngine
    from mplc.scenario import Scenario
    from test_compaction_gpu import _both, _check
    x, y = digits_as_mnist()
    y = np.argmax(np.array(y), 1)
    rng = np.random.default_rng(0)
    flip = rng.random(1500) < 0.6
    y[np.arange(1500)[flip]] = rng.integers(0, 10, size=int(flip.sum()))
    ds = ArrayDataset(x[:1500], y[:1500], x[1500:], y[1500:])
    sc = Scenario(4, [0.1, 0.2, 0.3, 0.4], dataset=ds, minibatch_count=2, gradient_updates_per_pass_count=16,
                  epoch_count=24, is_early_stopping=True, server_optimizer={"name": "muon", "lr": 0.01}).provision()
    eng = CoalitionEngine.for_scenario(sc, memory_budget_bytes=8 << 30, eval_budget_bytes=1 << 30)
    out = _both(eng, [c for r in range(1, 5) for c in combinations(range(4), r)])
    print(out[0.0][0]["epochs_done"], out[1.0][1])
    _check(out)
