"""The memory budget of lockstep batches with a server optimizer: its rows and its step's workspace are counted."""
import ctypes
import itertools

import numpy as np
import pytest


def engine(model, budget, streams, optimizer="muon"):
    """A CoalitionEngine's planner alone (no device)."""
    from mplc import engine as e
    from mplc.muon import ServerMuon
    eng = object.__new__(e.CoalitionEngine)
    eng.model_impl = e.model_class(model)()
    eng.batch_sizes = [4] * 10
    eng.memory_budget_bytes = budget
    eng.concurrent_batches = streams
    eng.server_optimizer, eng._server_step = (ServerMuon(optimizer) if optimizer else None), None
    return eng


def step_workspaces(model, models):
    """Bytes of workspace of one group's steps, every matrix's by its own query."""
    from mplc import muon
    out = []
    for _, rows, cols in muon.ServerMuon.matrices(model.KERAS_LAYERS):
        t = muon.MuonT()
        t.n_models, t.rows, t.cols, t.steps, t.invariant = min(models, muon.ServerMuon.GROUP), rows, cols, 5, 1
        out.append(int(muon._lib().mplc_muon_step_workspace_bytes(ctypes.byref(t))))
    return out


@pytest.mark.parametrize("streams", [1, 2])
@pytest.mark.parametrize("model", ["mnist_cnn", "cifar10_cnn"])
def test_planned_batches_fit_with_the_steps_workspace(model, streams):
    coals = [c for k in range(1, 11) for c in itertools.combinations(range(10), k)]
    for budget in (1 << 30, 4 << 30, 16 << 30):
        eng = engine(model, budget, streams)
        batches = eng.plan_batches(coals)
        assert sorted(i for b in batches for i in b) == list(range(len(coals))) and len(batches) > 1
        stride = eng.model_impl.STRIDE
        for b in batches:
            rows = sum(len(coals[i]) * eng.replica_bytes(4) for i in b)
            n = len(b)  # dealt to the streams; coalition rows, momenta, rows at the round's start, differences of the groups in work
            rows += 4 * stride * (3 * n + min(n, 64 * streams))
            per = -(-n // streams)
            if n > 1:
                assert rows + sum(max(step_workspaces(eng.model_impl, (n + k) // streams)) for k in range(streams)) <= budget
    plain = engine(model, 4 << 30, streams, None)
    assert plain.server_bytes(100) == 0


@pytest.mark.gpu
def test_two_stream_batches_with_a_server_optimizer_stay_within_the_budget():
    """Peak reserved memory above the data: training budget, evaluation budget and the allocator's rounding."""
    import torch
    from mplc.dataset import Cifar10
    from mplc.engine import CoalitionEngine
    from mplc.scenario import Scenario
    ds = Cifar10(synthetic=True, n_train=1200, n_test=300, signal=0.3)
    sc = Scenario(6, [0.1, 0.15, 0.15, 0.2, 0.2, 0.2], dataset=ds, epoch_count=1, minibatch_count=2,
                  gradient_updates_per_pass_count=8, is_early_stopping=False, server_optimizer="muon").provision()
    coals = [c for k in range(2, 7) for c in itertools.combinations(range(6), k)]
    probe = CoalitionEngine.for_scenario(sc)
    whole = sum(len(c) * probe.replica_bytes(max(probe.batch_sizes[p] for p in c)) for c in coals)
    del probe
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    budget, eval_budget = int(1.15 * whole), 64 << 20  # every coalition in one batch, were the step's memory not counted
    eng = CoalitionEngine.for_scenario(sc, memory_budget_bytes=budget, eval_budget_bytes=eval_budget)
    assert eng.concurrent_batches == 2 and len(eng.plan_batches(coals)) > 1
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    v = eng.evaluate(coals)
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_reserved() - base
    print(f"budget {budget >> 20} MiB + eval {eval_budget >> 20} MiB, peak reserved above the data {peak >> 20} MiB")
    assert np.isfinite(v).all()
    assert peak <= 1.1 * (budget + eval_budget) + (64 << 20), (peak, budget)
