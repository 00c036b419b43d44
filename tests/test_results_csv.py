"""CPU: results.csv of an experiment whose scenarios differ in their columns (main.py, mplc.utils.append_results)."""
import types

import numpy as np
import pandas as pd

from mplc import scenario, utils


def test_scenarios_with_and_without_a_server_optimizer(tmp_path, monkeypatch):
    """One YAML, server_optimizer: [null, muon]: every value under its own column."""
    import main

    def run(self):
        self.mpl = types.SimpleNamespace(history=types.SimpleNamespace(score=0.5, nb_epochs_done=1), learning_computation_time=2.0)
        self.nb_samples_used, self.final_relative_nb_samples = 10, [0.5, 0.5]
        self.append_contributivity(types.SimpleNamespace(
            name="Independent scores", contributivity_scores=np.array([0.25, 0.75]), scores_std=np.zeros(2),
            computation_time_sec=1.0, first_charac_fct_calls_count=2))
    monkeypatch.setattr(scenario.Scenario, "run", run)
    monkeypatch.setattr(main, "validate_scenario_list", lambda *a: None)
    monkeypatch.setenv("MPLC_SYNTHETIC_DATA", "1")
    monkeypatch.chdir(tmp_path)
    (tmp_path / "c.yml").write_text(
        "experiment_name: e\nn_repeats: 2\nscenario_params_list:\n  - dataset_name: [mnist]\n    partners_count: [2]\n"
        "    amounts_per_partner: [[0.5, 0.5]]\n    methods: [[Independent scores]]\n"
        "    server_optimizer: [null, {name: muon, lr: 0.05}]\n")
    assert main.main(["-f", "c.yml"]) == 0
    utils.logger.handlers.clear()  # the experiment folder's log files
    out = list(tmp_path.glob("experiments/*/results.csv"))
    df = pd.read_csv(out[0])
    assert len(df) == 2 * 2 * 2 and list(df["partner_id"]) == [0, 1] * 4
    assert list(df["contributivity_method"].unique()) == ["Independent scores"]
    assert list(df["contributivity_score"]) == [0.25, 0.75] * 4 and list(df["scenario_id"]) == [0, 0, 1, 1] * 2
    with_it = df["server_optimizer"].notna()
    assert list(with_it) == [False, False, True, True] * 2 and "muon" in df["server_optimizer"][2]
    assert list(df["random_state"]) == [0] * 4 + [1] * 4


def test_rows_that_lack_columns_and_quoted_values(tmp_path):
    f = tmp_path / "results.csv"
    a = pd.DataFrame({"x": [1, 2], "text": ['a, "b"\nc', ""]})
    utils.append_results(f, a)
    assert f.read_text() == a.to_csv(index=False)
    utils.append_results(f, a)  # the same columns: rows as they were written before
    assert f.read_text() == a.to_csv(index=False) + a.to_csv(index=False, header=False)
    utils.append_results(f, pd.DataFrame({"more": [[0.5, 0.25]], "x": [3]}))
    utils.append_results(f, pd.DataFrame({"x": [4]}))
    df = pd.read_csv(f, keep_default_na=False)
    assert list(df.columns) == ["x", "text", "more"] and list(df["x"]) == [1, 2, 1, 2, 3, 4]
    assert list(df["text"]) == ['a, "b"\nc', ""] * 2 + ["", ""] and list(df["more"]) == [""] * 4 + ["[0.5, 0.25]", ""]
