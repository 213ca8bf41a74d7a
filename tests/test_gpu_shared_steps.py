"""Which steps of forked requests give up their graph for attention over the shared pages: those of models whose attention reads them so."""
import pytest
import torch

import selovik_models
import tiny

pytestmark = pytest.mark.gpu


def one_token_each(folder, monkeypatch, longest):
    """A decode-only step of a request and three forks, with nothing asked of what sharing saves; the runner, and how many plans were made."""
    from hipinfer_b200.engine import StepEntry
    from hipinfer_b200.engine.runner import ModelRunner
    from hipinfer_b200.kernels import ops

    plans = []
    real = ops.SharedPlan
    monkeypatch.setattr(ops, "SharedPlan", lambda *a, **kw: plans.append(a) or real(*a, **kw))
    monkeypatch.setattr(ModelRunner, "SHARED_STEP_BYTES", 1)
    runner = ModelRunner.from_folder(folder, dtype="float32", page_size=16, num_pages=64, max_num_seqs=8, max_model_len=longest)
    V = runner.vocab_size
    runner.step([StepEntry("p", tiny.random_tokens(32, V, 3), [])])
    for rid in ("f0", "f1", "f2"):
        runner.step([StepEntry(("own", rid), tiny.random_tokens(32, V, 3)[:runner.fork("p", rid)], [])])
    got = runner.step([StepEntry(r, [5], [0]) for r in ("f0", "f1", "f2")]).clone()
    graphs = len(runner._graphs)
    want = runner.step([StepEntry(("own", r), [5], [0]) for r in ("f0", "f1", "f2")]).clone()
    assert float((got - want).abs().max()) <= 2e-5 * float(want.abs().max())
    return graphs, len(plans)


def test_a_model_whose_attention_shares_reads_runs_eagerly(tmp_path, monkeypatch):
    folder = tiny.make_model_folder(tmp_path, "a", torch.bfloat16)
    assert one_token_each(folder, monkeypatch, 64) == (0, 1)


def test_a_model_of_another_attention_keeps_its_graph(tmp_path, monkeypatch):
    """(The samples share its memory; their reads are their own.)"""
    folder = selovik_models.make_folder(tmp_path, "d", seed=1, dtype=torch.float32)[0]
    assert one_token_each(folder, monkeypatch, 64) == (1, 0)
