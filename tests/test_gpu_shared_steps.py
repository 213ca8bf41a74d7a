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


@pytest.mark.parametrize("dtype, tol", [("float32", 2e-5), ("bfloat16", 2.5e-2)])
def test_eager_steps_over_forks_with_heads_of_128(monkeypatch, dtype, tol):
    """Rows of 1 to 30 tokens beside each other, drafts among them taken back, against requests with pages of their own. (The bounds are those of
    the smaller heads' test.)"""
    from hipinfer_b200.config import config_from_dict
    from hipinfer_b200.engine import StepEntry
    from hipinfer_b200.engine.runner import ModelRunner
    from hipinfer_b200.kernels import ops

    plans = []
    real = ops.SharedPlan
    monkeypatch.setattr(ops, "SharedPlan", lambda *a, **kw: plans.append(real(*a, **kw)) or plans[-1])
    config = config_from_dict(dict(tiny.TINY_C, num_attention_heads=12, num_key_value_heads=4, head_dim=128, num_hidden_layers=3))
    runner = ModelRunner.from_random(config, seed=3, std=0.05, dtype=dtype, page_size=16, num_pages=400, max_num_seqs=16, max_model_len=1000,
                                     cuda_graphs=False)
    V, prompt = runner.vocab_size, tiny.random_tokens(530, 1000, 3)
    texts = {"p": list(prompt)}
    runner.step([StepEntry("p", prompt, [])])
    for i in range(5):
        texts[f"f{i}"] = prompt[:runner.fork("p", f"f{i}")]
    for rid, tokens in texts.items():
        runner.step([StepEntry(("own", rid), tokens, [])])
    for step, lens in enumerate([dict(p=1, f0=3, f1=18, f2=5, f3=30, f4=19), dict(f0=1, f1=1, f2=1, f3=1, f4=1, p=1), dict(f0=5, f1=5, f2=2, f4=7)]):
        new = {rid: tiny.random_tokens(n, V, 10 * step + i) for i, (rid, n) in enumerate(lens.items())}
        before = len(plans)
        got = runner.step([StepEntry(r, t, range(len(t))) for r, t in new.items()]).clone()
        assert len(plans) == before + 1 and plans[-1].tensor_cores == (dtype == "bfloat16")
        want = torch.cat([runner.step([StepEntry(("own", r), t, range(len(t)))]).clone() for r, t in new.items()])
        assert float((got - want).abs().max()) <= tol * float(want.abs().max())
        for r in new:
            for rid in (r, ("own", r)):
                runner.truncate(rid, runner.length(rid) - lens[r] // 3)
    runner.cache.check()
