"""Requests that share pages, through the engine: steps over forked requests give the logits of requests with pages of their own, and
many samples of one prompt, with and without drafts, are the plain implementation's tokens, in 32-bit and in bfloat16."""
import ast
import subprocess
import sys

import pytest
import torch

import plain_llama as plain
import tiny

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "bfloat16"]
# logits of two ways through the kernels, of the largest one: 32-bit sums in another order; in bfloat16 each of a few layers rounds its
# attention and its products to 2^-9 once more, the bound that the engine's other tests use against the plain implementation
TOL = {"float32": 2e-5, "bfloat16": 2.5e-2}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for which in ("a", "b", "c", "d", "e"):
        f = tiny.make_model_folder(tmp_path_factory.mktemp(f"smp_{which}"), which, torch.bfloat16)
        out[which] = (f,) + plain.read_model(f)
    return out


def engine(folder, dtype, **kw):
    from hipinfer_b200 import Engine

    return Engine(folder, dtype=dtype, **kw)


def check_greedy(cfg, w, prompt, got, dtype, what):
    """Token identity with the plain implementation; in bfloat16 up to the first place where its two best logits nearly tie."""
    seq = list(prompt)
    logits = plain.forward(cfg, w, seq + list(got))
    for i, t in enumerate(got):
        row = logits[len(seq) - 1 + i]
        if t != plain.argmax_lowest(row):
            top = torch.topk(row.float(), 2).values
            gap = float(top[0] - top[1]) / float(row.abs().max())
            assert dtype == "bfloat16" and gap < 0.02, f"{what}: token {i} is {t} (relative gap {gap:.4f})"
            return


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["a", "c", "d", "e"])
def test_steps_over_forks_are_steps_over_copies(folders, which, dtype):
    """Forks of one prompt with rows of 1 to 21 tokens, cut back and run on, beside a request of its own and forks of a fork."""
    from hipinfer_b200.engine import StepEntry
    from hipinfer_b200.engine.runner import ModelRunner

    folder, cfg, _ = folders[which]
    V = cfg["vocab_size"]
    longest = min(512, cfg["max_position_embeddings"])
    runner = ModelRunner.from_folder(folder, dtype=dtype, page_size=16, num_pages=400, max_num_seqs=20, max_model_len=longest)
    prompt = tiny.random_tokens(longest // 2 + 5, V, 3)
    whole = len(prompt) // 16 * 16
    for rid in ("p", "copy"):
        runner.step([StepEntry(rid, prompt, [])])
    forks = [f"f{i}" for i in range(5)]
    texts = {"p": list(prompt)}
    for i, rid in enumerate(forks):
        assert runner.fork("p", rid) == whole
        texts[rid] = prompt[:whole]
    runner.step([StepEntry("lone", prompt[:7], [])])
    texts["lone"] = prompt[:7]
    for rid in list(texts):                    # the same requests with pages of their own
        runner.step([StepEntry(("own", rid), texts[rid], [])])
    step = 0

    def both(lens):
        nonlocal step
        step += 1
        new = {rid: tiny.random_tokens(n, V, 100 * step + i) for i, (rid, n) in enumerate(lens.items())}
        got = runner.step([StepEntry(r, t, range(len(t))) for r, t in new.items()]).clone()
        for r, t in new.items():
            texts[r] += t
        want = torch.cat([runner.step([StepEntry(("own", r), t, range(len(t)))]).clone() for r, t in new.items()])
        worst = float((got - want).abs().max() / want.abs().max())
        assert torch.isfinite(got).all() and worst <= TOL[dtype], (which, lens, worst)
        runner.cache.check()

    both({"p": 1, "f0": 6, "f1": 21, "lone": 3, "f2": 5, "f3": 1, "f4": 2})
    for rid in ("f1", "f2"):
        texts[rid] = texts[rid][:whole + 2]
        for r in (rid, ("own", rid)):
            runner.truncate(r, whole + 2)
    for graphs in (True, False):               # one token each: replayed from a graph, and with the shared pages read once
        runner.cuda_graphs = graphs
        both({"f0": 1, "f1": 1, "f2": 1, "f3": 1, "f4": 1, "p": 1})
    runner.end("p")                            # the forks keep its pages
    both({"f0": 3, "f1": 18, "f2": 2})
    for rid in ("g0", "g1"):
        runner.step([StepEntry(("own", rid), texts["f1"][:runner.fork("f1", rid)], [])])
        texts[rid] = texts["f1"][:runner.length(rid)]
    both({"f3": 2, "f1": 1, "g0": 4, "g1": 1, "f4": 1})
    for rid in runner.live_requests():
        runner.end(rid)
    runner.cache.check()
    assert runner.cache.free_pages() == [400] and runner.cache.slots.free_count == 20


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which, n_prompt, n, n_new, n_draft", [("a", 5, 3, 12, 0), ("a", 32, 4, 20, 4), ("b", 49, 2, 16, 3), ("b", 1, 3, 9, 2),
                                                                ("c", 150, 6, 24, 5), ("e", 67, 1, 16, 7), ("d", 33, 3, 1, 4)])
def test_greedy_samples_are_the_plain_tokens(folders, which, n_prompt, n, n_new, n_draft, dtype):
    folder, cfg, w = folders[which]
    prompt = tiny.random_tokens(n_prompt, cfg["vocab_size"], 7 + n_prompt)
    if n_draft:                                # something to look up
        prompt = (prompt[:n_prompt // 2] * 2 + prompt)[:n_prompt]
    eng = engine(folder, dtype, max_batch=6, max_seq=256 if which == "c" else 100, max_prefill=16)
    got, logprobs = eng.sample_many(prompt, n, n_new, n_draft=n_draft, logprobs=True)
    eng.runner.cache.check()
    assert eng.runner.cache.slots.free_count == 6 and not eng.runner.live_requests()
    assert len(got) == n and all(len(g) == n_new for g in got) and [len(x) for x in logprobs] == [n_new] * n
    if dtype == "float32":
        assert all(g == got[0] for g in got) and got[0] == eng.generate(prompt, n_new)
    for i, g in enumerate(got):
        check_greedy(cfg, w, prompt, g, dtype, f"{which} {dtype} sample {i}")
        rows = plain.forward(cfg, w, prompt + g)[len(prompt) - 1:-1].double()
        want = torch.log_softmax(rows, -1)[torch.arange(n_new), torch.tensor(g)]
        # (a logarithm of probability moves by twice what the logits move by at most)
        assert float((torch.tensor(logprobs[i], dtype=torch.float64) - want).abs().max()) <= 2 * TOL[dtype] * float(rows.abs().max()) + 1e-4
    eng.close()


def test_drafts_are_accepted_and_save_steps(folders):
    """Greedy continuations of a tiny model soon repeat themselves: with drafts the same tokens take fewer steps."""
    from hipinfer_b200.engine.samples import sample_many

    folder, cfg, w = folders["a"]
    prompt = tiny.random_tokens(20, cfg["vocab_size"], 1)
    eng = engine(folder, "float32", max_batch=4, max_seq=128, max_prefill=64)
    runs = [sample_many(eng, prompt, 2, 80, 0.0, 0, k, (), True) for k in (0, 6)]
    eng.close()
    assert runs[0].outputs == runs[1].outputs and runs[0].steps == 79
    assert runs[1].steps < 60


@pytest.mark.parametrize("dtype", DTYPES)
def test_temperature_samples(folders, dtype):
    """Equal seeds repeat, others differ, samples differ among themselves, and each token's logarithm of probability is the plain
    implementation's at that temperature, with drafts as without."""
    folder, cfg, w = folders["c"]
    prompt = tiny.random_tokens(40, cfg["vocab_size"], 2) * 2
    eng = engine(folder, dtype, max_batch=4, max_seq=256, max_prefill=64)
    for k in (0, 3):
        got, logprobs = eng.sample_many(prompt, 4, 30, temperature=0.7, seed=5, n_draft=k, logprobs=True)
        assert got == eng.sample_many(prompt, 4, 30, temperature=0.7, seed=5, n_draft=k)
        assert got != eng.sample_many(prompt, 4, 30, temperature=0.7, seed=6, n_draft=k)
        assert len({tuple(g) for g in got}) == 4
        for g, lp in zip(got, logprobs):
            rows = plain.forward(cfg, w, prompt + g)[len(prompt) - 1:-1].double() / 0.7
            want = torch.log_softmax(rows, -1)[torch.arange(30), torch.tensor(g)]
            assert float((torch.tensor(lp, dtype=torch.float64) - want).abs().max()) <= 2 * TOL[dtype] * float(rows.abs().max()) + 1e-4
    eng.close()


def test_stop_tokens_and_pages_that_only_sharing_leaves(folders):
    folder, cfg, w = folders["a"]
    prompt = tiny.random_tokens(70, cfg["vocab_size"], 9)
    eng = engine(folder, "float32", max_batch=8, max_seq=128, max_prefill=32, num_pages=20)     # 8 copies of the prompt take 40
    want = eng.generate(prompt, 20)
    assert eng.sample_many(prompt, 8, 20, n_draft=3) == [want] * 8
    stop = want[7]
    cut = want[:want.index(stop) + 1]
    for k in (0, 5):
        assert eng.sample_many(prompt, 3, 20, n_draft=k, stop_token_ids=[stop]) == [cut] * 3
    with pytest.raises(ValueError, match="pages"):
        eng.sample_many(prompt, 8, 58)
    eng.runner.cache.check()
    assert eng.runner.cache.free_pages() == [20]
    assert eng.generate(prompt, 20) == want                  # the scheduler's requests go on as before
    eng.close()


def test_refusals(folders, tmp_path):
    import torirax_models

    folder, cfg, _ = folders["a"]
    eng = engine(folder, "float32", max_batch=2, max_seq=64)
    good = dict(prompt=[1, 2, 3], n=2, n_new=4)
    for bad in (dict(prompt=[]), dict(prompt=[-1]), dict(prompt=[cfg["vocab_size"]]), dict(n=0), dict(n=3), dict(n_new=0), dict(n_new=62),
                dict(temperature=-1.0), dict(n_draft=-1), dict(n_draft=64)):
        with pytest.raises(ValueError):
            eng.sample_many(**{**good, **bad})
    assert len(eng.sample_many(**good)) == 2
    eng.close()
    state, _, _ = torirax_models.make_folder(tmp_path / "state", "p", seed=1, dtype=torch.float32)
    eng = engine(state, "float32", max_batch=2, max_seq=64)
    with pytest.raises(ValueError, match="state"):
        eng.sample_many(**good)
    eng.close()


def test_command_line(folders):
    folder, cfg, w = folders["b"]
    prompt = tiny.random_tokens(19, cfg["vocab_size"], 5)
    r = subprocess.run([sys.executable, "-m", "hipinfer_b200", "generate", "--model", folder, "--tokens", *map(str, prompt), "--new", "6",
                        "--mode", "fp32", "--max-seq", "64", "--max-batch", "3", "--samples", "3", "--drafts", "2"], capture_output=True,
                       text=True, timeout=600, cwd=tiny.ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [ast.literal_eval(x) for x in r.stdout.strip().splitlines()[-3:]]
    want, _ = plain.generate_greedy(cfg, w, prompt, 6)
    assert lines == [want] * 3
