"""The cache in 8 bits through the engine: logits against a plain model that stores and reads its cache as the operators' formulas say, in
portions of any size; forks inside a page; many samples of one prompt; the commands.

Tolerances, of the largest logit. The plain model's keys and values differ from the engine's by their own rounding, and where one stands next to the
middle between two codes the two round apart, by a whole step: 2^-6 of a number at most for int8 (1 / 127 of its block's largest) and 2^-3 of it for
e4m3. In 32 bits (numbers off by some 2^-20, a step of 2^-7) that is one number in some thousands, in a result that averages all of a row's keys and
dimensions; 2e-3 allows for one of them at full weight. In bfloat16 numbers are off by 2^-9 and every fourth int8 code may differ by one: noise of
half a step, 2^-8 of a block's largest, or what two or three more roundings to bfloat16 are; the bound is the one that steps over shared pages have."""
import subprocess
import sys

import pytest
import torch

import plain_cache8
import plain_llama as plain
import tiny

pytestmark = pytest.mark.gpu
TOL = {"float32": 2e-3, "bfloat16": 2.5e-2}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {}
    for which in ("a", "b", "c", "d", "e"):
        f = tiny.make_model_folder(tmp_path_factory.mktemp(f"c8_{which}"), which, torch.bfloat16)
        out[which] = (f,) + plain.read_model(f)
    return out


class Plain8:
    """One request of the plain model over a cache in 8 bits, in pages one after the other."""

    def __init__(self, cfg, weights, codes, page_size=16):
        self.cfg, self.w, self.ps, self.length = cfg, weights, page_size, 0
        self.D, self.Hq, self.Hkv = plain.head_dim_of(cfg), cfg["num_attention_heads"], plain.kv_heads_of(cfg)
        pages, blocks = -(-cfg["max_position_embeddings"] // page_size), -(-page_size // 16)
        self.cache = [[(torch.zeros(pages, self.Hkv, page_size, self.D, dtype=torch.uint8).view(codes), torch.zeros(pages, self.Hkv, blocks))
                       for _ in range(2)] for _ in range(cfg["num_hidden_layers"])]

    def step(self, tokens):
        c, w = self.cfg, self.w
        T, at = len(tokens), list(range(self.length, self.length + len(tokens)))
        eps = c.get("rms_norm_eps", 1e-6)
        cos, sin = plain.rope_cos_sin(at, plain.rope_inv_freq(self.D, c.get("rope_theta", 10000.0), c.get("rope_scaling")))
        x = plain.embed(tokens, w["model.embed_tokens.weight"])
        for layer in range(c["num_hidden_layers"]):
            p = f"model.layers.{layer}."
            xn = plain.rmsnorm(x, w[p + "input_layernorm.weight"], eps)
            q, k, v = (xn @ w[p + f"self_attn.{n}_proj.weight"].T for n in "qkv")
            q, k = (plain.apply_rope(y.reshape(T, -1, self.D), cos, sin) for y in (q, k))
            self.cache[layer] = [plain_cache8.store(rows.reshape(T, -1), at, *plane) for rows, plane in zip((k, v), self.cache[layer])]
            keys, values = (torch.from_numpy(plain_cache8.numbers(*plane)).float().transpose(1, 2).reshape(-1, self.Hkv, self.D)[:at[-1] + 1]
                            for plane in self.cache[layer])
            o = plain.attention_scores_softmax_values(q, keys, values, at, range(at[-1] + 1))
            x = x + o.reshape(T, -1) @ w[p + "self_attn.o_proj.weight"].T
            xn = plain.rmsnorm(x, w[p + "post_attention_layernorm.weight"], eps)
            x = x + plain.swiglu_mlp(xn, *(w[p + f"mlp.{n}_proj.weight"] for n in ("gate", "up", "down")))
        self.length += T
        head = w["model.embed_tokens.weight"] if c.get("tie_word_embeddings", False) else w["lm_head.weight"]
        return plain.lm_head(x, w["model.norm.weight"], head, eps)


def runner_of(folder, dtype, codes, **kw):
    from hipinfer_b200.engine.runner import ModelRunner

    return ModelRunner.from_folder(folder, dtype=dtype, cache_dtype=codes, **{**dict(page_size=16, num_pages=200, max_num_seqs=8, max_model_len=None), **kw})


CUTS = [("a", [7, 1, 1, 30, 2, 1, 1, 1]), ("b", [40, 1, 17, 1, 1]), ("c", [70, 1, 1, 33, 1, 1, 5, 1]), ("c", [300, 1, 1, 1]), ("d", [21, 1, 40, 1]), ("e", [33, 1, 1])]


@pytest.mark.parametrize("which, cuts, page_size", [(w, c, 16) for w, c in CUTS] + [(w, c, ps) for w, c in (CUTS[0], CUTS[2]) for ps in (64, 8)])
@pytest.mark.parametrize("dtype, codes", [("float32", "int8"), ("float32", "float8_e4m3fn"), ("bfloat16", "int8")])
def test_logits_are_those_of_a_plain_model_over_such_a_cache(folders, which, cuts, page_size, dtype, codes):
    from hipinfer_b200.engine import StepEntry
    from hipinfer_b200.engine.runner import cache8_dtype

    folder, cfg, w = folders[which]
    runner, want = runner_of(folder, dtype, codes, page_size=page_size), Plain8(cfg, w, cache8_dtype(codes), page_size)
    tokens, at = tiny.random_tokens(sum(cuts), cfg["vocab_size"], 5), 0
    for i, n in enumerate(cuts):
        part = tokens[at:at + n]
        at += n
        entries = [StepEntry("r", part, range(n))]
        if i == 1:                                                       # beside another request
            entries.append(StepEntry("other", tokens[:9], [8]))
        got, ref = runner.step(entries)[:n].float().cpu(), want.step(part)
        err = float((got - ref).abs().max()) / float(ref.abs().max())
        assert err <= TOL[dtype], f"portion {i} of {n}: {err:.2e}"


@pytest.mark.parametrize("codes", [None, "int8", "float8_e4m3fn"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forks_inside_a_page_go_on_as_their_parent_does(folders, dtype, codes):
    """Bit for bit: steps of one request each, the same tokens."""
    from hipinfer_b200.engine import StepEntry

    folder, cfg, _ = folders["c"]
    runner = runner_of(folder, dtype, codes)
    text = tiny.random_tokens(60, cfg["vocab_size"], 9)
    runner.step([StepEntry("p", text[:45], [])])
    assert runner.fork("p", "x", 45) == 45 and runner.fork("p", "y", 45) == 45 and runner.fork("p", "short", 37) == 37
    runner.cache.check()
    for t in text[45:]:
        rows = [runner.step([StepEntry(r, [t], [0])]).clone() for r in ("y", "p", "x")]
        assert torch.equal(rows[0], rows[1]) and torch.equal(rows[2], rows[1])
    a = runner.step([StepEntry("short", text[37:45], [7])]).float()
    assert torch.isfinite(a).all()
    runner.end("p")
    runner.cache.check()
    assert runner.fork("x", "z", 50) == 50
    for r in ("x", "y", "z", "short"):
        runner.end(r)
    assert runner.cache.free_pages() == [200]


def test_a_fork_with_no_page_left_changes_nothing(folders):
    from hipinfer_b200.cache import OutOfPages
    from hipinfer_b200.engine import StepEntry

    runner = runner_of(folders["c"][0], "bfloat16", "int8", num_pages=3)
    runner.step([StepEntry("p", list(range(40)), [])])
    with pytest.raises(OutOfPages):
        runner.fork("p", "x", 40)
    assert not runner.cache.has_request("x") and runner.fork("p", "y", 32) == 32
    runner.cache.check()


@pytest.mark.parametrize("n_draft", [0, 3])
@pytest.mark.parametrize("n_prompt", [37, 48, 5])
def test_greedy_samples_are_what_generate_gives(folders, n_prompt, n_draft):
    from hipinfer_b200 import Engine

    folder, cfg, _ = folders["c"]
    eng = Engine(folder, dtype="float32", max_batch=5, max_seq=256, cache_dtype="int8")
    assert eng.kv_bytes_per_token == 2 * 2 * 2 * (64 + 4 / 16)
    prompt = tiny.random_tokens(n_prompt, cfg["vocab_size"], 3)
    want = eng.generate(prompt, 14)
    for got in eng.sample_many(prompt, 4, 14, n_draft=n_draft):
        assert got == want
    assert eng.runner.cache.free_pages() == [eng.runner.cache.pools[0].num_pages]
    drawn = eng.sample_many(prompt, 4, 14, temperature=0.9, seed=2, n_draft=n_draft)
    assert drawn == eng.sample_many(prompt, 4, 14, temperature=0.9, seed=2, n_draft=n_draft) and len({tuple(t) for t in drawn}) > 1
    eng.close()


def test_decoding_from_graphs_beside_eager_steps(folders):
    """The same requests with and without graphs (their launches are cut for longer positions): the same logits up to the last bits' order."""
    from hipinfer_b200.engine import StepEntry

    folder, cfg, _ = folders["c"]
    a, b = (runner_of(folder, "bfloat16", "int8", cuda_graphs=g) for g in (True, False))
    prompts = [tiny.random_tokens(n, cfg["vocab_size"], n) for n in (20, 333, 64)]
    for r in (a, b):
        r.step([StepEntry(i, p, []) for i, p in enumerate(prompts)])
    for s in range(20):
        tokens = tiny.random_tokens(3, cfg["vocab_size"], 50 + s)
        x, y = (r.step([StepEntry(i, [t], [0]) for i, t in enumerate(tokens)]).float() for r in (a, b))
        assert float((x - y).abs().max()) <= TOL["bfloat16"] * float(y.abs().max())


def test_a_scheduled_batch_with_preemption(folders):
    from hipinfer_b200 import Engine

    folder, cfg, _ = folders["c"]
    prompts = [tiny.random_tokens(n, cfg["vocab_size"], n) for n in (30, 60, 45, 20)]
    roomy = Engine(folder, dtype="float32", max_batch=4, max_seq=128, cache_dtype="int8")
    tight = Engine(folder, dtype="float32", max_batch=4, max_seq=128, cache_dtype="int8", num_pages=13)
    want = roomy.generate(prompts, 24)
    got = tight.generate(prompts, 24)
    # (a request that comes back runs its text as one portion: its blocks are stored at once, not token by token, so its tokens may part from the others')
    assert [len(t) for t in got] == [24] * 4 and sum(a == b for a, b in zip(got, want)) >= 1
    tight.runner.cache.check()
    for e in (roomy, tight):
        e.close()


def test_other_models_and_names_are_refused(tmp_path):
    import torirax_models as tm
    from hipinfer_b200 import Engine

    folder, cfg, _ = tm.make_folder(tmp_path, "p", seed=7, dtype=torch.float32)
    with pytest.raises(ValueError, match="8 bits"):
        Engine(folder, cache_dtype="int8", max_batch=1, max_seq=64)
    with pytest.raises(ValueError, match="cache type"):
        Engine(config=tiny.TINY_A, random_weights=0, cache_dtype="int4", max_batch=1, max_seq=64)


def test_the_commands(folders, tmp_path):
    folder, cfg, _ = folders["c"]
    out = subprocess.run([sys.executable, "-m", "hipinfer_b200", "generate", "--model", folder, "--tokens", "1", "2", "3", "--new", "5", "--cache-dtype", "fp8"],
                         check=True, capture_output=True, text=True, cwd=tiny.ROOT).stdout
    assert len(eval(out.strip().splitlines()[-1])) == 5
    trace = '{"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [0, 2]}], "end": ["a"]}\n'
    subprocess.run([sys.executable, "-m", "hipinfer_b200", "replay", "--model", folder, "--dtype", "float32", "--out", str(tmp_path), "--max-tokens", "64",
                    "--page-size", "8", "--cache-dtype", "int8"], check=True, input=trace, text=True, cwd=tiny.ROOT, capture_output=True)
    from hipinfer_b200.engine.runner import cache8_dtype

    got = torch.frombuffer(bytearray((tmp_path / "0.f32").read_bytes()), dtype=torch.float32).view(2, -1)
    ref = Plain8(cfg, folders["c"][2], cache8_dtype("int8"), 8).step([5, 17, 3])[[0, 2]]
    assert float((got - ref).abs().max()) <= TOL["float32"] * float(ref.abs().max())
