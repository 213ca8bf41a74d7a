"""Drafts that are refused over a cache in 8 bits: what is stored afterwards, bit for bit, and the logits behind a draft that stands out.

The bound of the logits is that of the engine's other tests in 32 bits (2e-3 of the largest: a number next to the middle between two codes may round to either side where
steps of other sizes computed it)."""
import pytest
import torch

import tiny
from hipinfer_b200.kernels import ops
from test_gpu_cache8_engine import TOL, folders, runner_of

pytestmark = pytest.mark.gpu


def planes(runner):
    n = runner.cache.pools[0].num_pages                              # (those that are handed out)
    return [t[:, :n].clone() for t in runner.storage.kv[0].values()]


def same(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("codes", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page_size", [16, 64, 8])
def test_the_cache_is_what_the_kept_rows_alone_leave(folders, dtype, codes, page_size):
    from hipinfer_b200.engine import StepEntry

    folder, cfg, _ = folders["c"]
    runner = runner_of(folder, dtype, codes, page_size=page_size)
    held, n, keep = [37, 20, 5, 64, 15], [6, 4, 20, 5, 3], [2, 4, 13, 1, 2]      # (the second keeps all of its drafts, the fourth begins a block)
    for r, h in enumerate(held):
        runner.step([StepEntry(r, tiny.random_tokens(h, cfg["vocab_size"], r), [])])
    before = planes(runner)
    runner.step([StepEntry(r, tiny.random_tokens(m, cfg["vocab_size"], 90 + r), range(m)) for r, m in enumerate(n)], drafts=True)
    rows, slots = list(runner._kept.rows), runner._kept.slot_maps
    tables = [list(runner.cache.block_table(r, 0)) for r in range(5)]
    for r, (h, k) in enumerate(zip(held, keep)):
        runner.truncate(r, h + k)
    runner.store_accepted()
    after = planes(runner)
    runner.store_accepted()                                          # (nothing is left to be done)
    assert same(after, planes(runner)) and len(rows) == cfg["num_hidden_layers"]
    kept = torch.tensor([s if i < k else -1 for r, k in enumerate(keep) for i, s in enumerate(slots[r][0])], dtype=torch.int32, device="cuda:0")
    names = list(runner.storage.kv[0])
    for layer, (_, k, v) in enumerate(rows):
        want = dict(zip(names, [t[layer].contiguous() for t in before]))
        ops.store_cache8(k, v, kept, ops.Cache8(*(want[x] for x in ("k", "v", "k_scale", "v_scale"))))
        got = dict(zip(names, [t[layer] for t in after]))
        for r, (h, m) in enumerate(zip(held, keep)):                 # every place that a request holds, and its block's scale
            for p in range(h + m):
                page, place = tables[r][p // page_size], p % page_size
                for x in "kv":
                    assert torch.equal(want[x][page, :, place].view(torch.uint8), got[x][page, :, place].view(torch.uint8))
                    assert torch.equal(want[x + "_scale"][page, :, place // 16], got[x + "_scale"][page, :, place // 16])


@pytest.mark.parametrize("codes", ["int8", "float8_e4m3fn"])
def test_a_refused_draft_that_stands_out_leaves_nothing_behind(folders, codes):
    """A token whose values are many times those of the others, drafted and refused: the logits behind it are those of a run that never saw it."""
    from hipinfer_b200.engine import StepEntry

    from hipinfer_b200.config import config_from_dict
    from hipinfer_b200.engine.runner import ModelRunner

    _, cfg, w = folders["c"]
    w = {name: t.clone().cuda() for name, t in w.items()}
    # token 3 has its all in one dimension, which the first layer's values make much of
    w["model.embed_tokens.weight"][3] = 0
    w["model.embed_tokens.weight"][3, 0] = 1
    w["model.layers.0.self_attn.v_proj.weight"][:, 0] *= 20
    text, far = [t if t != 3 else 4 for t in tiny.random_tokens(60, cfg["vocab_size"], 9)], []
    for undo in (True, False):
        drafted, alone = (ModelRunner(config_from_dict(cfg), dict(w), dtype="float32", cache_dtype=codes, page_size=16, num_pages=20, max_num_seqs=2) for _ in range(2))
        for r in (drafted, alone):
            r.step([StepEntry("p", text[:37], [])])
        drafted.step([StepEntry("p", [text[37], 3, 3, 5], range(4))], drafts=True)
        alone.step([StepEntry("p", [text[37]], [0])])
        drafted.truncate("p", 38)
        if undo:
            drafted.store_accepted()
        worst = 0.0
        for t in text[38:47]:
            a, b = (r.step([StepEntry("p", [t], [0])]).float() for r in (drafted, alone))
            worst = max(worst, float((a - b).abs().max() / b.abs().max()))
        far.append(worst)
    assert far[0] <= TOL["float32"] and far[1] > 2 * far[0], far


def test_requests_that_end_before_the_kept_rows_are_stored_touch_nothing(folders):
    """Their pages are free, or another request's of the same name."""
    from hipinfer_b200.engine import StepEntry

    folder, cfg, _ = folders["c"]
    runner = runner_of(folder, "bfloat16", "int8")
    text = tiny.random_tokens(60, cfg["vocab_size"], 9)
    runner.step([StepEntry("a", text[:37], []), StepEntry("b", text[:45], []), StepEntry("c", text[:50], [])])
    runner.step([StepEntry("a", text[37:41], range(4)), StepEntry("b", text[45:49], range(4))], drafts=True)
    for r in ("a", "b"):
        runner.end(r)
    assert runner.fork("c", "a", 39) == 39                          # (its copy lies where one of them ended)
    before = planes(runner)
    runner.store_accepted()
    assert same(before, planes(runner))
