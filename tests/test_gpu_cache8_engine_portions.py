"""The engine's prompts over a cache in 8 bits with their portions on the flash kernel (the limit is set here): logits against the plain model over such a cache, within the
bound of the engine's other tests (test_gpu_cache8_engine.py), which is int8's.

For e4m3 the bound is twice that. Where the engine's number and the plain model's are d apart, and codes s, they round to different codes with probability d / s, and are then s
apart: an error whose root mean square is sqrt(d / s) s = sqrt(d s). d is the same for both code types. A number x has e4m3's s between 2^-4 |x| and 2^-3 |x|, some 2^-3.5 of it; int8's is 1 / 127
of its block's largest, 3.2 times the numbers' root mean square among 1,024 of them: 2^-5.3 of that. sqrt(2^-3.5 / 2^-5.3) = 1.9."""
import pytest

import tiny
from hipinfer_b200.kernels import cache8
from test_gpu_cache8_engine import TOL, Plain8, folders, runner_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which, cuts, page_size", [("c", [300, 1, 1, 40, 1], 16), ("c", [70, 129, 1, 16, 2], 64), ("c", [33, 17, 250, 1], 32)])
@pytest.mark.parametrize("codes", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("some_at_a_time", [False, True])
def test_logits_behind_portions(folders, which, cuts, page_size, codes, some_at_a_time, monkeypatch):
    from hipinfer_b200.engine import StepEntry
    from hipinfer_b200.engine.runner import cache8_dtype

    folder, cfg, w = folders[which]
    made, real = [], cache8._Portions
    monkeypatch.setattr(cache8, "_portion_limit", lambda *a: 16)
    monkeypatch.setattr(cache8, "_Portions", lambda *a: made.append(a[-1]) or real(*a))
    if some_at_a_time:
        monkeypatch.setattr(cache8, "PORTION_BYTES", 1)
    runner, want = runner_of(folder, "bfloat16", codes, page_size=page_size), Plain8(cfg, w, cache8_dtype(codes), page_size)
    tokens, at = tiny.random_tokens(sum(cuts), cfg["vocab_size"], 5), 0
    for i, n in enumerate(cuts):
        part = tokens[at:at + n]
        at += n
        entries = [StepEntry("r", part, range(n))]
        if i == 1:                                                       # beside other requests
            entries += [StepEntry("other", tokens[:9], [8]), StepEntry("third", tokens[:50], [49])]
        before = len(made)
        got, ref = runner.step(entries)[:n].float().cpu(), want.step(part)
        # (laid out at the first layer, for each of the step's portions or for all together)
        long = sum(len(e.tokens) >= 16 for e in entries)
        assert len(made) - before == (long if some_at_a_time else min(long, 1))
        assert float((got - ref).abs().max()) / float(ref.abs().max()) <= TOL["bfloat16"] * (2 if codes != "int8" else 1), f"portion {i} of {n}"
