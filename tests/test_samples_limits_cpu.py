"""Engine.sample_many's limits, with a runner that only counts (no GPU)."""
import math
from types import SimpleNamespace

import pytest

from hipinfer_b200.engine import samples


def engine(**kw):
    return SimpleNamespace(**{**dict(vocab=100, max_seq=512, max_prefill=64, runner=None), **kw})


@pytest.mark.parametrize("temperature", [math.nan, -1.0, -math.inf])
def test_a_temperature_that_is_none_is_refused(temperature):
    with pytest.raises(ValueError, match="temperature"):
        samples.sample_many(engine(), [1, 2], 2, 4, temperature, 0, 0, (), True)


class CountingRunner:
    """Keeps requests' lengths and every step's rows and wanted rows."""

    def __init__(self, slots):
        self.lengths, self.steps, self.page_size, self.device, self.vocab_size = {}, [], 16, "cpu", 100
        self.model, self.spec = SimpleNamespace(state_specs={}), SimpleNamespace(eos_token_ids=())
        self.cache = SimpleNamespace(groups=[], has_request=self.lengths.__contains__, slots=SimpleNamespace(free_count=slots))

    def length(self, rid):
        return self.lengths.get(rid, 0)

    def step(self, entries):
        assert len({e.request_id for e in entries}) == len(entries)
        self.steps.append((sum(len(e.tokens) for e in entries), sum(len(list(e.want)) for e in entries)))
        for e in entries:
            self.lengths[e.request_id] = self.length(e.request_id) + len(e.tokens)

    def fork(self, rid, new):
        self.lengths[new] = self.length(rid) // self.page_size * self.page_size

    def truncate(self, rid, length):
        assert 0 < length <= self.lengths[rid]
        self.lengths[rid] = length

    def end(self, rid):
        del self.lengths[rid]


@pytest.mark.parametrize("n_prompt, n, n_draft, max_prefill", [(50, 64, 63, 128), (15, 40, 4, 64), (31, 8, 0, 8), (16, 5, 3, 5), (33, 20, 2, 7), (7, 3, 63, 1),
                                                               (300, 1, 9, 16), (47, 8, 4, 1024)])
def test_a_step_keeps_to_the_token_budget(monkeypatch, n_prompt, n, n_draft, max_prefill):
    """However many samples and drafts; every sample is there in full, and within the budget a step is one."""
    monkeypatch.setattr(samples.torch, "Generator", lambda device: SimpleNamespace(manual_seed=lambda seed: None))
    drawn = []

    def take(self, logits, starts, drafts, live):
        drawn.append(([len(d) for d in drafts], list(live)))
        assert len(starts) == len(drafts) == len(live)
        for i, d in zip(live, drafts):         # one draft is kept of those that there are
            new = ([7] * (1 + (len(d) > 0)))[:self.n_new - len(self.outputs[i])]
            self.texts[i].extend(new)
            self.outputs[i] += new
            self.logprobs[i] += [0.0] * len(new)

    monkeypatch.setattr(samples.Sampling, "_take", take)
    monkeypatch.setattr(samples.DraftLookup, "propose", lambda self, k: [7] * k)
    runner = CountingRunner(n)
    call = samples.sample_many(engine(runner=runner, max_prefill=max_prefill), [1] * n_prompt, n, 12, 0.0, 0, n_draft, (), True)
    assert [len(x) for x in call.outputs] == [12] * n
    assert max(rows for rows, _ in runner.steps) <= max_prefill
    assert not runner.lengths
    if n * (1 + n_draft) + n * 15 <= max_prefill:           # the prompt, then a step for all of them at a time, with all their drafts
        assert all(live == list(range(n)) for _, live in drawn) and max(max(d) for d, _ in drawn) == n_draft
    if n_draft and max_prefill >= 2 * n:
        assert max(max(d) for d, _ in drawn) > 0
