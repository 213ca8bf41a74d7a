"""Many continuations of one prompt. The prompt is run once; every sample is a fork of it that holds the prompt's pages, so that a step
reads their keys and values once for all samples (ops.attention_shared) where a layer's attention does that
(Mixer.reads_shared_pages: attention without a window; others share the memory alone). A sample brings its newest token and, after it, tokens drafted by
looking up what followed the same tokens earlier in its own text; the step's logits accept or refuse them (ops.verify_drafts), and the
cache gives back what was refused. What is drawn is distributed as if each token had been drawn alone; over a cache in 8 bits (cache_dtype)
up to that cache's rounding, in which a step's drafts have part: the block of 16 tokens that they share with the newest ones is rounded to the scale of its largest,
a draft among them. A refused draft has none in later steps (ModelRunner.store_accepted).

The reference copies a prompt into every batch slot (src/api.cu:1409-1411) and keeps drafts for a caller of its `verify_step` (2029-2060).
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache import OutOfPages
from ..kernels import ops
from .batch import StepEntry
from .runner import StepError


class DraftLookup:
    """Drafts from a request's own tokens: what followed the most recent earlier occurrence of its last `longest` tokens, or of fewer."""

    def __init__(self, tokens: Sequence[int] = (), longest: int = 3, base: Optional["DraftLookup"] = None):
        self.longest = base.longest if base is not None else longest
        self.base = base                                   # the prompt's, shared by all samples and not changed any more
        self.tokens: List[int] = list(base.tokens) if base is not None else []
        self._after: Dict[Tuple[int, ...], int] = {}       # tokens -> the position behind their last occurrence that has one
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            n = len(self.tokens)
            for m in range(1, min(self.longest, n) + 1):
                self._after[tuple(self.tokens[n - m:])] = n
            self.tokens.append(int(t))

    def propose(self, k: int) -> List[int]:
        """Up to k tokens."""
        for m in range(min(self.longest, len(self.tokens)), 0, -1):
            key = tuple(self.tokens[-m:])
            at = self._after.get(key)
            if at is None and self.base is not None:
                at = self.base._after.get(key)
            if at is not None:
                return self.tokens[at:at + k]
        return []


class Sampling:
    """One call of Engine.sample_many: its requests, from the prompt to the last token."""

    def __init__(self, engine, prompt, n, n_new, temperature, seed, n_draft, stop_tokens):
        self.runner, self.max_prefill = engine.runner, engine.max_prefill
        self.prompt, self.n, self.n_new, self.n_draft, self.stop = prompt, n, n_new, n_draft, stop_tokens
        self.temperature = float(temperature)
        dev = self.runner.device
        self.random = torch.Generator(device=dev).manual_seed(seed)
        self.rids = [("sample", id(self), i) for i in range(n)]
        self.outputs: List[List[int]] = [[] for _ in range(n)]
        self.logprobs: List[List[float]] = [[] for _ in range(n)]
        self.steps = 0
        if self.temperature <= 0:
            self.noise = torch.ones(1, self.runner.vocab_size, dtype=torch.float32, device=dev)

    def run(self):
        try:
            logits = self._run_prompt()
            base = DraftLookup(self.prompt)
            self.texts = [DraftLookup(base=base) for _ in self.rids]
            self._take(logits, [0] * self.n, [[]] * self.n, list(range(self.n)))
            while True:
                live = [i for i in range(self.n) if not self._done(i)]
                for i in range(self.n):
                    if i not in live and self.runner.cache.has_request(self.rids[i]):
                        self.runner.end(self.rids[i])
                if not live:
                    return
                self._step(live)
        finally:
            for rid in self.rids:
                if self.runner.cache.has_request(rid):
                    self.runner.end(rid)

    def _done(self, i) -> bool:
        out = self.outputs[i]
        return len(out) >= self.n_new or (bool(out) and out[-1] in self.stop)

    def _run_prompt(self) -> torch.Tensor:
        """The prompt as sample 0's, in portions; the others are forked from it where its last whole page ends (later, a window's
        pages that they read may be gone) and run the rest with their first step, or at its end, with a copy of its last page. Returns the logits behind the prompt."""
        P, at, forks = len(self.prompt), 0, self.rids[1:] if self.n_new > 1 else []
        # a cache in 8 bits: the forks begin behind the prompt, the page that it ends inside of copied. Run again beside other tokens, the
        # rest would be rounded to another block's scale than the prompt's own.
        copied = getattr(self.runner, "cache_dtype", None) is not None
        whole = P if copied else P // self.runner.page_size * self.runner.page_size
        for end in sorted({whole if forks else P, P} - {0}):
            while at < end:
                part = self.prompt[at:min(end, at + self.max_prefill)]
                at += len(part)
                logits = self.runner.step([StepEntry(self.rids[0], part, [len(part) - 1] if at == P else [])])
            if end == whole:
                for rid in forks:
                    self.runner.fork(self.rids[0], rid, *([P] if copied else []))
        return logits

    def _behind(self, i) -> int:
        """Tokens of sample i that are still to be run: its newest, and in a fork's first step the prompt's last, partial page."""
        return len(self.texts[i].tokens) - self.runner.length(self.rids[i])

    def _step(self, live) -> None:
        """The live samples' newest tokens with drafts behind them, in one step where there are no more samples than a step may have rows."""
        if sum(map(self._behind, live)) > self.max_prefill:
            self._catch_up(live)
        for at in range(0, len(live), self.max_prefill):
            self._step_of(live[at:at + self.max_prefill])

    def _catch_up(self, live) -> None:
        """All but their newest tokens, which do not fit into one step beside each other."""
        entries, room = [], self.max_prefill
        for i in live:
            at, rows = self.runner.length(self.rids[i]), self.texts[i].tokens[:-1]
            while at < len(rows):
                part = rows[at:at + room]
                entries.append(StepEntry(self.rids[i], part, []))
                at, room = at + len(part), room - len(part)
                if not room:
                    self.runner.step(entries)
                    entries, room = [], self.max_prefill
        if entries:
            self.runner.step(entries)

    def _step_of(self, live) -> None:
        most = min(self.n_draft, (self.max_prefill - sum(map(self._behind, live))) // len(live))      # (the rest of the step's rows)
        entries, starts, drafts, row = [], [], [], 0
        for i in live:
            text = self.texts[i]
            d = text.propose(min(most, self.n_new - len(self.outputs[i]) - 1))
            rows = text.tokens[-self._behind(i):] + d
            entries.append(StepEntry(self.rids[i], rows, range(len(rows) - 1 - len(d), len(rows))))
            starts.append(row)
            drafts.append(d)
            row += len(d) + 1
        keep = any(drafts) and getattr(self.runner, "cache_dtype", None) is not None
        logits = self.runner.step(entries, drafts=True) if keep else self.runner.step(entries)
        self._take(logits, starts, drafts, live)
        for i in live:
            self.runner.truncate(self.rids[i], len(self.texts[i].tokens) - 1)      # all but the token that is still to be run
        if keep:
            self.runner.store_accepted()
        self.steps += 1

    def _take(self, logits, starts, drafts, live) -> None:
        """Draws behind each request's rows of logits and adds what was accepted and drawn to its text."""
        R, V, dev = len(live), self.runner.vocab_size, self.runner.device
        K = max(len(d) for d in drafts)
        host = torch.zeros(R, K + 2, dtype=torch.int32, pin_memory=True)
        numbers = host.numpy()
        numbers[:, 0], numbers[:, 1] = starts, [len(d) for d in drafts]
        for r, d in enumerate(drafts):
            numbers[r, 2:2 + len(d)] = d
        sent = host.to(dev, non_blocking=True)
        if self.temperature > 0:
            noise = torch.empty(R, V, dtype=torch.float32, device=dev).exponential_(generator=self.random)
            uniform = torch.rand(R, K, dtype=torch.float32, device=dev, generator=self.random)
        else:
            noise, uniform = self.noise.expand(R, V), torch.zeros(R, K, dtype=torch.float32, device=dev)
        temperature = torch.full((R,), self.temperature, dtype=torch.float32, device=dev)
        tokens, counts, logprobs = ops.verify_drafts(logits, sent[:, 0].contiguous(), sent[:, 1].contiguous(), sent[:, 2:].contiguous(), temperature,
                                                     uniform, noise)
        got = torch.cat([counts[:, None], tokens, logprobs.view(torch.int32)], 1).cpu().numpy()
        ops.check_device_status()
        for r, i in enumerate(live):
            n = int(got[r, 0])
            if n < 1:
                raise RuntimeError(f"sample {i}: no token was drawn")
            new = got[r, 1:1 + n].tolist()
            lps = np.ascontiguousarray(got[r, K + 2:K + 2 + n]).view(np.float32).tolist()
            for j, t in enumerate(new):
                if t in self.stop:                             # nothing is kept behind a stop token
                    new, lps = new[:j + 1], lps[:j + 1]
                    break
            self.texts[i].extend(new)
            self.outputs[i] += new
            self.logprobs[i] += lps


def sample_many(engine, prompt, n, n_new, temperature, seed, n_draft, stop_token_ids, ignore_eos) -> Sampling:
    """Checks the arguments and runs the call; Engine.sample_many describes it."""
    runner, prompt = engine.runner, [int(t) for t in prompt]
    if not prompt or any(not 0 <= t < engine.vocab for t in prompt):
        raise ValueError(f"sample_many needs a prompt of tokens below {engine.vocab}")
    if n < 1 or n_new < 1 or not temperature >= 0:      # (a NaN too)
        raise ValueError(f"sample_many: {n} samples of {n_new} tokens at temperature {temperature}")
    if not 0 <= n_draft <= ops.MAX_DRAFTS:
        raise ValueError(f"sample_many: {n_draft} drafts a step, 0 to {ops.MAX_DRAFTS} are possible")
    if len(prompt) + n_new > engine.max_seq:
        raise ValueError(f"{len(prompt)} + {n_new} tokens exceed the longest sequence {engine.max_seq}")
    if runner.model.state_specs:
        raise ValueError("sample_many: this model keeps per-request state, which forked requests cannot share")
    if n_draft and any(g.kind != "full" for g in runner.cache.groups):
        raise ValueError("sample_many: drafts need a model that keeps every token, so that refused ones can be taken back")
    if n > runner.cache.slots.free_count:
        raise ValueError(f"{n} samples, {runner.cache.slots.free_count} requests more can be live")
    stop = set(stop_token_ids) | (set() if ignore_eos else set(runner.spec.eos_token_ids))
    call = Sampling(engine, prompt, n, n_new, temperature, seed, n_draft, stop)
    try:
        call.run()
    except (StepError, OutOfPages) as e:
        raise ValueError(str(e)) from None
    return call
