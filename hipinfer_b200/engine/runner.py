"""The step function. `ModelRunner.step(entries)` takes a batch of (request, its next tokens):
portions of prompts beside single decoded tokens, cut anywhere. It makes room in the cache,
runs only the tokens it is given, as one batch, from the cache earlier steps left, and returns
the 32-bit logits at the wanted places, in the order of the entries and of their `want`.
Generation, the scheduler and trace replay all go through this one function.

A request is known from the first step that names it until `end(request_id)`; its position is
the number of tokens it has been given so far.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import numpy as np
import torch

from ..cache import CacheManager, CacheStorage, OutOfPages
from ..config import ModelConfig, get_architecture, load_config
from ..kernels import ops
from ..models.decoder import DecoderModel
from ..parts.registry import BuildContext
from ..weights import load_weights, random_weights
from .batch import StepBatch, StepEntry, build_step_batch, shared_prefixes

DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16, "float32": torch.float32, "fp32": torch.float32}


CACHE_DTYPES = {"int8": torch.int8, "float8_e4m3fn": torch.float8_e4m3fn, "fp8": torch.float8_e4m3fn}


class StepError(ValueError):
    """A step that cannot run: a token outside the vocabulary, a request beyond the longest
    sequence, a `want` outside the entry (the reference returns -1 for such arguments,
    src/api.cu:1827-1839)."""


class ModelRunner:
    def __init__(self, config: ModelConfig, tensors: Dict[str, torch.Tensor], dtype="bfloat16", device="cuda:0",
                 page_size: int = 16, num_pages: Optional[int] = None, max_model_len: Optional[int] = None,
                 max_num_seqs: int = 8, cuda_graphs: bool = True, cache_dtype=None):
        if not torch.cuda.is_available():
            raise RuntimeError("hipinfer_b200 runs on a CUDA device (sm_100a); none is visible and there is no "
                               "CPU implementation")
        self.config = config
        self.dtype = DTYPES[dtype] if isinstance(dtype, str) else dtype
        self.device = torch.device(device)
        torch.cuda.set_device(self.device)
        self.spec = get_architecture(config.architecture).build_spec(config)
        self.max_model_len = int(min(max_model_len or self.spec.max_position, self.spec.max_position))
        self.page_size = int(page_size)
        self.cache_dtype = cache8_dtype(cache_dtype)
        self.ctx = BuildContext(self.dtype, self.device, self.page_size, self.max_model_len, self.cache_dtype)
        self.model = DecoderModel(self.spec, self.ctx)
        if self.cache_dtype is not None:
            check_cache8(self.model)
        self.model.load(tensors)
        pages_per_seq = -(-self.max_model_len // self.page_size)
        n_pages = int(num_pages) if num_pages is not None else pages_per_seq * max_num_seqs
        groups = self.model.cache_groups
        self.cache = CacheManager(groups, self.page_size, [n_pages] * len(groups), max_num_seqs)
        self.storage = CacheStorage(groups, [n_pages] * len(groups), self.page_size, self.dtype, self.device,
                                    self.model.state_specs, max_num_seqs, self.cache_dtype, max_num_seqs)
        self.vocab_size = self.spec.vocab_size
        self.steps_run = 0
        # decode-only steps (one token per request, every row wanted) are replayed from a CUDA
        # graph captured per number of requests: same kernels, one launch
        self.cuda_graphs = bool(cuda_graphs)
        self._graphs: Dict[tuple, dict] = {}
        self._graph_pool = None
        self._table_widths = [pages_per_seq] * len(groups)
        self._np_tables: Dict[object, list] = {}
        self._forked: set = set()              # requests that began with another's pages
        self._kept: Optional[_KeptStep] = None # what the last step's refused drafts leave behind is undone with (store_accepted)

    # ---------------------------------------------------------------- construction helpers
    @classmethod
    def from_folder(cls, folder: str, **kw) -> "ModelRunner":
        config = load_config(folder)
        spec = get_architecture(config.architecture).build_spec(config)
        from ..parts.spec import spec_param_specs

        dt = kw.get("dtype", "bfloat16")
        exact = (DTYPES[dt] if isinstance(dt, str) else dt) == torch.float32
        tensors = load_weights(folder, spec_param_specs(spec), device=kw.get("device", "cuda:0"),
                               ignore=_ignorable(spec), half_as=torch.float32 if exact else torch.bfloat16)
        return cls(config, tensors, **kw)

    @classmethod
    def from_random(cls, config: ModelConfig, seed: int = 0, std: float = 0.02, norm_std: float = 0.0,
                    weights_dtype=torch.bfloat16, **kw) -> "ModelRunner":
        from ..parts.spec import spec_param_specs

        spec = get_architecture(config.architecture).build_spec(config)
        tensors = random_weights(spec_param_specs(spec), seed, std, norm_std, weights_dtype,
                                 device=kw.get("device", "cuda:0"))
        return cls(config, tensors, **kw)

    # ---------------------------------------------------------------- the step
    def length(self, request_id) -> int:
        return self.cache.get(request_id).length if self.cache.has_request(request_id) else 0

    def check_entries(self, entries: Sequence[StepEntry]) -> list:
        """Raises StepError for a batch that cannot run; returns the entries' tokens as int64 arrays."""
        seen, arrays = set(), []
        for e in entries:
            if e.request_id in seen:
                raise StepError(f"request {e.request_id!r} appears twice in one step")
            seen.add(e.request_id)
            n = len(e.tokens)
            if n < 1:
                raise StepError(f"request {e.request_id!r}: an entry needs at least one token")
            toks = np.asarray(e.tokens, dtype=np.int64)          # one pass, not a Python loop: a portion may have thousands
            if toks.ndim != 1:
                raise StepError(f"request {e.request_id!r}: tokens must be a flat sequence of ints")
            bad = (toks < 0) | (toks >= self.vocab_size)
            if bad.any():
                raise StepError(f"request {e.request_id!r}: token {int(toks[bad][0])} is outside the vocabulary of "
                                f"{self.vocab_size}")
            if self.length(e.request_id) + n > self.max_model_len:
                raise StepError(f"request {e.request_id!r}: {self.length(e.request_id)} + {n} tokens exceed the "
                                f"longest sequence of {self.max_model_len}")
            for w in e.want:
                if not (0 <= int(w) < n):
                    raise StepError(f"request {e.request_id!r}: want {w} is outside its {n} tokens")
            arrays.append(toks)
        return arrays

    def step(self, entries: Sequence[StepEntry], device_tokens: Optional[torch.Tensor] = None,
             token_map: Optional[Sequence[int]] = None, dump: Optional[dict] = None, drafts: bool = False) -> torch.Tensor:
        """Run one batch; float32 logits [number of wanted places, vocab] on the device.
        Raises OutOfPages (nothing changed) when the cache cannot hold the new tokens.
        `device_tokens` (int32 [rows], on the device) replaces the entries' token values, which
        are then placeholders: tokens sampled on the device feed the next step without a trip to
        the host (the reference keeps token and position on the device for the same reason,
        README.md:510-512). With `token_map` (one int per row) only rows with an entry >= 0 take
        their token from device_tokens[entry]; the others keep the value the entry gives.
        `dump` (a dict): the step runs eagerly and leaves named planes of every layer in it (parts/planes.py).
        `drafts`: some of the step's tokens may be taken back (truncate) before the next one; `store_accepted` then belongs between."""
        entries = list(entries)
        self._kept = None
        token_arrays = self.check_entries(entries)
        if not entries:
            return torch.empty(0, self.vocab_size, dtype=torch.float32, device=self.device)
        # room for everything first, so that a failure leaves no request half advanced
        new = [e.request_id for e in entries if not self.cache.has_request(e.request_id)]
        need = [0] * len(self.cache.groups)
        for e in entries:
            for g, n in enumerate(self.cache.pages_needed(e.request_id, len(e.tokens))):
                need[g] += n
        for g, n in enumerate(need):
            if n > self.cache.pools[g].free_count:
                raise OutOfPages(f"cache group {self.cache.groups[g].name!r}: this step needs {n} more pages, "
                                 f"{self.cache.pools[g].free_count} are free")
        if len(new) > self.cache.slots.free_count:
            from ..cache import OutOfStateSlots
            raise OutOfStateSlots(f"{len(new)} new requests, {self.cache.slots.free_count} state slots free")
        ctx_lens, slots, tables, slot_maps = [], [], [], []
        for e in entries:
            if not self.cache.has_request(e.request_id):
                rc = self.cache.add_request(e.request_id)
                self.storage.zero_state_slot(rc.state_slot)
                self._np_tables.pop(e.request_id, None)    # an id that comes back (after preemption) starts afresh
            rc = self.cache.get(e.request_id)
            ctx_lens.append(rc.length)
            slots.append(rc.state_slot)
            slot_maps.append(self.cache.append(e.request_id, len(e.tokens), as_arrays=True))
            tables.append(self._table_rows(rc))
        shared = self._shared_prefixes(tables, ctx_lens) if len(entries) > 1 else ()
        keep = drafts and self.cache_dtype is not None
        graph = dump is None and not keep and self.cuda_graphs and all(len(e.tokens) == 1 and list(e.want) == [0] for e in entries)
        if graph and any(shared) and self._saved_bytes(shared) >= self.SHARED_STEP_BYTES * len(self.spec.order):
            graph = False
        if graph:
            logits = self._graph_step(entries, ctx_lens, slots, tables, slot_maps, device_tokens, token_map)
        else:
            batch = build_step_batch(entries, ctx_lens, slots, tables, slot_maps, len(self.cache.groups), self.device,
                                     token_map=token_map, token_arrays=token_arrays)
            self._feed(batch.tokens, batch.token_map, device_tokens, token_map)
            batch.dump, batch.shared = dump, shared
            if keep:
                batch.kept_rows = []
                self._kept = _KeptStep(entries, ctx_lens, tables, slot_maps, self.page_size, [p.num_pages for p in self.cache.pools], batch.kept_rows)
                self._kept.requests = [self.cache.get(e.request_id) for e in entries]
                for g, (src, dst) in enumerate(self._kept.copies()):
                    if src:
                        self.storage.copy_pages(g, src, dst)
            logits = self.model.forward(batch, self.storage)
        for e in entries:
            if self.cache.release_behind_window(e.request_id):
                self._np_tables.pop(e.request_id, None)
        if len(self._np_tables) > len(self.cache.requests):      # requests freed through the cache manager (the scheduler does)
            for rid in [r for r in self._np_tables if not self.cache.has_request(r)]:
                del self._np_tables[rid]
            self._forked.intersection_update(self.cache.requests)
        self.steps_run += 1
        return logits

    def _shared_prefixes(self, tables, ctx_lens):
        """Per cache group that keeps everything and whose layers make use of it, the neighbours in this step that hold the same pages
        (of forked requests)."""
        if not self._forked:
            return ()
        return [shared_prefixes([t[g] for t in tables], ctx_lens, self.page_size) if spec.kind == "full" and self.model.shared_layers[g]
                else [] for g, spec in enumerate(self.cache.groups)]

    # A decode-only step of forked requests may be replayed from its graph, every request reading all its pages, or run eagerly with
    # attention over the shared pages (whose plan changes every step). Reading is 6 TB/s; launching a layer eagerly takes the host
    # 50 us more. Measured on 16 layers of 32 heads over 8 of 64 in bfloat16, ms a step from the graph and shared: 32 requests behind
    # 2,000 tokens (0.13 GB a layer saved) 1.81 and 2.44, 32 behind 8,000 (0.51 GB) 2.42 and 2.47, 64 behind 4,000 (0.52 GB) 2.95 and 2.90,
    # 128 behind 2,000 (0.52 GB) 4.09 and 3.71, 64 behind 8,000 (1.03 GB) 3.94 and 2.95, 64 behind 15,000 5.86 and 2.99.
    SHARED_STEP_BYTES = 0.5e9

    def _saved_bytes(self, shared) -> float:
        """Bytes of the cache that the step's layers read once instead of once a request."""
        per_token = [spec.elements_per_token() // spec.n_layers * n * self.dtype.itemsize
                     for spec, n in zip(self.cache.groups, self.model.shared_layers)]
        return sum((n - 1) * tokens * b for runs, b in zip(shared, per_token) for _, n, tokens in runs)

    def _table_rows(self, rc):
        """The request's block tables as int32 arrays, kept between steps and extended by the new pages only."""
        rows = self._np_tables.setdefault(rc.request_id, [[np.full(16, -1, dtype=np.int32), 0] for _ in rc.tables])
        out = []
        for slot, table in zip(rows, rc.tables):
            arr, n = slot
            if len(table) > arr.shape[0]:
                grown = np.full(2 * len(table), -1, dtype=np.int32)
                grown[:n] = arr[:n]
                slot[0] = arr = grown
            if len(table) > n:
                arr[n:len(table)] = table[n:]
                slot[1] = len(table)
            out.append(arr[:len(table)])
        return out

    @staticmethod
    def _feed(tokens, map_dev, device_tokens, token_map):
        if device_tokens is None:
            return
        if token_map is None:
            tokens.copy_(device_tokens, non_blocking=True)
        else:
            from ..kernels import ops
            ops.feed_tokens(tokens, device_tokens, map_dev)

    GRAPH_LENGTH_QUANTUM = 512     # tokens by which the length class of a decode graph grows
    MAX_GRAPHS = 128               # captured graphs kept, least recently used first to go (each holds its batch buffer
                                   # and its logits; what a step allocates besides comes from one pool they share)

    def _graph_step(self, entries, ctx_lens, slots, tables, slot_maps, device_tokens=None, token_map=None) -> torch.Tensor:
        """A decode-only step through the CUDA graph for this many requests and this length class (captured at
        first use). The graph's batch lives in one static device buffer that each step overwrites; launch
        geometry is made for the longest position of the class (the step's longest request rounded up to
        GRAPH_LENGTH_QUANTUM tokens), so few blocks lie beyond a row's keys and those return at once; a new
        graph is captured when the longest request crosses into the next class. The logits tensor is the
        graph's own and is overwritten by the next such step."""
        R, G = len(entries), len(self.cache.groups)
        bound = min(self.max_model_len, (max(ctx_lens) // self.GRAPH_LENGTH_QUANTUM + 1) * self.GRAPH_LENGTH_QUANTUM)
        key = (R, bound)
        g = self._graphs.get(key)
        args = dict(n_groups=G, device=self.device, table_widths=self._table_widths, max_pos=bound - 1)
        if g is None:
            n_int = 4 * R + 4 * R + R + sum(R * w for w in self._table_widths) + G * R
            static = torch.zeros(n_int, dtype=torch.int32, device=self.device)
            batch = build_step_batch(entries, ctx_lens, slots, tables, slot_maps, static=static, token_map=token_map, **args)
            self._feed(batch.tokens, batch.token_map, device_tokens, token_map)
            first = self.model.forward(batch, self.storage)    # this step itself, run eagerly: allocations, plans, lazy set-up
            torch.cuda.synchronize()
            from ..kernels import library
            before = library.launches[0]
            graph = torch.cuda.CUDAGraph()
            if self._graph_pool is None:
                self._graph_pool = torch.cuda.graph_pool_handle()
            # one memory pool for all graphs: they never run at the same time, and what a step allocates and frees
            # on its way is the same memory in every graph (only the logits, which stay alive, are a graph's own)
            with torch.cuda.graph(graph, pool=self._graph_pool):     # recorded, not run
                logits = self.model.forward(batch, self.storage)
            while len(self._graphs) >= self.MAX_GRAPHS:
                self._graphs.pop(next(iter(self._graphs)))
            self._graphs[key] = dict(graph=graph, static=static, logits=logits, tokens=batch.tokens,
                                   token_map=batch.token_map, launches=library.launches[0] - before)
            # the step has run once already: replaying the graph now would run it a second time, which a mixer
            # with state of its own (its state advances with every run) must not see
            return first
        else:
            self._graphs[key] = self._graphs.pop(key)          # most recently used last
            build_step_batch(entries, ctx_lens, slots, tables, slot_maps, static=g["static"], token_map=token_map, **args)
            self._feed(g["tokens"], g["token_map"], device_tokens, token_map)
        g["graph"].replay()
        from ..kernels import library
        library.launches[0] += g["launches"]
        return g["logits"]

    def end(self, request_id) -> None:
        """The request is finished: its pages and its state slot are given back."""
        self.cache.free_request(request_id)
        self._np_tables.pop(request_id, None)
        self._forked.discard(request_id)

    def fork(self, request_id, new_id, length: Optional[int] = None) -> int:
        """Request `new_id` begins with the whole pages of `request_id`, which both hold from then on (neither writes them);
        returns how many tokens those are. With `length` it begins with exactly so many tokens: a page that they end inside of is
        copied (ops.copy_pages). Requests that stand side by side in a step and hold the same pages attend to them
        together (ops.attention_shared). In a cache in 8 bits the copy has the parent's codes, in whose scale the parent's tokens behind
        `length` in that block have had part. Raises StepError for a model that keeps state besides the pages, OutOfPages (nothing
        changed) where the cache has no page for the copy."""
        if self.model.state_specs:
            raise StepError("a request of a model with per-request state cannot be forked: its state is not in the pages")
        rc = self.cache.fork(request_id, new_id, length)
        for g, pages in enumerate(rc.copied):
            if pages is not None:
                self.storage.copy_pages(g, [pages[0]], [pages[1]])
        self._np_tables.pop(new_id, None)
        self._forked.add(new_id)
        return rc.length

    def truncate(self, request_id, length: int) -> None:
        """The request's tokens from position `length` on are taken back (drafts that were refused). In a cache in 8 bits the block that the
        others end inside of keeps the scale and the roundings that the tokens taken back gave it, but for the last step's (store_accepted)."""
        if self.model.state_specs:
            raise StepError("a request of a model with per-request state cannot be cut: its state has run on")
        self.cache.truncate(request_id, length)
        for kept, table in zip(self._np_tables.get(request_id, ()), self.cache.get(request_id).tables):
            kept[1] = min(kept[1], len(table))             # (the pages that come next replace those that went)

    def store_accepted(self) -> None:
        """After a step with `drafts` and its truncations: a cache in 8 bits holds what it would if the step had brought the tokens that were kept alone
        (a block's scale is that of the largest of the rows stored with it: a draft that stands out, refused, would leave its block's other tokens
        coarser for good). The blocks that the step began inside of are put back, and the kept rows stored into them again: a launch a layer."""
        kept, self._kept = self._kept, None
        if kept is None:
            return
        # (one that has ended meanwhile, its name perhaps another's by now, has nothing to be put back)
        lengths = [rc.length if self.cache.requests.get(rid) is rc else 0 for rid, rc in zip(kept.ids, kept.requests)]
        if not kept.damaged(lengths):
            return
        for g, (dst, src) in enumerate(kept.copies(lengths)):
            if src:
                self.storage.copy_pages(g, src, dst)
        slots = [torch.from_numpy(s).pin_memory().to(self.device, non_blocking=True) for s in kept.accepted(lengths)]
        for cache, k, v in kept.rows:
            ops.store_cache8(k, v, slots[cache.group], cache.cache8)

    def live_requests(self):
        return list(self.cache.requests)


class _KeptStep:
    """A step over a cache in 8 bits, some of whose tokens may be taken back: which requests brought how many rows to which places, the page that each
    began inside of (and a spare page of its group, behind the `pages` that are handed out, for what it held), and every layer's rows."""

    def __init__(self, entries, ctx_lens, tables, slot_maps, page_size: int, pages: Sequence[int], rows: list):
        self.ids, self.held, self.n = [e.request_id for e in entries], list(ctx_lens), [len(e.tokens) for e in entries]
        self.page_size, self.pages, self.slot_maps, self.rows = page_size, list(pages), slot_maps, rows
        self.begun = [[int(t[h // page_size]) if self._inside(h) else -1 for t in groups] for groups, h in zip(tables, self.held)]

    def _inside(self, length: int) -> int:
        """How many places of its block lie ahead of a token at that place."""
        return length % self.page_size % ops.BLOCK8

    def damaged(self, lengths: Sequence[int]) -> List[int]:
        """The requests (by their places) of which tokens are kept that share a block with the step's that were taken back, from their lengths now."""
        return [r for r, (length, h, n) in enumerate(zip(lengths, self.held, self.n)) if length < h + n and length > max(h, length) - self._inside(max(h, length))]

    def copies(self, lengths: Optional[Sequence[int]] = None):
        """Per group, the pages that the step's requests began inside of and the spare pages of what they held; of the damaged ones, with `lengths`."""
        which = range(len(self.ids)) if lengths is None else self.damaged(lengths)
        for g, pages in enumerate(self.pages):
            there = [r for r in which if self.begun[r][g] >= 0]
            yield [self.begun[r][g] for r in there], [pages + r for r in there]

    def accepted(self, lengths: Sequence[int]) -> List[np.ndarray]:
        """Per group, the step's rows' places: of the damaged requests' kept rows; -1 for all others."""
        damaged = set(self.damaged(lengths))
        return [np.concatenate([np.where(np.arange(n) < (lengths[r] - h if r in damaged else 0), np.asarray(self.slot_maps[r][g], dtype=np.int64), -1)
                                for r, (h, n) in enumerate(zip(self.held, self.n))]).astype(np.int32) for g in range(len(self.pages))]


def cache8_dtype(name) -> Optional[torch.dtype]:
    """The codes of a cache in 8 bits by name ("int8", "float8_e4m3fn" or "fp8") or type; None: a cache of the compute type."""
    if name is None:
        return None
    dtype = CACHE_DTYPES.get(name) if isinstance(name, str) else name
    if dtype not in CACHE_DTYPES.values():
        raise ValueError(f"cache type {name!r}: one of {sorted(CACHE_DTYPES)} is possible, or None")
    return dtype


def check_cache8(model: DecoderModel) -> None:
    """Raises ValueError for a model with a layer whose mixer keeps what 8 bits do not hold."""
    for i, (st, plan) in enumerate(zip(model.spec.order, model.cache_plan)):
        mixer = model.layers[st.layer].mixer
        if plan is not None and not mixer.takes_cache8:
            raise ValueError(f"a cache in 8 bits is not possible: the mixer of step {i} ({type(mixer).__name__}) keeps its cache in the compute type")


def _ignorable(spec) -> List[str]:
    """Tensors a checkpoint may carry that the model does not read: a stored copy of the head
    of a model whose head is tied to the embedding is NOT among them (it would be silently
    dropped); rotary inv_freq buffers of older files are."""
    return [f"{ls.prefix}self_attn.rotary_emb.inv_freq" for ls in spec.layers]
