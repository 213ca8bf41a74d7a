"""Operators of a paged cache in 8 bits: storing a step's keys and values, reading pages back, attention over it; and copying pages of a cache
of any type, as forks inside a page need it. Reached as `ops.Cache8`, `ops.new_cache8`, `ops.store_cache8`, `ops.expand_cache8`, `ops.attention_cache8`
and `ops.copy_pages` (csrc/cache8_store.cu: storing and reading back; cache8_attention_mma.cu: attention of single rows and short portions on
warp MMAs; attention_prefill_tc.cu: of longer portions; cache8_attention.cu: of any other sizes; copy_pages.cu; cache8_binding.cpp: calls without
the interpreter).

A cache holds, for keys and for values, codes [page, kv head, page_size, head_dim] (int8, or e4m3) and scales float32 [page, kv head, blocks], one
for each block of 16 places of a page (the last block of a page may have fewer); a place's numbers are code * scale.

The reference keeps its cache in the activations' type (src/api.cu:1409-1411) and copies nothing within it."""
from __future__ import annotations

import ctypes as C
import functools
import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import library, ops

_p, _i, _l, _f = C.c_void_p, C.c_int, C.c_long, C.c_float
ops._SIGS["cache8"] = {
    "hb_cache8_store": [_p, _p, _l, _l, _i, _p, _i, _i, _i, _i, _l, _i, _p, _p, _p, _p, _p],
    "hb_cache8_expand": [_p, _p, _p, _p, _i, _p, _l, _l, _i, _i, _i, _p, _p, _i, _p],
    "hb_cache8_attention_any": [_p, _i, _l, _p, _p, _p, _p, _i, _l, _i, _i, _i, _p, _l, _i, _i, _p, _p, _i, _i, _i, _f, _p, _p],
    "hb_cache8_attention_mma": [_p, _i, _l, _p, _p, _p, _p, _i, _l, _i, _i, _i, _p, _l, _i, _i, _p, _p, _i, _i, _i, _i, _i, _f, _p, _i, _p],
    "hb_cache8_attention_mma_supported": [_i, _i, _i, _l],
    "hb_cache8_attention_mma_clusters": [_i, _i, _i, _i, _i],
    "hb_cache8_portions": [_p, _p, _p, _p, _i, _p, _p, _l, _l, _i, _i, _i, _f, _p, _p, _p, _i, _p],
    "hb_copy_pages": [_p, _i, _p, _p, _i, _p],
}
BLOCK8 = 16                                                        # places of a page that share a scale
CODES = {torch.int8: 2, torch.float8_e4m3fn: 3}                    # csrc/cache8.cuh


def cache8_blocks(page_size: int) -> int:
    """Scales of a page and head."""
    return -(-page_size // BLOCK8)


@dataclass(frozen=True, eq=False)
class Cache8:
    """A layer's cache in 8 bits: codes k, v [pages, n_kv_heads, page_size, head_dim], scales k_scale, v_scale [pages, n_kv_heads, blocks], none of them
    negative."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self):
        k, v = self.k, self.v
        if k.dtype not in CODES or v.dtype != k.dtype or k.dim() != 4 or v.shape != k.shape or not k.is_contiguous() or not v.is_contiguous():
            raise ops.KernelError(f"a cache in 8 bits has codes [pages, heads, page_size, head_dim] of {' or '.join(str(t) for t in CODES)}, keys and values "
                                  f"alike, side by side; got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        scales = k.shape[:2] + (cache8_blocks(k.shape[2]),)
        for s in (self.k_scale, self.v_scale):
            if s.dtype != torch.float32 or s.shape != scales or not s.is_contiguous():
                raise ops.KernelError(f"a cache in 8 bits of {tuple(k.shape)} has float32 scales {tuple(scales)}, got {tuple(s.shape)} {s.dtype}")
        if k.numel() and min(k.shape[1:]) < 1:
            raise ops.KernelError(f"a cache in 8 bits of {tuple(k.shape)}")
        object.__setattr__(self, "code", CODES[k.dtype])
        object.__setattr__(self, "tensors", (k, v, self.k_scale, self.v_scale))
        object.__setattr__(self, "mma", None)                      # see _on_tensor_cores
        # as the binding reads it (Cache in csrc/cache8_binding.cpp); -1: not on one GPU
        one = k.is_cuda and {t.device for t in self.tensors} == {k.device}
        numbers = np.array([t.data_ptr() for t in self.tensors] + list(k.shape) + [self.code, k.device.index if one else -1], dtype=np.int64)
        object.__setattr__(self, "_native", numbers)
        object.__setattr__(self, "native", numbers.ctypes.data)

    def __reduce__(self):                                          # (a copy has addresses of its own)
        return Cache8, self.tensors

    @property
    def n_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]


def new_cache8(pages: int, n_kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.int8, device="cuda:0") -> Cache8:
    """An empty cache (zeros: every place is the number 0)."""
    if dtype not in CODES or min(pages, n_kv_heads, page_size, head_dim) < 1:
        raise ops.KernelError(f"a cache in 8 bits of {pages} pages, {n_kv_heads} heads, {page_size} places, {head_dim}, {dtype}")
    codes = lambda: torch.zeros(pages, n_kv_heads, page_size, head_dim, dtype=torch.uint8, device=device).view(dtype)
    scales = lambda: torch.zeros(pages, n_kv_heads, cache8_blocks(page_size), dtype=torch.float32, device=device)
    return Cache8(codes(), codes(), scales(), scales())


def _here(what: str, *tensors) -> None:
    """The kernels run on the current device's current stream: everything has to be there."""
    ops._need_cuda(*tensors)
    device = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.device.index != device:
            raise ops.KernelError(f"{what}: a tensor on {t.device}, the current device is cuda:{device}")


def _ints(what: str, name: str, x: torch.Tensor, n: Optional[int] = None) -> None:
    if x.dtype != torch.int32 or x.dim() != 1 or not x.is_contiguous() or (n is not None and x.numel() != n):
        raise ops.KernelError(f"{what}: {name} {tuple(x.shape)} {x.dtype}, strides {x.stride()}; int32 [{'n' if n is None else n}] side by side is expected")


_rows = {}


def row_places(device, n: int) -> torch.Tensor:
    """0 .. n - 1 (int32): the places of a step's rows in pages of one place. Older, shorter tensors are kept: a captured graph may hold their addresses.
    Not made while a graph is captured."""
    held = _rows.setdefault(device, [])
    if not held or held[-1].numel() < n:
        if torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise ops.KernelError(f"row_places: {n} rows are more than before; run the step once before it is captured")
        # (copied from the host, which waits: streams other than the current one may read it)
        held.append(torch.arange(max(n, 4096, 2 * held[-1].numel() if held else 0), dtype=torch.int32).to(device))
    return held[-1][:n]


def store_cache8(k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor, cache: Cache8) -> Cache8:
    """Rows k, v [T, n_kv_heads * head_dim] (float32 or bfloat16; rows may be part of wider ones) stored at the places slot_map (int32 [T], page *
    page_size + place; a number outside of the cache stores nothing).

    Rows may come in any order; of several for one place the last counts, and the others are as if they were not there. A block (16 places of a page)
    one of whose rows goes to its first place begins anew: its scale is max(a, 1e-30) / M, a being the largest |x| of the block's rows and head, M
    the largest code (127, or 448). In any other block the scale grows to that where it is larger, and the codes that are there are rounded to it once
    more: half a step each time that it grows. Numbers that are not finite do not count for a: infinities become the largest code, NaN becomes 0.
    Places of a block that no row goes to keep their codes where the scale stays or begins anew. A cache has at most 2^31 - 1 places."""
    bound = _binding() if _bound is None and k.is_cuda else _bound
    if bound and k.is_cuda:
        done = bound.store(k, v, slot_map, cache.native)
        if done is not None:
            _done(done, 1)
            return cache
    _here("store_cache8", k, v, slot_map, *cache.tensors)
    width = cache.n_kv_heads * cache.head_dim
    if k.dim() != 2 or k.shape != v.shape or k.shape[1] != width or k.dtype != v.dtype or (width > 1 and (k.stride(1) != 1 or v.stride(1) != 1)):
        raise ops.KernelError(f"store_cache8: keys {tuple(k.shape)} {k.dtype}, values {tuple(v.shape)} {v.dtype}, strides {k.stride()} and {v.stride()}; rows "
                              f"of {cache.n_kv_heads} heads of {cache.head_dim} are expected")
    T = k.shape[0]
    _ints("store_cache8", "slot_map", slot_map, T)
    dt = ops._dt(k)
    if not T or not cache.k.numel():
        return cache
    ops._call("cache8", "hb_cache8_store", k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), dt, slot_map.data_ptr(), T, cache.n_kv_heads,
              cache.page_size, cache.head_dim, cache.k.shape[0], cache.code, *(t.data_ptr() for t in cache.tensors), ops._stream())
    return cache


def expand_cache8(cache: Cache8, pages: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The numbers of `pages` (int32 [n]) as keys and values [n, n_kv_heads, page_size, head_dim] in float32 or bfloat16; zeros for a page number
    outside of the cache."""
    bound = _binding() if _bound is None and pages.is_cuda else _bound
    if bound and pages.is_cuda and dtype in ops._DT:
        done = bound.expand(pages, cache.native, ops._DT[dtype])
        if done is not None:
            return _done(done, 1)
    _here("expand_cache8", pages, *cache.tensors)
    _ints("expand_cache8", "pages", pages)
    if dtype not in ops._DT:
        raise ops.KernelError(f"expand_cache8: element type {dtype} is not supported (float32 and bfloat16 are)")
    k, v = (torch.empty((pages.numel(),) + cache.k.shape[1:], dtype=dtype, device=cache.k.device) for _ in range(2))
    if k.numel() and not cache.k.numel():
        return k.zero_(), v.zero_()
    if k.numel():
        ops._call("cache8", "hb_cache8_expand", *(t.data_ptr() for t in cache.tensors), cache.code, pages.data_ptr(), pages.numel(), cache.k.shape[0],
                  *cache.k.shape[1:], k.data_ptr(), v.data_ptr(), ops._DT[dtype], ops._stream())
    return k, v


def attention_cache8(q: torch.Tensor, cache: Cache8, batch, group: int, n_heads: int, window: int = 0, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the step's rows (`batch`: an engine.batch.StepBatch) over their requests' pages of cache group `group`, whose keys and values,
    the step's own among them, are in `cache`. q [T, n_heads * head_dim] (bfloat16 or float32; rows may be part of wider ones), out [T, n_heads *
    head_dim] of its type; query head h reads kv head h // (n_heads / n_kv_heads). A row at position p sees the keys j <= p (and j > p - window,
    for a window above 0) whose pages are in the block table and in the cache; one that sees none is 0. scale: 1 / sqrt(head_dim) by default. Scores,
    softmax and sums are 32-bit. On their way into the second product weights are rounded: to float16 for rows of the kernel on warp MMAs (for
    float32 rows to two of them), to bfloat16 for portions on the flash kernel, whose results are off by 2.3e-3 of themselves where the others are by 1.7e-3, most of it the result's own
    rounding. Which of the two a bfloat16 request of 16 to 127 rows goes through is a matter of the whole step (_portion_limit), and so are its last bits. Codes at places that a row of the step sees are numbers (e4m3 has a NaN; storing leaves none).

    A graph that a call is captured into wants the batch, with its tensors, to live as long as itself. A step in which a request brings several rows is
    laid out by the host at the batch's first call, from the lengths that the batch was built with: it has to have run once before it is captured, and is
    replayed for those lengths; a step of one row a request follows positions and tables that are written over the batch's."""
    table, T, D = batch.block_tables[group], batch.n_rows, cache.head_dim
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    tensor_cores = q.is_cuda and _on_tensor_cores(cache)
    limit = 0
    if tensor_cores and batch.max_q_len >= PORTION_ROWS[0] and batch.n_requests <= FLASH_REQUESTS and cache.k.shape[0] \
            and _flash_takes(q, cache, out, n_heads, scale):
        limit = _portion_limit(batch, cache, n_heads, window)
    others = tensor_cores and T and (not limit or any(0 < n < limit for n in batch.h_q_len))
    if tensor_cores and T:
        bound = _binding() if _bound is None else _bound
        if bound:
            cut = _cut(batch, cache, ops._dt(q), n_heads, window, limit) if others else None
            groups = [_portions(batch, cache, table, n_heads, window, limit, g) for g in _portion_groups(batch, cache, window, limit)] if limit else [None]
            to = out
            for flash in groups:
                done = bound.attend(q, cache.native, table, batch.positions, cut and cut.tiles, cut.native if cut else 0, scale, to, flash.native if flash else 0)
                if done is None:
                    break
                to = _done(done, bool(cut) + 2 * bool(flash))
                cut = None                                         # (the other rows are done with the first group)
            else:
                return to
    _here("attention_cache8", q, table, batch.positions, batch.row_request, *cache.tensors, out)
    _heads(cache, n_heads, window)
    if D > 256:
        raise ops.KernelError(f"attention_cache8: heads of {D}, at most 256")
    if q.shape != (T, n_heads * D) or q.stride(1) != 1:
        raise ops.KernelError(f"attention_cache8: q {tuple(q.shape)}, strides {q.stride()}; {T} rows of {n_heads} heads of {D} are expected")
    dt = ops._dt(q)
    if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.shape[0] != batch.n_requests \
            or table.shape[1] * cache.page_size <= batch.max_pos:
        raise ops.KernelError(f"attention_cache8: block table {tuple(table.shape)} {table.dtype}; {batch.n_requests} requests of up to {batch.max_pos + 1} "
                              f"tokens in pages of {cache.page_size}")
    for name in ("positions", "row_request"):
        _ints("attention_cache8", name, getattr(batch, name), T)
    if out is None:
        out = torch.empty(T, n_heads * D, dtype=q.dtype, device=q.device)
    elif out.shape != (T, n_heads * D) or out.dtype != q.dtype or not out.is_contiguous():
        raise ops.KernelError(f"attention_cache8: out {tuple(out.shape)} {out.dtype}, strides {out.stride()}")
    if not T:
        return out
    if not tensor_cores:
        ops._call("cache8", "hb_cache8_attention_any", q.data_ptr(), dt, q.stride(0), *(t.data_ptr() for t in cache.tensors), cache.code, cache.k.shape[0],
                  cache.n_kv_heads, cache.page_size, D, table.data_ptr(), table.stride(0), table.shape[0], table.shape[1],
                  None if _single_rows(batch) else batch.row_request.data_ptr(), batch.positions.data_ptr(), T, n_heads // cache.n_kv_heads, int(window), scale,
                  out.data_ptr(), ops._stream())
        return out
    if others:
        cut = _cut(batch, cache, dt, n_heads, window, limit)
        ops._call("cache8", "hb_cache8_attention_mma", q.data_ptr(), dt, q.stride(0), *(t.data_ptr() for t in cache.tensors), cache.code, cache.k.shape[0],
                  cache.n_kv_heads, cache.page_size, D, table.data_ptr(), table.stride(0), table.shape[0], table.shape[1], batch.positions.data_ptr(),
                  ops._ptr(cut.tiles), cut.n_tiles, cut.nt, cut.ranks, n_heads // cache.n_kv_heads, int(window), scale, out.data_ptr(), bool(limit), ops._stream())
    if limit:
        for group in _portion_groups(batch, cache, window, limit):
            _attend_portions(q, cache, batch, table, n_heads, int(window), scale, out, limit, group, others)
            others = False
    return out


def _heads(cache: Cache8, n_heads: int, window: int) -> None:
    if n_heads < 1 or n_heads % cache.n_kv_heads:
        raise ops.KernelError(f"attention_cache8: {n_heads} heads are not a multiple of {cache.n_kv_heads} kv heads")
    if not 0 <= window < 2 ** 31:
        raise ops.KernelError(f"attention_cache8: window {window}")


def _on_tensor_cores(cache: Cache8) -> bool:
    """Whether the kernel on warp MMAs takes the cache's sizes and place in memory (csrc/cache8_attention_mma.cu)."""
    if cache.mma is None:
        object.__setattr__(cache, "mma", (cache.k.data_ptr() | cache.v.data_ptr()) % 16 == 0
                           and bool(ops._fn("cache8", "hb_cache8_attention_mma_supported")(cache.n_kv_heads, cache.page_size, cache.head_dim, cache.k.shape[0])))
    return cache.mma and ops.fast_kernels_on()


PORTION_ROWS = (16, 32, 64, 128)
FLASH_REQUESTS = 65535                                             # of a step that the flash kernel takes


def _portion_limit(batch, cache: Cache8, n_heads: int, window: int) -> int:
    """From how many rows on a request's pages are expanded for the flash kernel (one of PORTION_ROWS; 0: none are). Per (row, head) and key the
    flash kernel takes a third of the warp MMAs' time, but works in tiles of 128 rows, walks a tile's keys one after the other and wants the keys
    expanded; the choice is the least of the step's estimated times. Both as measured, us: 32 heads over 8 of 128, one portion of 64 rows behind 500
    tokens 12.8 on warp MMAs and 15.5 with the flash kernel, behind 8,000 46.8 and 101; 256 rows behind 2,000 49.7 and 35.8, behind 24,000 474 and 290;
    heads of 64: 11.3 and 18.7, 33.0 and 122; 42.4 and 41.5, 329 and 343. The estimates are off by a sixth at most where the times are not alike."""
    key = ("cache8 limit", n_heads, cache.n_kv_heads, cache.head_dim, cache.code, window)
    if key not in batch.extra:
        rows, held = np.array(batch.h_q_len, dtype=np.float64), np.array(batch.h_ctx_len, dtype=np.float64)
        keys = np.minimum(held, window) + rows if window else held + rows
        best, before = None, 0
        for limit in PORTION_ROWS + (0,):
            flash = rows >= limit if limit else rows < 0
            count = np.count_nonzero(flash)
            if limit and count in (0, before):                                # none, or the same as with the limit before
                continue
            before = count
            us, wide = 0.0, cache.head_dim == 128
            if count:
                n, k = rows[flash], keys[flash]
                padded = np.ceil(n / 128) * 128 * (k - n / 2)                 # (row, key) pairs of whole tiles; or one tile's keys in their order
                us += 8 + k.sum() * cache.n_kv_heads * cache.head_dim * 6 / 5.5e6 + max((0.8e-6 if wide else 0.45e-6) * n_heads * padded.sum(),
                                                                                   (1.35 if wide else 1.72) / 128 * k.max())
            if rows[~flash].any():
                n, k = rows[~flash], keys[~flash]
                G, most = n_heads // cache.n_kv_heads, int(k.max())
                nt = min(4, -(-int(n.max()) * G // 8))
                tiles = np.ceil(n * G / (8 * nt)) * cache.n_kv_heads
                ranks = _ranks(int(tiles.sum()), most, float(k.mean()), functools.partial(_clusters, 1, cache.code, cache.head_dim, nt))
                one = 0.0027 + 0.0021 * nt if wide else 0.0016 + 0.0014 * nt  # a key of a tile on a full SM; by itself a block takes 1.7 times as long
                us += 6.5 + max((tiles * (k - n / 2)).sum() / 148 * one, most / ranks * 1.7 * one, k.sum() * cache.n_kv_heads * cache.head_dim * 2 / 6e6)
            if best is None or us < best[0]:
                best = us, limit
        batch.extra[key] = best[1]
    return batch.extra[key]


def _flash_takes(q, cache: Cache8, out, n_heads: int, scale: float) -> bool:
    return (q.dtype == torch.bfloat16 and q.is_contiguous() and scale > 0 and (q.data_ptr() | (0 if out is None else out.data_ptr())) % 16 == 0
            and _flash_sizes(n_heads, cache.n_kv_heads, cache.head_dim, cache.page_size))


@functools.lru_cache(maxsize=None)
def _flash_sizes(n_heads: int, n_kv_heads: int, head_dim: int, page_size: int) -> bool:
    return n_heads > 0 and n_heads % n_kv_heads == 0 and ops.fast.flash_prefill_tc_supported(n_heads, n_kv_heads, head_dim, page_size)


_AHEAD = 32             # C8_AHEAD of csrc/cache8_store.cu


# The pages that a step's portions see are expanded for some of its requests at a time, so that their codes in 16 bits take no more than this (but for a single request's, which
# are one flash call's keys): 260,000 tokens of 8 heads of 128. Eight portions behind 100,000 tokens would be 3.3 GB at once beside a cache that was given the GPU's memory.
PORTION_BYTES = 1 << 30


def _portion_groups(batch, cache: Cache8, window: int, limit: int) -> list:
    """(first, end) of neighbouring requests whose portions of `limit` rows or more are expanded together."""
    key = ("cache8 groups", cache.k.shape[1:], window, limit, PORTION_BYTES)
    if key not in batch.extra:
        groups, first, held, page = [], 0, 0, 4 * cache.k[0].numel()
        for r, n in _portion_pages(batch, cache.page_size, window, limit):
            if held and (held + n) * page > PORTION_BYTES:
                groups.append((first, r))
                first, held = r, 0
            held += n
        batch.extra[key] = groups + [(first, batch.n_requests)]
    return batch.extra[key]


def _portion_pages(batch, page_size: int, window: int, limit: int):
    """(request, how many pages its rows see) of the portions of `limit` rows or more."""
    for r, (held, rows) in enumerate(zip(batch.h_ctx_len, batch.h_q_len)):
        if rows >= limit:
            yield r, -(-(held + rows) // page_size) - (max(0, held - window + 1) // page_size if window else 0)


class _Portions:
    """A step's portions of `limit` rows or more, of the requests `group` (first, end), as the binding reads them (Portions in csrc/cache8_binding.cpp)."""

    def __init__(self, batch, cache: Cache8, table, n_heads: int, window: int, limit: int, group: tuple):
        _heads(cache, n_heads, window)
        self.index, self.places, self.base = _pages_of_portions(batch, cache.page_size, table.shape[1], window, limit, group)
        q_len = batch.req_q_len if group == (0, batch.n_requests) else _rows_of_group(batch, group)
        self.lengths = batch.req_q_start, q_len, batch.req_ctx_len
        n = self.index.numel()
        self.scales = n * cache8_blocks(cache.page_size) + 2 * _AHEAD
        self._native = np.array([batch.n_rows, batch.n_requests, table.shape[1], n, self.scales, limit, batch.max_q_len, n_heads // cache.n_kv_heads, window,
                                 batch.max_pos] + [t.data_ptr() for t in (self.index, self.places, self.base) + self.lengths] + [ops.fast._status_ptr()],
                                dtype=np.int64)
        self.native = self._native.ctypes.data


def _portions(batch, cache: Cache8, table, n_heads: int, window: int, limit: int, group: tuple) -> _Portions:
    key = ("cache8 portions", cache.k.shape[1:], table.shape[1], n_heads, window, limit, group)
    return _on_stream(batch, key, lambda: _Portions(batch, cache, table, n_heads, window, limit, group))


def _rows_of_group(batch, group: tuple) -> torch.Tensor:
    """The requests' numbers of rows (int32 on the device), 0 for those outside of the group: the flash kernel passes them over."""
    lengths = lambda: np.array([n if group[0] <= r < group[1] else 0 for r, n in enumerate(batch.h_q_len)], dtype=np.int32)
    return _on_stream(batch, ("cache8 rows", group), lambda: _to_device(lengths(), batch))[0]


def _attend_portions(q, cache: Cache8, batch, table, n_heads: int, window: int, scale: float, out, limit: int, group: tuple, beside: bool) -> None:
    """Requests of `limit` rows or more: the codes of the pages that they see as 16-bit numbers, side by side, their scales beside them, and the flash
    kernel over both."""
    p = _portions(batch, cache, table, n_heads, window, limit, group)      # (one page at least: a row sees its own key)
    n, device = p.index.numel(), q.device
    k, v = (torch.empty((n,) + cache.k.shape[1:], dtype=torch.bfloat16, device=device) for _ in range(2))
    scales = torch.empty(cache.n_kv_heads, p.scales, 4, dtype=torch.float32, device=device)
    ops._call("cache8", "hb_cache8_portions", *(t.data_ptr() for t in cache.tensors), cache.code, table.data_ptr(), p.index.data_ptr(), n, cache.k.shape[0],
              *cache.k.shape[1:], scale, k.data_ptr(), v.data_ptr(), scales.data_ptr(), beside, ops._stream())
    ops.fast.flash_prefill_tc_cache8(q, k, v, p.places, *p.lengths, out, batch.max_q_len, n_heads, cache.n_kv_heads, cache.head_dim, cache.page_size, window,
                                     limit, scales, p.base)


def _pages_of_portions(batch, page_size: int, width: int, window: int, limit: int, group: Optional[tuple] = None):
    """For requests of `limit` rows or more (of those from group[0] to group[1] - 1): where in the block table the pages stand that their rows see (int32 [n]), the table of the n pages side
    by side (int32 [requests, width], -1: none), and at which of the n pages' blocks of 16 places each request's first key would stand (int32)."""
    group = group or (0, batch.n_requests)

    def pages():
        index, places, n = [], np.full((batch.n_requests, width), -1, dtype=np.int32), 0
        base, blocks = np.zeros(batch.n_requests, dtype=np.int32), cache8_blocks(page_size)
        for r, (held, rows) in enumerate(zip(batch.h_ctx_len, batch.h_q_len)):
            if rows < limit or not group[0] <= r < group[1]:
                continue
            first, end = max(0, held - window + 1) // page_size if window else 0, -(-(held + rows) // page_size)
            index.append(np.arange(first, end, dtype=np.int32) + r * width)
            places[r, first:end] = np.arange(n, n + end - first, dtype=np.int32)
            base[r] = (n - first) * blocks + _AHEAD
            n += end - first
        return np.concatenate(index + [places.ravel(), base])

    both, R = _on_stream(batch, ("cache8 pages", page_size, width, window, limit, group), lambda: _to_device(pages(), batch))[0], batch.n_requests
    n = both.numel() - R * (width + 1)
    return both[:n], both[n:n + R * width].view(R, width), both[n + R * width:]


def _on_stream(batch, key, make):
    """What `make` lays out on the device for the batch, kept with it: a stream has its own, since another one need not wait for it. A stream that is
    being captured makes none (it would be there only when the graph is replayed) and takes what there is, which capturing begins behind."""
    stream = ops._stream() if batch.tokens.is_cuda else None
    kept = batch.extra.setdefault(key, {})
    if stream not in kept:
        if stream is not None and torch.cuda.is_current_stream_capturing():
            if not kept:
                raise ops.KernelError("attention_cache8: a step in which a request brings several rows has to have run once before it is captured")
            return next(iter(kept.values()))
        kept[stream] = make()
    return kept[stream]


def _to_device(numbers: np.ndarray, batch):
    """(on the device, the host's copy, which stays until the other is over)"""
    host = torch.from_numpy(numbers)
    if batch.tokens.is_cuda:
        host = host.pin_memory()
    return host.to(batch.tokens.device, non_blocking=True), host


class _Cut:
    """How the rows of requests of fewer than `limit` rows (0: of all) are cut into tiles of 8 nt (row, query head) pairs of a kv head, whose keys
    `ranks` blocks share. tiles: int32 [n, 4] on the device, (request, row and query head, of its kv head's, of the first pair, pairs); None where row t is request t's."""

    def __init__(self, batch, cache: Cache8, dt: int, n_heads: int, window: int, limit: int):
        _heads(cache, n_heads, window)
        G = n_heads // cache.n_kv_heads
        some = [(r, a, c, n) for r, (a, c, n) in enumerate(zip(batch.h_q_start, batch.h_ctx_len, batch.h_q_len)) if n < limit or not limit]
        most, last = max([1] + [n for *_, n in some]), batch.max_pos if not limit else max(c + n - 1 for _, _, c, n in some)
        self.nt = min(4, -(-most * G // 8))
        self.tiles, self.n_tiles, tiles = None, batch.n_rows, batch.n_rows * -(-G // (8 * self.nt))
        if not _single_rows(batch):
            counts = np.array([-(-n * G // (8 * self.nt)) for *_, n in some])
            numbers = np.empty((int(counts.sum()), 4), dtype=np.int32)
            request, row, pairs = (np.repeat(np.array(x, dtype=np.int64), counts) for x in ([r for r, *_ in some], [a for _, a, *_ in some], [n * G for *_, n in some]))
            pair = (np.arange(len(numbers)) - np.repeat(np.cumsum(counts) - counts, counts)) * 8 * self.nt
            for i, column in enumerate((request, row + pair // G, pair % G, np.minimum(8 * self.nt, pairs - pair))):
                numbers[:, i] = column
            self.tiles, self._host = _to_device(numbers, batch)
            self.n_tiles = tiles = len(numbers)
        seen = min(last + 1, window + most) if window else last + 1
        mean = sum(min(c + n, seen) for _, _, c, n in some) / max(1, len(some))
        self.ranks = _ranks(tiles * cache.n_kv_heads, seen, mean, functools.partial(_clusters, dt, cache.code, cache.head_dim, self.nt))
        # as the binding reads it (Cut in csrc/cache8_binding.cpp)
        self._native = np.array([batch.n_rows, batch.n_requests, self.n_tiles, self.nt, self.ranks, G, window, batch.max_pos], dtype=np.int64)
        self.native = self._native.ctypes.data


def _cut(batch, cache: Cache8, dt: int, n_heads: int, window: int, limit: int) -> _Cut:
    key = ("cache8 cut", cache.code, cache.k.shape[1:], dt, n_heads, window, limit)
    if _single_rows(batch):                                        # (nothing of it is on the device)
        cut = batch.extra.get(key)
        if cut is None:
            cut = batch.extra[key] = _Cut(batch, cache, dt, n_heads, window, limit)
        return cut
    return _on_stream(batch, key, lambda: _Cut(batch, cache, dt, n_heads, window, limit))


def _single_rows(batch) -> bool:
    """Whether row t is request t's, for all rows."""
    return batch.max_q_len == 1 and batch.n_rows == batch.n_requests


@functools.lru_cache(maxsize=None)
def _clusters(dt: int, code: int, head_dim: int, nt: int, ranks: int) -> int:
    """Clusters of `ranks` blocks of the kernel on warp MMAs that are on the GPU at once; 0 where it has no room for one (16 are more than every GPU need take)."""
    n = ops._fn("cache8", "hb_cache8_attention_mma_clusters")(dt, code, head_dim, nt, ranks)
    if n < 0:
        raise ops.KernelError(library.load("cache8").hb_last_error().decode())
    return n


def _ranks(tiles: int, keys: int, mean: float, clusters) -> int:
    """Blocks (1 to 16, a cluster) that share a tile's keys (`keys` the longest's, `mean` of all): as many as are on the GPU at once (`clusters`: of so
    many blocks), with 64 keys each while there is one on an SM, or two and clusters of 2, 4 and 8; else 270, or 512 in clusters of 3, 5, 6 and 7, which fill the
    GPU less evenly; more than 8 where they have an SM each, 16 with 128 keys each, 9 to 15 with 512. Measured, us within a graph: one request of 700 tokens (8 kv heads of 64)
    5.8 with 2, 4.9 with 4, 4.4 with 8, of 2,000 5.2 with 8, 5.0 with 16, of 8,000 9.4 and 7.5; 5 of 900 5.6 with 4, 6.3 with 7; 4 of 2,000 7.1 with 4, 6.4 with 8; 8 of
    2,000 8.5 with 4 and 7.7 to 8.1 with 8 (where the rule takes 4); 16 of 1,500 11.0 with 2, 9.7 with 4, 14.3 with 8; 32 of 500 7.4 with 1 and 8.2 with 2, of 700 10.1 and 9.6; 24 of 1,300 12.2 with 2 and 15.0
    with 3. Where lengths differ a wave of blocks ends with its longest: while a block still has 2,048 keys of a
    tile, or 1,450 of lengths that differ much, up to four waves (heads of 128: 64 requests of 8,000 tokens 169 as one wave of one block a tile, 163 as two, 167
    with four blocks; 64 of 4 to 8 thousand 140, 137 and 133; 48 of 3 to 6 thousand 79, 82 and 76; 96 of 2 to 4 thousand 111 and 102; 64 of 2,000 46 and 48)."""
    def fits(r):
        even = r in (2, 4, 8)
        if r > 8:
            least = 128 if r == 16 else 512
        elif tiles * r <= (2 * 148 if even else 148):
            least = 64
        else:
            least = 270 if even else 512
        return keys >= least * r and (r <= 8 or tiles * r <= 148) and clusters(r) >= tiles

    ranks = next((r for r in range(16, 1, -1) if fits(r)), 1)
    while 2 * ranks <= 8 and tiles <= 4 * clusters(2 * ranks) and keys >= (4096 if mean > 0.85 * keys else 2900) * ranks:
        ranks *= 2
    return ranks


COPY_PLANES, COPY_PAIRS = 8, 960                                   # CP_PLANES, CP_PAIRS of csrc/copy_pages.cu: of one launch


def copy_pages(planes: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Page src[i] to page dst[i], for every i, in all layers of all `planes` ([layers, pages, ...] each, a page's numbers side by side; of any types
    and sizes). src and dst are numbers of the host: pages below 0 or outside of a plane, a page copied to twice, and one both copied from and to
    are refused. A source may be copied to several pages."""
    there = bool(planes) and planes[0].is_cuda
    bound = _binding() if _bound is None and there else _bound
    if bound and there:
        done = bound.copy(planes, src, dst)
        if done is not None:
            _done(done, _copies(len(planes), len(src)))
            return
    pairs = [np.ascontiguousarray(x, dtype=np.int64) for x in (src, dst)]
    src, dst = pairs
    if src.ndim != 1 or src.shape != dst.shape:
        raise ops.KernelError(f"copy_pages: {src.shape} pages to {dst.shape}")
    _here("copy_pages", *planes)
    numbers = []
    for t in planes:
        inner = int(np.prod(t.shape[2:], dtype=np.int64)) if t.dim() >= 2 else 0
        if t.dim() < 2 or (t.numel() and not t[0, 0].is_contiguous()) or (t.shape[1] > 1 and inner and t.stride(1) < inner) or \
                (t.shape[0] > 1 and t.numel() and t.stride(0) < (t.shape[1] - 1) * t.stride(1) + inner):
            raise ops.KernelError(f"copy_pages: a plane {tuple(t.shape)}, strides {t.stride()}; [layers, pages, ...] with a page's numbers side by side is expected")
        if len(src) and (min(src.min(), dst.min()) < 0 or max(src.max(), dst.max()) >= t.shape[1]):
            raise ops.KernelError(f"copy_pages: pages {min(src.min(), dst.min())} to {max(src.max(), dst.max())} of a plane of {t.shape[1]}")
        if t.numel():
            e = t.element_size()
            numbers.append((t.data_ptr(), t.shape[0], t.stride(0) * e, t.stride(1) * e, inner * e))
    if len(set(dst.tolist())) != len(dst) or set(src.tolist()) & set(dst.tolist()):
        raise ops.KernelError("copy_pages: a page is copied to twice, or both copied from and to")
    if not len(src) or not numbers:
        return
    numbers, src, dst = np.array(numbers, dtype=np.int64), src.astype(np.int32), dst.astype(np.int32)
    library.launches[0] += _copies(len(numbers), len(src)) - 1      # (and the one that every call counts)
    ops._call("cache8", "hb_copy_pages", numbers.ctypes.data, len(numbers), src.ctypes.data, dst.ctypes.data, len(src), ops._stream())


def _copies(planes: int, pairs: int) -> int:
    """Launches that copying so many pairs of pages in so many planes takes."""
    return -(-planes // COPY_PLANES) * -(-pairs // COPY_PAIRS)


_bound = None


def _binding():
    """The binding (csrc/cache8_binding.cpp), at the addresses of the library's calls; False where it cannot be had."""
    global _bound
    lib, module = library.load("cache8"), library.load_binding("cache8")
    if module is not None:
        module.bind(*(C.cast(getattr(lib, name), C.c_void_p).value
                      for name in ("hb_cache8_store", "hb_cache8_expand", "hb_cache8_attention_mma", "hb_copy_pages", "hb_cache8_portions")),
                    C.cast(library.load("fast").hb_flash_prefill_tc_cache8, C.c_void_p).value)
    _bound = module or False
    return _bound


def _done(result, launches: int):
    """What a call through the binding gave; an int other than 0: which library's call failed (above 0 cache8's, below the flash kernel's), whose words say why."""
    if result.__class__ is int and result:
        raise ops.KernelError(library.load("cache8" if result > 0 else "fast").hb_last_error().decode())
    library.launches[0] += launches
    return result
