"""Operators of a paged cache in 8 bits: storing a step's keys and values, reading pages back, attention over it; and copying pages of a cache
of any type, as forks inside a page need it. Reached as `ops.Cache8`, `ops.new_cache8`, `ops.store_cache8`, `ops.expand_cache8`, `ops.attention_cache8`
and `ops.copy_pages` (csrc/cache8_store.cu, cache8_attention.cu, copy_pages.cu).

A cache holds, for keys and for values, codes [page, kv head, page_size, head_dim] (int8, or e4m3) and scales float32 [page, kv head, blocks], one
for each block of 16 places of a page (the last block of a page may have fewer); a place's numbers are code * scale.

The reference keeps its cache in the activations' type (src/api.cu:1409-1411) and copies nothing within it."""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import library, ops

_p, _i, _l, _f = C.c_void_p, C.c_int, C.c_long, C.c_float
ops._SIGS["cache8"] = {
    "hb_cache8_store": [_p, _p, _l, _l, _i, _p, _i, _i, _i, _i, _l, _i, _p, _p, _p, _p, _p],
    "hb_cache8_expand": [_p, _p, _p, _p, _i, _p, _p, _l, _l, _i, _i, _i, _p, _p, _i, _p],
    "hb_cache8_attention_any": [_p, _i, _l, _p, _p, _p, _p, _i, _l, _i, _i, _i, _p, _l, _i, _i, _p, _p, _i, _i, _i, _f, _p, _p],
    "hb_cache8_attention_mma": [_p, _i, _l, _p, _p, _p, _p, _i, _l, _i, _i, _i, _p, _l, _i, _i, _p, _p, _p, _i, _i, _i, _i, _i, _f, _p, _p],
    "hb_cache8_attention_mma_supported": [_i, _i, _i, _l],
    "hb_copy_pages": [_p, _i, _p, _p, _i, _p],
}
BLOCK8 = 16                                                        # places of a page that share a scale
CODES = {torch.int8: 2, torch.float8_e4m3fn: 3}                    # csrc/cache8.cuh


def cache8_blocks(page_size: int) -> int:
    """Scales of a page and head."""
    return -(-page_size // BLOCK8)


@dataclass(frozen=True)
class Cache8:
    """A layer's cache in 8 bits: codes k, v [pages, n_kv_heads, page_size, head_dim], scales k_scale, v_scale [pages, n_kv_heads, blocks]."""

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


def store_cache8(k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor, cache: Cache8) -> Cache8:
    """Rows k, v [T, n_kv_heads * head_dim] (float32 or bfloat16; rows may be part of wider ones) stored at the places slot_map (int32 [T], page *
    page_size + place; a number outside of the cache stores nothing).

    Rows may come in any order; of several for one place the last counts, and the others are as if they were not there. A block (16 places of a page)
    one of whose rows goes to its first place begins anew: its scale is max(a, 1e-30) / M, a being the largest |x| of the block's rows and head, M
    the largest code (127, or 448). In any other block the scale grows to that where it is larger, and the codes that are there are rounded to it once
    more: half a step each time that it grows. Numbers that are not finite do not count for a: infinities become the largest code, NaN becomes 0.
    Places of a block that no row goes to keep their codes where the scale stays or begins anew. A cache has at most 2^31 - 1 places."""
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
    _here("expand_cache8", pages, *cache.tensors)
    _ints("expand_cache8", "pages", pages)
    return _expand(cache, pages, None, pages.numel(), dtype)


def _expand(cache: Cache8, table: torch.Tensor, index: Optional[torch.Tensor], n: int, dtype: torch.dtype):
    """Page i of the result is page table[i], or table.flatten()[index[i]], of the cache."""
    if dtype not in ops._DT:
        raise ops.KernelError(f"expand_cache8: element type {dtype} is not supported (float32 and bfloat16 are)")
    k, v = (torch.empty((n,) + cache.k.shape[1:], dtype=dtype, device=cache.k.device) for _ in range(2))
    if n and k.numel():
        ops._call("cache8", "hb_cache8_expand", *(t.data_ptr() for t in cache.tensors), cache.code, table.data_ptr(), ops._ptr(index), n, cache.k.shape[0],
                  *cache.k.shape[1:], k.data_ptr(), v.data_ptr(), ops._DT[dtype], ops._stream())
    return k, v


def attention_cache8(q: torch.Tensor, cache: Cache8, batch, group: int, n_heads: int, window: int = 0, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the step's rows (`batch`: an engine.batch.StepBatch) over their requests' pages of cache group `group`, whose keys and values,
    the step's own among them, are in `cache`. q [T, n_heads * head_dim] (bfloat16 or float32; rows may be part of wider ones), out [T, n_heads *
    head_dim] of its type; query head h reads kv head h // (n_heads / n_kv_heads). A row at position p sees the keys j <= p (and j > p - window,
    for a window above 0) whose pages are in the block table and in the cache; one that sees none is 0. scale: 1 / sqrt(head_dim) by default. Scores,
    softmax and sums are 32-bit. Codes at places that a row of the step sees are numbers (e4m3 has a NaN; storing leaves none)."""
    table = batch.block_tables[group]
    _here("attention_cache8", q, table, batch.positions, batch.row_request, *cache.tensors, out)
    T, D = batch.n_rows, cache.head_dim
    if n_heads < 1 or n_heads % cache.n_kv_heads:
        raise ops.KernelError(f"attention_cache8: {n_heads} heads are not a multiple of {cache.n_kv_heads} kv heads")
    if D > 256:
        raise ops.KernelError(f"attention_cache8: heads of {D}, at most 256")
    if q.shape != (T, n_heads * D) or q.stride(1) != 1:
        raise ops.KernelError(f"attention_cache8: q {tuple(q.shape)}, strides {q.stride()}; {T} rows of {n_heads} heads of {D} are expected")
    dt = ops._dt(q)
    if table.dim() != 2 or table.dtype != torch.int32 or table.stride(1) != 1 or table.shape[0] != batch.n_requests:
        raise ops.KernelError(f"attention_cache8: block table {tuple(table.shape)} {table.dtype} of {batch.n_requests} requests")
    if window < 0:
        raise ops.KernelError(f"attention_cache8: window {window}")
    if out is None:
        out = torch.empty(T, n_heads * D, dtype=q.dtype, device=q.device)
    elif out.shape != (T, n_heads * D) or out.dtype != q.dtype or not out.is_contiguous():
        raise ops.KernelError(f"attention_cache8: out {tuple(out.shape)} {out.dtype}, strides {out.stride()}")
    if not T:
        return out
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    single = batch.max_q_len == 1 and T == batch.n_requests
    if _on_tensor_cores(cache):
        _attend_mma(q, dt, cache, batch, table, single, n_heads // cache.n_kv_heads, int(window), scale, out)
        return out
    ops._call("cache8", "hb_cache8_attention_any", q.data_ptr(), dt, q.stride(0), *(t.data_ptr() for t in cache.tensors), cache.code, cache.k.shape[0],
              cache.n_kv_heads, cache.page_size, D, table.data_ptr(), table.stride(0), table.shape[0], table.shape[1],
              None if single else batch.row_request.data_ptr(), batch.positions.data_ptr(), T, n_heads // cache.n_kv_heads, int(window), scale,
              out.data_ptr(), ops._stream())
    return out


def _on_tensor_cores(cache: Cache8) -> bool:
    """Whether the kernel on warp MMAs takes the cache's sizes and place in memory (csrc/cache8_attention_mma.cu)."""
    return (ops.fast_kernels_on() and (cache.k.data_ptr() | cache.v.data_ptr()) % 16 == 0
            and bool(ops._fn("cache8", "hb_cache8_attention_mma_supported")(cache.n_kv_heads, cache.page_size, cache.head_dim, cache.k.shape[0])))


def _attend_mma(q, dt, cache: Cache8, batch, table, single: bool, G: int, window: int, scale: float, out) -> None:
    pairs = G if single else batch.max_q_len * G
    nt = 1 if pairs <= 8 else 2 if pairs <= 16 else 4
    tiles = None if single else _tiles(batch, G, nt)
    n_tiles = batch.n_rows if single else tiles.shape[0]
    keys = min(batch.max_pos + 1, window + batch.max_q_len) if window else batch.max_pos + 1
    ops._call("cache8", "hb_cache8_attention_mma", q.data_ptr(), dt, q.stride(0), *(t.data_ptr() for t in cache.tensors), cache.code, cache.k.shape[0],
              cache.n_kv_heads, cache.page_size, cache.head_dim, table.data_ptr(), table.stride(0), table.shape[0], table.shape[1],
              None, batch.positions.data_ptr(), ops._ptr(tiles), n_tiles, nt,
              _ranks(n_tiles * (-(-G // (8 * nt)) if single else 1) * cache.n_kv_heads, keys), G, window, scale, out.data_ptr(), ops._stream())


def _ranks(tiles: int, keys: int) -> int:
    """Blocks that share a tile's keys."""
    ranks = 1
    while ranks < 8 and tiles * ranks < 4 * 148 and keys > 64 * ranks:
        ranks *= 2
    return ranks


def _tiles(batch, G: int, nt: int) -> torch.Tensor:
    """int32 [tiles, 4] on the device: (request, its first row, first (row, head) pair, pairs of its rows), pairs in tiles of 8 nt."""
    key = ("cache8 tiles", G, nt)
    if key not in batch.extra:
        parts = []
        for r, (start, n) in enumerate(zip(batch.h_q_start, batch.h_q_len)):
            first = np.arange(0, n * G, 8 * nt, dtype=np.int32)
            part = np.empty((len(first), 4), dtype=np.int32)
            part[:, 0], part[:, 1], part[:, 2], part[:, 3] = r, start, first, n * G
            parts.append(part)
        host = torch.from_numpy(np.concatenate(parts))
        host = host.pin_memory() if batch.tokens.is_cuda else host
        batch.extra[key] = host.to(batch.tokens.device, non_blocking=True), host       # (the host's copy until the other is over)
    return batch.extra[key][0]


def copy_pages(planes: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Page src[i] to page dst[i], for every i, in all layers of all `planes` ([layers, pages, ...] each, a page's numbers side by side; of any types
    and sizes). src and dst are numbers of the host: pages below 0 or outside of a plane, a page copied to twice, and one both copied from and to
    are refused. A source may be copied to several pages."""
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
    if len(np.unique(dst)) != len(dst) or np.intersect1d(src, dst).size:
        raise ops.KernelError("copy_pages: a page is copied to twice, or both copied from and to")
    if not len(src) or not numbers:
        return
    numbers, src, dst = np.array(numbers, dtype=np.int64), src.astype(np.int32), dst.astype(np.int32)
    ops._call("cache8", "hb_copy_pages", numbers.ctypes.data, len(numbers), src.ctypes.data, dst.ctypes.data, len(src), ops._stream())
