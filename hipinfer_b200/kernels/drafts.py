"""Operators of a step that samples many continuations behind shared pages, with drafted tokens: attention over a paged cache in which
groups of requests share a long prefix (computed once for all of a group's rows), and the verification of drafted tokens against the
target's logits. Reached as `ops.SharedPlan`, `ops.attention_shared` and `ops.verify_drafts` (csrc/shared_plan.cu, attention_shared.cu, attention_shared_tc.cu,
verify_drafts.cu; drafts_binding.cpp makes the calls whose arguments are as they should be).

The reference has neither: its batch slots hold a copy of the prompt each (src/api.cu:1409-1411), and its `verify_step` (2029-2060) returns
logits and leaves the choice to the caller."""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import library, ops

_p, _i, _l, _f = C.c_void_p, C.c_int, C.c_long, C.c_float
ops._SIGS["drafts"] = {
    "hb_shared_plan": [_p, _p, _i, _p, _i, _i, _i, _i, _i, _i, _i, _f, _f, _f, _i, _f, _p, _i],
    "hb_attention_shared": [_p, _l, _p, _p, _l, _p, _i, _p, _p, _p, _p, _f, _i, _p, _p],
    "hb_shared_items_tc_supported": [_i, _i, _i, _i],
    "hb_verify_drafts": [_p, _i, _l, _i, _i, _p, _p, _p, _i, _i, _p, _p, _p, _l, _p, _i, _l, _l, _p, _p, _p, _p, _p],
    "hb_verify_drafts_workspace": [_i, _i, _i, _i],
}
MAX_DRAFTS = 63

# the header of a plan (csrc/shared_plan.h)
_ITEMS, _CTAS, _PARTS, _TOKENS, _MAX_ROWS, _OFF_ITEMS, _OFF_CTAS, _OFF_TOKENS, _INTS, _MASKED = range(10)
_HEADER = 16


def plan_numbers(q_lens, ctx_lens, groups, n_heads: int, n_kv_heads: int, tile_tokens: int, narrow_tokens: int, key_tile: int, n_ctas: int,
                 item_cost: float, wide_cost: float, part_cost: float, few_tokens: int = 0, few_cost: float = 1.0) -> np.ndarray:
    """The plan as int32 numbers (csrc/shared_plan.cu, which runs on the host); raises KernelError for lengths that make none."""
    q, c = (np.ascontiguousarray(x, dtype=np.int32) for x in (q_lens, ctx_lens))
    g = np.ascontiguousarray(groups, dtype=np.int32).reshape(-1, 3)
    if q.ndim != 1 or q.shape != c.shape:
        raise ops.KernelError(f"a plan needs one number of rows and one length a request, got {q.shape} and {c.shape}")
    fn = ops._fn("drafts", "hb_shared_plan")
    cap = 32768 + 16 * int(q.clip(0).sum())
    while True:
        out = np.empty(cap, dtype=np.int32)
        n = fn(q.ctypes.data, c.ctypes.data, len(q), g.ctypes.data, len(g), n_heads, n_kv_heads, tile_tokens, narrow_tokens, key_tile, n_ctas,
               item_cost, wide_cost, part_cost, few_tokens, few_cost, out.ctypes.data, cap)
        if n > 0:
            return out[:n]
        if n == 0:
            raise ops.KernelError(library.load("drafts").hb_last_error().decode())
        cap = -n


class SharedPlan:
    """How a step's rows attend to a paged cache whose requests share prefixes; made from the lengths alone, once a step, and used by every
    layer of that step whose heads and pages are these.

    q_lens[r] rows of request r (its rows are consecutive, requests one after the other) stand at positions ctx_lens[r], ...; a row sees the
    keys up to its own. groups: (first request, requests, shared tokens): the block tables of these requests name the same pages for the
    positions below `shared tokens` (which need not be a multiple of the page size). Requests of no group, and groups of which fewer than two
    bring rows, attend on their own. The plan's numbers are copied to the device on the current stream, and a call's kernels read them: on
    another stream it is used, and let go, only when that one has waited for this and the other way round, as with any tensor."""

    def __init__(self, q_lens: Sequence[int], ctx_lens: Sequence[int], groups: Sequence[Tuple[int, int, int]], n_heads: int, n_kv_heads: int,
                 head_dim: int, page_size: int, dtype: torch.dtype, device="cuda:0"):
        if n_kv_heads < 1 or n_heads < n_kv_heads or n_heads % n_kv_heads:
            raise ops.KernelError(f"attention_shared: {n_heads} heads are not a multiple of {n_kv_heads} kv heads")
        if not 1 <= head_dim <= 256 or page_size < 1 or dtype not in ops._DT:
            raise ops.KernelError(f"attention_shared: heads of {head_dim}, pages of {page_size}, {dtype} are not supported")
        self.n_heads, self.n_kv_heads, self.head_dim, self.page_size, self.dtype = n_heads, n_kv_heads, head_dim, page_size, dtype
        self.device = torch.device(device)
        self.n_requests = len(q_lens)
        group = n_heads // n_kv_heads
        # on the tensor cores: one CTA an SM, items of two chains of up to 128 rows each
        self.tensor_cores = (dtype == torch.bfloat16 and ops.fast_kernels_on()
                             and bool(ops._fn("drafts", "hb_shared_items_tc_supported")(n_heads, n_kv_heads, head_dim, page_size)))
        # (costs in key tiles of an item of few rows, 1.3 us; of 37 settings the best over 76 sizes, an item at 0.9 was 2 % slower; csrc/shared_plan.cu)
        if self.tensor_cores:
            cut, costs = (2 * (128 // group), 128 // group, 128, _sms(self.device)), (1.6, 1.8, head_dim * 1e-6)
        else:
            cut = (max(1, 64 // group), 0, 64, (2 if head_dim <= 64 else 1) * _sms(self.device))         # (as many as are resident)
            costs = (0.6, 1.0, head_dim * 1e-6, 16 // group, 0.4)      # (in tiles of 64 rows; up to 16 rows go another way)
        numbers = plan_numbers(q_lens, ctx_lens, groups, n_heads, n_kv_heads, *cut, *costs)
        self.rows, self.parts = int(numbers[_TOKENS]), int(numbers[_PARTS])
        self.ctas, self.max_rows = int(numbers[_CTAS]), int(numbers[_MAX_ROWS])
        self.most_keys = max((int(c) + int(n) for c, n in zip(ctx_lens, q_lens) if n), default=0)
        self.q_shape, self.page_shape = (self.rows, n_heads * head_dim), (n_kv_heads, page_size, head_dim)
        self.size, self.default_scale = 2 if dtype == torch.bfloat16 else 4, 1.0 / math.sqrt(head_dim)
        self.workspace = self.parts * (head_dim + 2) + 4           # floats
        self._launch = np.array([self.rows, self.ctas, self.max_rows, cut[1], self.parts, self.tensor_cores, ops._DT[dtype], n_heads, n_kv_heads,
                                 head_dim, page_size, numbers[_OFF_ITEMS], numbers[_OFF_CTAS], numbers[_OFF_TOKENS], numbers[_MASKED]],
                                dtype=np.int32)      # SharedLaunch of csrc/attention_shared.cu
        self.launch = self._launch.ctypes.data
        host = torch.from_numpy(numbers)
        if self.device.type == "cuda":
            host = host.pin_memory()
        self.numbers = host.to(self.device, non_blocking=True)
        self._host = host                     # until the copy is over
        # as the binding reads it (Plan in csrc/drafts_binding.cpp)
        self._native = np.array([self.rows, n_heads * head_dim, n_kv_heads, page_size, head_dim, ops._DT[dtype], self.n_requests, self.most_keys,
                                 self.workspace if self.parts else 0, self.ctas, self.numbers.data_ptr(), self.launch, 0], dtype=np.int64)
        self._native[12:].view(np.float64)[0] = self.default_scale
        self.native = self._native.ctypes.data


def _sms(device) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count if device.type == "cuda" else 148


def attention_shared(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, plan: SharedPlan,
                     out: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the plan's rows over their requests' pages. q [T, Hq D] (rows may be part of wider ones); caches [page, Hkv, page_size, D]
    of the same type; block_table int32 [R, pages]; out [T, Hq D]; scale 1 / sqrt(D) by default. Scores, softmax and sums are 32-bit; the
    keys' cut, and with it a result's last bits, is a matter of the plan."""
    if q.is_cuda:
        bound = _binding() if _bound is None else _bound
        if bound:
            result = bound.attend(q, k_cache, v_cache, block_table, plan.native, out, scale, ops.fast._status_ptr())
            if result is not None:
                return _done(result, 1 + (plan.ctas > 0))
    width, dtype, T, pages = plan.n_heads * plan.head_dim, plan.dtype, plan.rows, k_cache.shape
    if not (q.is_cuda and k_cache.is_cuda and v_cache.is_cuda and block_table.is_cuda):
        ops._need_cuda(q, k_cache, v_cache, block_table)
    if q.shape != plan.q_shape or q.dtype is not dtype or q.stride(1) != 1:
        raise ops.KernelError(f"attention_shared: q {tuple(q.shape)} {q.dtype}, strides {q.stride()}; the plan has {T} rows of {plan.n_heads} heads of "
                              f"{plan.head_dim}, {dtype}")
    if not (pages == v_cache.shape and pages[1:] == plan.page_shape and k_cache.dtype is dtype and v_cache.dtype is dtype and k_cache.is_contiguous()
            and v_cache.is_contiguous()):
        raise ops.KernelError(f"attention_shared: keys {tuple(pages)} {k_cache.dtype}, values {tuple(v_cache.shape)} {v_cache.dtype}; {pages[0]} pages of "
                              f"{plan.n_kv_heads} heads x {plan.page_size} tokens x {plan.head_dim}, {dtype}, are expected")
    if block_table.dim() != 2 or block_table.dtype is not torch.int32 or block_table.stride(1) != 1 or block_table.shape[0] != plan.n_requests \
            or block_table.shape[1] * plan.page_size < plan.most_keys:
        raise ops.KernelError(f"attention_shared: block table {tuple(block_table.shape)} {block_table.dtype}; the plan has {plan.n_requests} requests of up "
                              f"to {plan.most_keys} tokens in pages of {plan.page_size}")
    if out is None:
        out = torch.empty(T, width, dtype=dtype, device=q.device)
    elif out.shape != plan.q_shape or out.dtype is not dtype or not out.is_contiguous() or not out.is_cuda:
        ops._need_cuda(out)
        raise ops.KernelError(f"attention_shared: out {tuple(out.shape)} {out.dtype}, strides {out.stride()}")
    if not T:
        return out
    ws = torch.empty(plan.workspace, dtype=torch.float32, device=q.device) if plan.parts else None
    qp, kp, vp, op, ld = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), q.stride(0)
    aligned = int((ld * plan.size) % 16 == 0 and (qp | kp | vp | op) % 16 == 0)
    library.launches[0] += plan.ctas > 0
    ops._call("drafts", "hb_attention_shared", qp, ld, kp, vp, pages[0], block_table.data_ptr(), block_table.stride(0), plan.numbers.data_ptr(), plan.launch,
              None if ws is None else ws.data_ptr(), op, plan.default_scale if scale is None else scale, aligned, ops.fast._status_ptr(),
              library.current_stream())
    return out


_bound = None


def _binding():
    """The binding (csrc/drafts_binding.cpp), at the addresses of the library's calls; False where it cannot be had."""
    global _bound
    lib, module = library.load("drafts"), library.load_binding("drafts")
    if module is not None:
        module.bind(*(C.cast(getattr(lib, name), C.c_void_p).value
                      for name in ("hb_attention_shared", "hb_verify_drafts", "hb_verify_drafts_workspace")))
    _bound = module or False
    return _bound


def _done(result, launches: int):
    """What a call through the binding gave."""
    if result.__class__ is int:
        raise ops.KernelError(library.load("drafts").hb_last_error().decode())
    library.launches[0] += launches
    return result


def verify_drafts(logits: torch.Tensor, start: torch.Tensor, n_drafts: torch.Tensor, drafts: torch.Tensor, temperature: torch.Tensor,
                  uniform: torch.Tensor, noise: torch.Tensor, draft_probs: Optional[torch.Tensor] = None):
    """Accepts or refuses drafted tokens so that what is produced is distributed as if the target, whose logits are given, alone had drawn it. (Where
    logits behind a cache in 8 bits are computed with drafts in the cache, the drafts have part in its rounding.)

    Request r has n_drafts[r] drafts in row r of `drafts` (int32 [R, K]) and n_drafts[r] + 1 rows of logits ([T, V], float32 or bfloat16) from row
    start[r] on; p_i is the softmax of the i-th over `temperature[r]` (float32 [R]; 0 or less: greedy, a point mass on the lowest index of the largest
    logit, which is also what a row without a finite largest logit is; NaN counts as above all). Draft i is accepted iff all before it are and
    uniform[r, i] * q_i(draft) < p_i(draft), with q_i = draft_probs[r, i] ([R, K, V], float32 or bfloat16), or 1 where no distributions are given (drafts
    that were looked up). The token behind the accepted ones is the arg max of w / noise[r] (float32 [R, V], exponential variates; ties: the lowest
    index), w = max(p_i - q_i, 0) at the first draft refused (p_i where that is 0 everywhere), p_{n+1} if none was.

    Returns (tokens int32 [R, K + 1]: accepted drafts, the token behind them, -1; counts int32 [R]: how many tokens; logprobs float32 [R, K + 1]:
    log p_i of each, at temperature 1 for a greedy request, 0 for a row without a finite largest logit and behind the last). A request whose
    first row lies outside the logits gets no token; where only its last ones do, the drafts that have no row behind them are not looked
    at, and the last row that is there is the one behind all drafts."""
    if logits.is_cuda:
        bound = _binding() if _bound is None else _bound
        if bound:
            result = bound.verify(logits, start, n_drafts, drafts, temperature, uniform, noise, draft_probs)
            if result is not None:
                return _done(result, 2)
    ops._need_cuda(logits, start, n_drafts, drafts, temperature, uniform, noise, draft_probs)
    if logits.dim() != 2 or drafts.dim() != 2:
        raise ops.KernelError(f"verify_drafts: logits {tuple(logits.shape)} and drafts {tuple(drafts.shape)}, [T, V] and [R, K] are expected")
    (T, V), (R, K) = logits.shape, drafts.shape
    if logits.stride(1) != 1 and V > 1:
        raise ops.KernelError(f"verify_drafts: logits with strides {logits.stride()}, rows side by side are expected")
    if K > MAX_DRAFTS:
        raise ops.KernelError(f"verify_drafts: {K} drafts a request, at most {MAX_DRAFTS}")
    _vector(drafts, torch.int32, R * K, "drafts")
    _vector(start, torch.int32, R, "start")
    _vector(n_drafts, torch.int32, R, "n_drafts")
    _vector(temperature, torch.float32, R, "temperature")
    _vector(uniform, torch.float32, R * K, "uniform")
    if noise.shape != (R, V) or noise.dtype != torch.float32 or (V > 1 and noise.stride(1) != 1):
        raise ops.KernelError(f"verify_drafts: noise {tuple(noise.shape)} {noise.dtype}, strides {noise.stride()}; float32 [{R}, {V}] is expected")
    probs = (None, 0, 0, 0)
    if draft_probs is not None:
        if draft_probs.shape != (R, K, V) or draft_probs.dtype not in ops._DT or (V > 1 and draft_probs.stride(2) != 1):
            raise ops.KernelError(f"verify_drafts: draft_probs {tuple(draft_probs.shape)} {draft_probs.dtype}, strides {draft_probs.stride()}; [{R}, {K}, {V}] "
                                  f"is expected")
        if K:
            probs = (draft_probs.data_ptr(), ops._DT[draft_probs.dtype], draft_probs.stride(0), draft_probs.stride(1))
    dt = ops._dt(logits)
    device = logits.device
    tokens, counts = torch.empty(R, K + 1, dtype=torch.int32, device=device), torch.empty(R, dtype=torch.int32, device=device)
    logprobs = torch.empty(R, K + 1, dtype=torch.float32, device=device)
    if not R:
        return tokens, counts, logprobs
    if not V:
        raise ops.KernelError("verify_drafts: empty vocabulary")
    ws = torch.empty(_workspace(R, K, V, dt), dtype=torch.float32, device=device)
    library.launches[0] += 1
    ops._call("drafts", "hb_verify_drafts", logits.data_ptr(), dt, logits.stride(0), T, V, start.data_ptr(), n_drafts.data_ptr(), drafts.data_ptr(), R, K,
              temperature.data_ptr(), uniform.data_ptr(), noise.data_ptr(), noise.stride(0), *probs, ws.data_ptr(), tokens.data_ptr(), counts.data_ptr(),
              logprobs.data_ptr(), library.current_stream())
    return tokens, counts, logprobs


@functools.lru_cache(maxsize=256)
def _workspace(R: int, K: int, V: int, dt: int) -> int:
    """Floats that the two kernels of a verification of this size meet in."""
    n = ops._fn("drafts", "hb_verify_drafts_workspace")(R, K, V, dt)
    if n < 0:
        raise ops.KernelError(f"verify_drafts: {R} requests of {K} drafts, a vocabulary of {V}: too many")
    return n


def _vector(x, dtype, n, what):
    if x.dtype is not dtype or x.numel() != n or not x.is_contiguous():
        raise ops.KernelError(f"verify_drafts: {what} {tuple(x.shape)} {x.dtype}, strides {x.stride()}; {n} of {dtype} side by side are expected")
