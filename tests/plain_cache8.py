"""Plain statements of the 8-bit cache's operators, row by row: storing in 32 bits, operation by operation as the kernels round them (the codes and
scales have to be equal), attention in 64 bits."""
import numpy as np
import torch

BLOCK = 16
MOST = {torch.int8: np.float32(127), torch.float8_e4m3fn: np.float32(448)}


def values(codes: torch.Tensor) -> np.ndarray:
    return codes.float().cpu().numpy()


def nearest(x: np.ndarray, dtype) -> torch.Tensor:
    x = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
    return x.round().to(torch.int8) if dtype == torch.int8 else x.to(dtype)


def store(rows: torch.Tensor, slots, codes: torch.Tensor, scales: torch.Tensor):
    """(codes, scales) after rows [T, heads * D] went to `slots`; the inputs stay as they are (all on the CPU)."""
    pages, heads, ps, D = codes.shape
    dtype, most = codes.dtype, MOST[codes.dtype]
    x = rows.float().numpy().reshape(len(slots), heads, D)
    codes, scales = codes.clone(), scales.numpy().copy()
    last = {s: t for t, s in enumerate(slots) if 0 <= s < pages * ps}                 # of several rows for one place the last
    for page, b in {(s // ps, s % ps // BLOCK) for s in last}:
        first = b * BLOCK
        there = [s for s in range(page * ps + first, page * ps + min(ps, first + BLOCK)) if s in last]
        part = x[[last[s] for s in there]]
        largest = np.where(np.isfinite(part), np.abs(part), np.float32(0)).max((0, 2))
        new = np.maximum(largest, np.float32(1e-30)) / most
        if page * ps + first not in last:
            old = scales[page, :, b].copy()
            for h in range(heads):
                if new[h] > old[h]:
                    at = codes[page, h, first:first + BLOCK]
                    at.view(torch.uint8).copy_(nearest(at.float().numpy() * (old[h] / new[h]), dtype).view(torch.uint8))
            new = np.maximum(old, new)
        scales[page, :, b] = new
        inv = np.float32(1) / new
        with np.errstate(invalid="ignore", over="ignore"):
            y = np.clip(part * inv[None, :, None], -most, most)
        y = nearest(np.where(np.isnan(y), np.float32(0), y), dtype).view(torch.uint8)
        for s, row in zip(there, y):
            codes.view(torch.uint8)[page, :, s % ps] = row
    return codes, torch.from_numpy(scales)


def numbers(codes: torch.Tensor, scales: torch.Tensor) -> np.ndarray:
    """[pages, heads, page_size, D] in 64 bits."""
    ps = codes.shape[2]
    return values(codes).astype(np.float64) * np.repeat(scales.double().cpu().numpy(), BLOCK, -1)[:, :, :ps, None]


def attend(q, cache, table, row_request, positions, n_heads, window, scale):
    """[T, heads * D] in 64 bits; cache: (k, v, k_scale, v_scale)."""
    k, v, ks, vs = cache
    K, V = numbers(k, ks), numbers(v, vs)
    pages, Hkv, ps, D = k.shape
    G = n_heads // Hkv
    q = q.double().cpu().numpy().reshape(len(positions), Hkv, G, D)
    out = np.zeros_like(q)
    for t, (r, p) in enumerate(zip(row_request, positions)):
        lo = max(0, p - window + 1) if window else 0
        at = [(int(table[r][j // ps]), j % ps) for j in range(lo, min(p + 1, len(table[r]) * ps))]
        at = [(a, b) for a, b in at if 0 <= a < pages]
        if not at:
            continue
        ids, places = np.array([a for a, _ in at]), np.array([b for _, b in at])
        s = np.einsum("hgd,nhd->hgn", q[t], K[ids, :, places]) * scale
        w = np.exp(s - s.max(-1, keepdims=True))
        out[t] = np.einsum("hgn,nhd->hgd", w, V[ids, :, places]) / w.sum(-1, keepdims=True)
    return out.reshape(len(positions), n_heads * D)
