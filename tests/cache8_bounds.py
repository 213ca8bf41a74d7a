"""How far a bf16 row of attention over a cache in 8 bits may be off, row by row and head by head.

o = sum_j p_j v_j (weights p of sum 1, values v_j of D numbers) is computed with weights that are rounded to 16 bits on their way to the tensor cores: p_j (1 + e_j),
|e_j| <= 2^-8 (bf16; f16 2^-11), while their sum is taken of the weights before that rounding; then o is rounded to bf16, 2^-8 of itself. Codes and scales
are exact, queries are (or are rounded to 16 bits of their row's largest number, 2^-16 of it, which moves a score by some 2^-14), sums are 32-bit.
Over the D dimensions, in the root mean square:
  the last rounding                     2^-8 rms(o) at most;
  weights whose errors are alike        2^-8 rms(o) at most (all of the row's weights the same number);
  weights whose errors are not          2^-8 sqrt(sum_j p_j^2 rms(v_j)^2): the sum of independent terms; twice that, so that for up to four
                                        weights, where nothing averages, it is what sum_j p_j rms(v_j) would be.
In all 2^-8 (2 rms(o) + 2 sqrt(sum_j p_j^2 rms(v_j)^2)). The root mean square has D numbers to average over, so a row that passes is off by rounding and not by a key, a
scale or a page: tests on the CPU apply it to results that lack one."""
import numpy as np
import torch

import plain_cache8 as plain


def attend(q, cache, tables, held, rows, heads, window=0, scale=None, weights=None, sums=False):
    """(results, bounds): [T, heads, D] and [T, heads] in 64 bits, for requests that hold `held` tokens and bring `rows` rows; `weights`: a type that weights are
    rounded to when their sum has been taken. With `sums` also sum_j p_j rms(v_j), [T, heads]."""
    k, v, ks, vs = cache
    K, V = (torch.from_numpy(plain.numbers(*plane)) for plane in ((k, ks), (v, vs)))
    pages, Hkv, ps, D = k.shape
    scale = D ** -0.5 if scale is None else scale
    G, x, at = heads // Hkv, q.double().cpu().view(-1, Hkv, heads // Hkv, D), 0
    out, bound, total = [], [], []
    for table, h, n in zip(tables, held, rows):
        if not n:
            continue
        j = torch.arange(h + n)
        page = torch.tensor([table[i] if i < len(table) else -1 for i in (j // ps).tolist()])
        there = (page >= 0) & (page < pages)
        kj, vj = (y[page.clamp(0, pages - 1), :, j % ps] if pages else torch.zeros(h + n, Hkv, D, dtype=torch.double) for y in (K, V))      # [keys, Hkv, D]
        for first in range(0, n, 256):
            p = torch.arange(h + first, h + min(n, first + 256))[:, None]
            seen = there[None] & (j[None] <= p)
            if window:
                seen &= j[None] > p - window
            s = torch.einsum("thgd,nhd->thgn", x[at + first:at + first + len(p)], kj) * scale
            s = s.masked_fill(~seen[:, None, None], -float("inf"))
            top = s.amax(-1, keepdim=True)
            w = torch.exp(s - torch.where(top.isinf(), 0.0, top))
            w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
            o = torch.einsum("thgn,nhd->thgd", w if weights is None else w.to(weights).double(), vj)
            spread = torch.einsum("thgn,nh->thg", w * w, vj.square().mean(-1)).sqrt()
            total.append(torch.einsum("thgn,nh->thg", w, vj.square().mean(-1).sqrt()).reshape(len(p), heads))
            out.append(o.reshape(len(p), heads, D))
            bound.append((2.0 ** -8 * (2 * o.square().mean(-1).sqrt() + 2 * spread)).reshape(len(p), heads))
        at += n
    return (torch.cat(out), torch.cat(bound)) + ((torch.cat(total),) if sums else ())


def beyond(got, want, bound):
    """The largest root mean square of a row's and head's errors over its bound (0 where both are 0)."""
    err = (got.double().cpu().view(want.shape) - want).square().mean(-1).sqrt()
    return float(torch.where(bound > 0, err / bound.clamp_min(1e-300), torch.where(err > 0, float("inf"), 0.0)).max()) if err.numel() else 0.0
