"""Attention over a cache in 8 bits in bfloat16 against 64 bits, within bounds that a missing key, another block's scale or a window off by one pass
(tests/cache8_bounds.py; test_cache8_bounds_cpu.py shows that they do): single rows and short portions."""
import pytest
import torch

import cache8_bounds as bounds
from hipinfer_b200.kernels import cache8, ops
from test_gpu_cache8 import CODES, DEV, STEPS, filled, ids, on_gpu, step

pytestmark = pytest.mark.gpu
SIZES = [(32, 8, 16, 64), (8, 2, 16, 128), (7, 1, 32, 128), (4, 4, 64, 64), (6, 2, 8, 64), (24, 1, 16, 64), (2, 1, 24, 80), (4, 2, 16, 256), (40, 1, 16, 128), (3, 1, 5, 3)]


def off(held, rows, heads, kv_heads, ps, D, codes, window=0, scale=None, seed=1):
    batch, tables, pages = step(held, rows, ps, window)
    q = torch.randn(sum(rows), heads * D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    cache = filled(pages, kv_heads, ps, D, codes)
    want, bound = bounds.attend(q, cache, tables, held, rows, heads, window, scale)
    return bounds.beyond(ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, heads, window=window, scale=scale), want, bound)


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("heads, kv_heads, ps, D", SIZES)
@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_attention(name, heads, kv_heads, ps, D, codes):
    held, rows = STEPS[name]
    assert off(held, rows, heads, kv_heads, ps, D, codes) <= 1


@pytest.mark.parametrize("window", [1, 2, 16, 100, 1000])
@pytest.mark.parametrize("name", ["decode", "drafts", "mixed"])
@pytest.mark.parametrize("heads, kv_heads, ps, D", [(8, 2, 16, 64), (4, 1, 32, 128), (4, 2, 8, 40)])
def test_a_window(window, name, heads, kv_heads, ps, D):
    held, rows = STEPS[name]
    assert off(held, rows, heads, kv_heads, ps, D, torch.int8, window, 0.2, 2) <= 1


@pytest.mark.parametrize("group", [1, 5, 8, 9, 17, 33])
@pytest.mark.parametrize("held", [[130, 700, 1500, 64], [5000, 17, 2049, 4096]])
def test_every_number_of_blocks_a_tile(group, held, monkeypatch):
    for ranks in range(1, 17):
        monkeypatch.setattr(cache8, "_ranks", lambda *a: ranks)
        assert off(held, [1] * 4, 2 * group, 2, 32, 64, torch.int8, seed=7) <= 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("heads, ps, D", [(2, 16, 64), (9, 32, 64), (2, 16, 128), (17, 64, 128), (2, 8, 80), (1, 5, 33)])
@pytest.mark.parametrize("window", [0, 2000])
def test_every_key_of_a_long_range_counts_once(dtype, heads, ps, D, window):
    """Scores that are all alike, and key j the value 1 in dimension j mod D alone: a result is how many of the keys that its row sees have that dimension, over their number."""
    held, rows = [5000, 2998, 15, 700], [1, 3, 2, 1]
    batch, tables, pages = step(held, rows, ps, window)
    k, v, ks, vs = filled(pages, 1, ps, D, torch.int8)
    v.zero_()
    for t, h, n in zip(tables, held, rows):
        for j in range(max(0, h - window + 1) if window else 0, h + n):
            v[t[j // ps], 0, j % ps, j % D] = 64
    vs[:] = 1 / 64
    q = torch.zeros(sum(rows), heads * D, dtype=dtype, device=DEV)
    got = ops.attention_cache8(q, on_gpu((k, v, ks, vs)), batch, 0, heads, window=window).double().cpu().view(-1, heads, D)
    at = 0
    for h, n in zip(held, rows):
        for p in range(h, h + n):
            lo = max(0, p - window + 1) if window else 0
            count = torch.bincount(torch.arange(lo, p + 1) % D, minlength=D).double()
            # (the number of a dimension is off by 2^-8 of itself in bfloat16 for the result's rounding alone, weights of one power of two being exact: of 152 at most, 0.6,
            # where D is 33, in which a lost key is one of 1)
            assert ((got[at] * (p + 1 - lo) - count).abs() < 0.75).all()
            at += 1
