"""Portions over a cache in 8 bits on the flash kernel: the limit from which on a request's rows go there is set by the tests, and every call asserts that it
was launched. Bounds: tests/cache8_bounds.py."""
import pytest
import torch

import cache8_bounds as bounds
from hipinfer_b200.kernels import cache8, library, ops
from test_gpu_cache8 import CODES, DEV, filled, ids, on_gpu, same, step

pytestmark = pytest.mark.gpu


@pytest.fixture
def portions(monkeypatch):
    """attention_cache8 with requests of `limit` rows and more on the flash kernel (two launches, and one for other requests' rows)."""
    def attend(q, cache, batch, heads, window=0, scale=None, limit=16, **more):
        monkeypatch.setattr(cache8, "_portion_limit", lambda *a: limit)
        before = library.launches[0]
        got = ops.attention_cache8(q, cache, batch, 0, heads, window=window, scale=scale, **more)
        flash, others = (any(n > 0 and (n >= limit > 0) == there for n in batch.h_q_len) for there in (True, False))
        assert library.launches[0] - before == 2 * flash + others and flash == (limit > 0)
        return got
    return attend


def queries(n, seed=1):
    return torch.randn(n, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("size", [1e-30, 1e-29, 1.2e-28, 1e-20, 1e20, 1e30])
@pytest.mark.parametrize("codes", CODES, ids=ids)
@pytest.mark.parametrize("D", [64, 128])
def test_values_near_the_least_and_the_largest_numbers(D, codes, size, portions):
    """Blocks as storing leaves them for values of any size: as rows of one token read them."""
    held, rows, ps, heads = [40, 7], [33, 1], 16, 4
    batch, tables, pages = step(held, rows, ps)
    v = (queries(pages * ps * 2 * D, 2) * size).view(pages * ps, 2 * D).to(DEV)
    k = queries(pages * ps * 2 * D, 3).view(pages * ps, 2 * D).to(DEV)
    cache = ops.new_cache8(pages, 2, ps, D, codes, DEV)
    ops.store_cache8(k, v, torch.arange(pages * ps, dtype=torch.int32, device=DEV), cache)
    q = queries(sum(rows) * heads * D).view(-1, heads * D).to(torch.bfloat16)
    want, bound = bounds.attend(q, [t.cpu() for t in cache.tensors], tables, held, rows, heads)
    got = portions(q.to(DEV), cache, batch, heads)
    assert bounds.beyond(got, want, bound) <= 1
    assert float(want.abs().max()) > size / 10
