"""Storing many rows into a cache in 8 bits (from 513 on a block has sixteen of the call's rows): bit for bit, in any order, the same place several times."""
import pytest
import torch

import plain_cache8 as plain
from hipinfer_b200.kernels import ops
from test_gpu_cache8 import CODES, DEV, filled, ids, on_gpu, same

pytestmark = pytest.mark.gpu


def places(kind, n, ps, pages, g):
    if kind == "runs":                                              # portions of several requests, pages in no order
        order = torch.randperm(pages, generator=g).tolist()
        out, at = [], 5 % ps
        for page in order:
            out += [page * ps + i for i in range(at, ps)]
            at = (at + 3) % ps
        return out[:n]
    if kind == "any order":
        return torch.randperm(pages * ps, generator=g)[:n].tolist()
    if kind == "again":                                             # most places several times
        return torch.randint(0, max(1, pages * ps // 8), (n,), generator=g).tolist()
    out = torch.randint(-ps, (pages + 1) * ps, (n,), generator=g)   # "gaps": places outside of the cache, runs of rows that are not stored
    out[torch.arange(n) // 7 % 3 == 0] = -1
    return out.tolist()


@pytest.mark.parametrize("kind", ["runs", "any order", "again", "gaps"])
@pytest.mark.parametrize("rows", [512, 513, 1531])
@pytest.mark.parametrize("heads, ps, D", [(8, 16, 64), (2, 32, 128), (5, 64, 128), (3, 24, 40), (1, 4, 7)])
@pytest.mark.parametrize("codes, dtype", [(torch.int8, torch.bfloat16), (torch.float8_e4m3fn, torch.float32), (torch.int8, torch.float32)], ids=ids)
def test_many_rows(kind, rows, heads, ps, D, codes, dtype):
    g = torch.Generator().manual_seed(rows + D)
    pages = 3 * -(-rows // ps) + 3
    cache, slots = filled(pages, heads, ps, D, codes, 4), places(kind, rows, ps, pages, g)
    assert len(slots) == rows
    k, v = (torch.randn(rows, heads * D, generator=g).mul_(torch.rand(rows, 1, generator=g) * 4).to(dtype) for _ in range(2))
    got = on_gpu(cache)
    ops.store_cache8(k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV), got)
    for x, c, s, gc, gs in ((k, cache[0], cache[2], got.k, got.k_scale), (v, cache[1], cache[3], got.v, got.v_scale)):
        wc, ws = plain.store(x, slots, c, s)
        assert same(gs, ws) and same(gc, wc)
