"""Attention over a cache in 8 bits where one key takes nearly all of a row's weight and has no value, and the result is what thousands of keys with tiny weights give.

float32 rows: a weight goes to the tensor cores in two f16 parts, the second times 2^12: the first is off by 2^-12 of the weight, or by 2^-25 where that is more, the second by as much of that again (or
2^-37); the largest weight of a warp's keys is 2^2 or more. A weight that is 2^-n of the largest is thus off by max(2^-23, 2^(n - 39)) of itself: 2^-15 for n = 24, of the first key's warp's keys alone (a
quarter at most, four warps having keys), of either sign. Its exponential is off by 2^-21, a score's 32-bit sum, of up to 2^4, by 2^-20. A row's error is below 2^-17 of sum_j p_j rms(v_j).
bfloat16 rows: one f16 part, off by 2^(n - 27) of a weight for n above 16: for n = 20 a quarter of the weights by 2^-7 at most, of either sign, which stays within tests/cache8_bounds.py."""
import pytest
import torch

import cache8_bounds as bounds
from hipinfer_b200.kernels import ops
from test_gpu_cache8 import CODES, DEV, filled, ids, on_gpu, step

pytestmark = pytest.mark.gpu


def sink(held, n, heads, kv_heads, D, codes, dtype, log2_first, seed=0):
    """Rows whose first key has 2^log2_first times the weight of a key whose score is 0; the others' scores are small."""
    batch, tables, pages = step([held], [n], 16)
    k, v, ks, vs = filled(pages, kv_heads, 16, D, codes, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(n, heads, D, generator=g)
    q[..., 0] = 8.0                                                 # the first dimension belongs to the first key alone
    k = (k.float() * 0.25).round() if codes == torch.int8 else k.float() * 0.25
    k[..., 0] = 0
    page = tables[0][0]
    k[page, :, 0] = 0
    k[page, :, 0, 0] = 100
    v = v.float()
    v[page, :, 0] = 0
    ks[page, :, 0] = log2_first * 0.6931471805599453 / (8.0 * 100 * D ** -0.5)
    return batch, tables, q.reshape(n, -1).to(dtype), (k.to(codes), v.to(codes), ks, vs)


@pytest.mark.parametrize("log2_first", [0, 8, 16, 24])
@pytest.mark.parametrize("held, n", [(5000, 1), (700, 1), (1500, 5)])
@pytest.mark.parametrize("heads, kv_heads, D", [(8, 2, 64), (4, 1, 128), (2, 2, 80)])
@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_in_float32(log2_first, held, n, heads, kv_heads, D, codes):
    batch, tables, q, cache = sink(held, n, heads, kv_heads, D, codes, torch.float32, log2_first)
    want, _, sums = bounds.attend(q, cache, tables, [held], [n], heads, sums=True)
    got = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, heads).double().cpu().view(want.shape)
    assert float(((got - want).square().mean(-1).sqrt() / sums).max()) <= 2.0 ** -17


@pytest.mark.parametrize("log2_first", [0, 8, 16, 20])
@pytest.mark.parametrize("held, n", [(5000, 1), (700, 1), (1500, 5)])
@pytest.mark.parametrize("heads, kv_heads, D", [(8, 2, 64), (4, 1, 128), (2, 2, 80)])
@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_in_bfloat16(log2_first, held, n, heads, kv_heads, D, codes):
    batch, tables, q, cache = sink(held, n, heads, kv_heads, D, codes, torch.bfloat16, log2_first)
    want, bound = bounds.attend(q, cache, tables, [held], [n], heads)
    assert bounds.beyond(ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, heads), want, bound) <= 1
