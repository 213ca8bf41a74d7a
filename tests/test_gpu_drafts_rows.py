"""Attention over shared prefixes: rows of q, and values behind a row, of kinds that the other tests do not have."""
import math

import pytest
import torch

from hipinfer_b200.kernels import ops
from test_gpu_drafts import BF16, DEV, F32, bound, case, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("stride", [0, 64, 256 - 16])
def test_rows_of_q_that_lie_over_each_other(stride, D, dtype):
    """One row for all (expand), and rows that begin inside of the one before."""
    q, c, groups, Hq, Hkv, ps = [2, 1, 1], [300, 290, 295], [(0, 3, 280)], 4, 2, 16
    x, k, v, table, scale = case(q, c, groups, Hq, Hkv, D, ps, dtype)
    x = x.contiguous().view(-1).as_strided((4, Hq * D), (stride, 1))
    plan = ops.SharedPlan(q, c, groups, Hq, Hkv, D, ps, dtype, DEV)
    got = ops.attention_shared(x, k, v, table, plan)
    out, mag, most, keys = oracle(x, k, v, table, q, c, groups, Hq, Hkv, D, ps, scale)
    assert ((got.double() - out).abs() <= bound(dtype, out, mag, most, keys, D)).all()
    ops.check_device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("stride", [0, 1, 8, 5000])
def test_one_row_of_any_stride(stride, dtype):
    x, k, v, table, scale = case([1], [200], [], 4, 2, 64, 16, dtype)
    plan = ops.SharedPlan([1], [200], [], 4, 2, 64, 16, dtype, DEV)
    want = ops.attention_shared(x.contiguous(), k, v, table, plan)
    got = ops.attention_shared(x.contiguous().as_strided((1, 256), (stride, 1)), k, v, table, plan)
    out, mag, most, keys = oracle(x, k, v, table, [1], [200], [], 4, 2, 64, 16, scale)
    assert ((got.double() - out).abs() <= bound(dtype, out, mag, most, keys, 64)).all()
    if stride % 8 == 0:
        assert torch.equal(got, want)


PORTIONS = [
    ("one item of few rows", [20, 1], [130, 133], [(0, 2, 128)], 4, 2),
    ("both chains with the same rows", [31], [0], [], 8, 2),
    ("a chain with half of the rows", [60, 5], [97, 150], [(0, 2, 90)], 8, 2),
    ("several items", [300, 17], [70, 64], [(0, 2, 64)], 8, 2),
    ("a head of its own", [200], [333], [], 2, 2),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name,q,c,groups,Hq,Hkv", PORTIONS, ids=[x[0] for x in PORTIONS])
def test_a_long_portions_rows_must_not_see_a_later_one(name, q, c, groups, Hq, Hkv, D, dtype):
    """Keys and values of a portion that are not finite stay out of the rows before them, to the bit, and are in those from them on."""
    ps = 16
    x, k, v, table, scale = case(q, c, groups, Hq, Hkv, D, ps, dtype)
    plan = ops.SharedPlan(q, c, groups, Hq, Hkv, D, ps, dtype, DEV)
    clean = ops.attention_shared(x, k, v, table, plan)
    at = torch.arange(sum(q), device=DEV)
    for i in sorted({0, 1, 7, 15, 16, q[0] // 2, q[0] - 2, q[0] - 1} | set(range(3, q[0], 29))):
        for bad, keys in ((math.nan, True), (math.inf, False), (-math.inf, False), (math.nan, False)):
            k2, v2 = k.clone(), v.clone()
            page, place = int(table[0, (c[0] + i) // ps]), (c[0] + i) % ps
            column = (37 * i) % D                  # one element of one kv head, or all of the token's
            (v2[page, :, place] if keys else v2[page, i % Hkv, place, column:column + 1]).fill_(bad)
            if keys:
                k2[page, :, place] = bad
            got = ops.attention_shared(x, k2, v2, table, plan).view(-1, Hkv, Hq // Hkv, D)
            sees = ((at >= i) & (at < q[0]))[:, None].expand(-1, Hkv) & (torch.ones(Hkv, dtype=torch.bool, device=DEV) if keys
                                                                        else torch.arange(Hkv, device=DEV) == i % Hkv)
            assert torch.equal(got[~sees], clean.view_as(got)[~sees]), (i, bad)
            assert not torch.isfinite(got[sees]).all(-1).any(), (i, bad)
            assert keys or not torch.isfinite(got[sees][..., column]).any()
    ops.check_device_status()


@pytest.mark.parametrize("D", [64, 128])
def test_many_places_of_a_long_portion_that_are_not_finite(D):
    """Places all over a portion of many rows and heads, in a call whose CTAs have several items each: which rows are not finite is a matter of the
    first such place, in every one of several calls."""
    q, c, Hq, Hkv, ps = [1500, 700], [40, 900], 8, 2, 16
    x, k, v, table, scale = case(q, c, [], Hq, Hkv, D, ps, BF16)
    plan = ops.SharedPlan(q, c, [], Hq, Hkv, D, ps, BF16, DEV)
    clean = ops.attention_shared(x, k, v, table, plan)
    first = (400, 333)
    gen = torch.Generator(device=DEV).manual_seed(2)
    for r in (0, 1):
        for i in [first[r]] + sorted(torch.randint(first[r], q[r], (20,), generator=gen, device=DEV).tolist()):
            v[int(table[r, (c[r] + i) // ps]), :, (c[r] + i) % ps, i % D] = math.inf
    hit = torch.cat([torch.arange(n, device=DEV) >= f for n, f in zip(q, first)])
    for _ in range(10):
        got = ops.attention_shared(x, k, v, table, plan)
        assert torch.equal(got[~hit], clean[~hit])
        assert not torch.isfinite(got[hit].view(-1, Hq, D)).all(-1).any()
    ops.check_device_status()
