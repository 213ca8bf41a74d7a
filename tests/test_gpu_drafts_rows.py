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
