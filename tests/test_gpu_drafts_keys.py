"""Attention over shared prefixes in bfloat16, over long ranges: values that make every missing key visible (a lost step of 64 keys moves a sum of
random values by less than the roundings may)."""
import pytest
import torch

from hipinfer_b200.kernels import ops
from test_gpu_drafts import BF16, DEV, bound, case, oracle

pytestmark = pytest.mark.gpu


def check(q, c, groups, Hq, Hkv, D, ps, v_of):
    x, k, v, table, scale = case(q, c, groups, Hq, Hkv, D, ps, BF16, seed=D)
    v.zero_()
    via = {r: (f, s) for f, n, s in groups for r in range(f, f + n) if sum(y > 0 for y in q[f:f + n]) > 1}
    for r, (n, held) in enumerate(zip(q, c)):
        first, shared = via.get(r, (r, 0))
        pos = torch.arange(held + n, device=DEV)
        page = torch.where(pos < shared, table[first].long()[pos // ps], table[r].long()[pos // ps])
        v[page, :, pos % ps] = v_of(pos).to(BF16)[:, None].expand(-1, Hkv, -1)
    got = ops.attention_shared(x, k, v, table, ops.SharedPlan(q, c, groups, Hq, Hkv, D, ps, BF16, DEV), scale=scale)
    out, mag, most, keys = oracle(x, k, v, table, q, c, groups, Hq, Hkv, D, ps, scale)
    assert ((got.double() - out).abs() <= bound(BF16, out, mag, most, keys, D)).all()
    ops.check_device_status()


LONG = [
    ("many chunks a row", [1, 2, 1], [20000, 20111, 20003], [(0, 3, 19999)], 8, 2),
    ("wide items", [4] * 24, [9000 + 50 * r for r in range(24)], [(0, 24, 8999)], 8, 2),
    ("many items a CTA", [1 + r % 4 for r in range(96)], [4000 + 13 * r for r in range(96)], [(0, 40, 3968), (40, 56, 777)], 32, 8),
    ("long portions", [300, 40, 17], [5000, 5100, 4990], [(0, 3, 4976)], 8, 2),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name,q,c,groups,Hq,Hkv", LONG, ids=[x[0] for x in LONG])
def test_every_block_of_keys_is_there(name, q, c, groups, Hq, Hkv, D):
    """Column d of the values is 1 in the blocks of 32 positions that are d modulo D: without one of a chain's steps two columns lose a tenth of what
    they sum, or more."""
    check(q, c, groups, Hq, Hkv, D, 16, lambda pos: torch.nn.functional.one_hot(pos // 32 % D, D))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name,q,c,groups,Hq,Hkv", LONG[:3], ids=[x[0] for x in LONG[:3]])
def test_every_key_is_there(name, q, c, groups, Hq, Hkv, D):
    """Single keys: a column has one of every D."""
    check(q, c, groups, Hq, Hkv, D, 16, lambda pos: torch.nn.functional.one_hot(pos % D, D))
