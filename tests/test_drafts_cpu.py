"""Plans of the shared-prefix attention (made on the host) and what the operators refuse, without a GPU."""
import os
import random

import numpy as np
import pytest
import torch

from hipinfer_b200.kernels import drafts, fast, library, ops

pytestmark = pytest.mark.skipif(not (os.path.isfile("/usr/local/cuda/bin/nvcc") or os.environ.get("HIPINFER_B200_NVCC")), reason="no nvcc")
NO_MASK, FRESH = 1 << 30, 16


def plan(q, c, groups, Hq=8, Hkv=2, tile=16, narrow=0, key_tile=64, ctas=10, item_cost=1.0, wide_cost=1.5, part_cost=1e-4):
    return drafts.plan_numbers(q, c, groups, Hq, Hkv, tile, narrow, key_tile, ctas, item_cost, wide_cost, part_cost)


def seen_keys(n, Hkv, G, narrow=0, key_tile=64):
    """Per (row, kv head): the (table, position) pairs that the plan has the row attend to, and the items by part row."""
    items = n[n[drafts._OFF_ITEMS]:][:8 * n[drafts._ITEMS]].reshape(-1, 8)
    ctas = n[n[drafts._OFF_CTAS]:][:n[drafts._CTAS] + 1]
    tokens = n[n[drafts._OFF_TOKENS]:][:12 * n[drafts._TOKENS]].reshape(-1, 12)
    assert ctas[0] == 0 and ctas[-1] == len(items) and (np.diff(ctas) > 0).all()
    owner = {}
    for table, token, count, pos, lo, hi, head, part in items.tolist():
        assert lo < hi and count > 0
        chains = 2 if count <= narrow else 1         # (two share a tile's keys)
        for ch in range(chains):
            for i in range(count):
                for g in range(G):
                    p = part + (ch * count + i) * G + g
                    assert p not in owner and 0 <= p < n[drafts._PARTS]
                    keys = [k for k in range(lo, hi) if k <= pos + i]
                    keys = [k for k in keys if k % key_tile // (key_tile // chains) == ch]
                    owner[p] = (token + i, head, g, table, keys)
    assert len(owner) == n[drafts._PARTS]
    out = []
    for t, (pb, pn, pr, ob, on, orows, table, first, fresh, *_) in enumerate(tokens.tolist()):
        for h in range(Hkv):
            for g in range(G):
                got = [(table, first + j) for j in range(fresh)]
                for base, count, rows in ((pb, pn, pr), (ob, on, orows)):
                    for k in range(count):
                        row, head, gg, tab, keys = owner.pop(base + (h * count + k) * rows + g)
                        assert (row, head, gg) == (t, h, g)
                        got += [(tab, key) for key in keys]
                out.append((t, h, g, sorted(got, key=lambda x: x[1])))
    assert not owner
    return out


def check(q, c, groups, Hq, Hkv, **kw):
    n = plan(q, c, groups, Hq, Hkv, **kw)
    G = Hq // Hkv
    reads = {}
    for first, count, shared in groups:
        if sum(q[r] > 0 for r in range(first, first + count)) > 1:
            reads.update({r: (first, shared) for r in range(first, first + count)})
    rows = [(r, c[r] + i) for r in range(len(q)) for i in range(q[r])]
    assert n[drafts._TOKENS] == len(rows)
    for t, h, g, got in seen_keys(n, Hkv, G, kw.get("narrow", 0), kw.get("key_tile", 64)):
        r, pos = rows[t]
        via, shared = reads.get(r, (r, 0))
        assert got == [(via if k < shared else r, k) for k in range(pos + 1)]
    return n


@pytest.mark.parametrize("q,c,groups", [
    ([1, 1], [300, 310], [(0, 2, 256)]),
    ([1], [0], []),                                          # a first token, nothing in the cache
    ([1, 2, 3], [0, 0, 0], [(0, 3, 0)]),
    ([1, 1], [64, 64], [(0, 2, 64)]),                        # nothing of their own
    ([4, 0, 2], [130, 100, 129], [(0, 3, 100)]),             # one of the group brings no rows
    ([4, 0, 0], [130, 100, 129], [(0, 3, 100)]),             # one alone: nothing is shared
    ([3, 5, 1, 2], [200, 77, 300, 65], [(2, 2, 63), (0, 1, 50)]),
    ([17, 1, 40], [100, 90, 1], [(0, 2, 33)]),               # portions of more rows than the joining kernel adds
    ([16, 16], [31, 33], [(0, 2, 31)]),
    ([], [], []),
    ([0, 0], [5, 5], [(0, 2, 5)]),
])
@pytest.mark.parametrize("narrow", [0, 8])
def test_every_row_sees_its_keys_once(q, c, groups, narrow):
    check(q, c, groups, 8, 2, narrow=narrow)
    check(q, c, groups, 3, 3, narrow=narrow, tile=5, ctas=3)


def test_random_plans_cover_every_key():
    rng = random.Random(5)
    for _ in range(60):
        q, c, groups = [], [], []
        for _ in range(rng.randint(1, 3)):
            s, count = rng.choice([0, 1, 63, 64, 65, 200, 333]), rng.randint(1, 4)
            groups.append((len(q), count, s))
            for _ in range(count):
                q.append(rng.choice([0, 1, 1, 2, 5, 16, 17, 30]))
                c.append(s + rng.choice([0, 0, 1, 50, 130]))
        Hkv, G = rng.choice([(1, 1), (2, 3), (1, 8)])
        check(q, c, groups, Hkv * G, Hkv, tile=rng.choice([1, 4, 7]), narrow=rng.choice([0, 2]), ctas=rng.choice([1, 2, 37]), key_tile=rng.choice([64, 128]))


def test_the_work_is_spread_over_the_ctas():
    """Of a long prefix no CTA has much more than its share."""
    n = plan([1] * 8, [20480 + 16 * i for i in range(8)], [(0, 8, 20480)], 32, 8, tile=64, narrow=32, key_tile=128, ctas=148, part_cost=0.0)
    items = n[n[drafts._OFF_ITEMS]:][:8 * n[drafts._ITEMS]].reshape(-1, 8)
    ctas = n[n[drafts._OFF_CTAS]:][:n[drafts._CTAS] + 1]
    tiles = [sum(-(-(i[5]) // 128) - i[4] // 128 for i in items[a:b]) for a, b in zip(ctas, ctas[1:])]
    assert len(tiles) == 148 and max(tiles) <= 1.35 * sum(tiles) / 148 + 2


@pytest.mark.parametrize("q,c,groups,kw,words", [
    ([1, 1], [5, 5], [(0, 3, 2)], {}, "outside"),
    ([1, 1], [5, 5], [(-1, 2, 2)], {}, "outside"),
    ([1, 1], [5, 5], [(0, 2, -2)], {}, "outside"),
    ([1, 1], [5, 5], [(0, 2, 2), (1, 1, 2)], {}, "in groups"),
    ([1, 1], [5, 4], [(0, 2, 5)], {}, "holds 4"),
    ([-1, 1], [5, 4], [], {}, "-1 rows"),
    ([1], [-2], [], {}, "-2 tokens"),
    ([1], [1 << 30], [], {}, "request 0"),
    ([1, 2], [3], [], {}, "a request"),
    ([1], [3], [], dict(Hq=3, Hkv=2), "heads"),
])
def test_lengths_that_make_no_plan(q, c, groups, kw, words):
    with pytest.raises(ops.KernelError, match=words):
        plan(q, c, groups, **kw)


@pytest.mark.parametrize("kw,words", [(dict(n_heads=6, n_kv_heads=4), "multiple"), (dict(head_dim=257), "257"), (dict(head_dim=0), "heads of 0"),
                                      (dict(page_size=0), "pages of 0"), (dict(dtype=torch.float16), "float16")])
def test_sizes_that_a_plan_refuses(kw, words):
    args = dict(n_heads=8, n_kv_heads=2, head_dim=64, page_size=16, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(ops.KernelError, match=words):
        ops.SharedPlan([1], [4], [], **{**args, **kw})


@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_call", lambda lib, name, *a: calls.append(name))
    monkeypatch.setattr(ops, "_need_cuda", lambda *t: None)
    monkeypatch.setattr(library, "current_stream", lambda: 0)
    monkeypatch.setattr(fast, "_status_ptr", lambda: 0)
    return calls


def attend(plan_kw={}, **kw):
    p = ops.SharedPlan([1, 2], [20, 30], [(0, 2, 16)], 4, 2, 64, 16, torch.float32, "cpu")
    a = dict(q=torch.zeros(3, 256), k_cache=torch.zeros(5, 2, 16, 64), v_cache=torch.zeros(5, 2, 16, 64), block_table=torch.zeros(2, 2, dtype=torch.int32),
             plan=p)
    return ops.attention_shared(**{**a, **kw})


def test_attention_shared_takes_what_it_is_made_for(launches):
    assert attend().shape == (3, 256) and launches == ["hb_attention_shared"]
    assert attend(q=torch.zeros(3, 300)[:, :256]).is_contiguous()


@pytest.mark.parametrize("kw,words", [
    (dict(q=torch.zeros(4, 256)), "3 rows"), (dict(q=torch.zeros(3, 255)), "heads of 64"), (dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)), "float32"),
    (dict(q=torch.zeros(256, 3).t()), "strides"), (dict(k_cache=torch.zeros(5, 2, 16, 32)), "keys"), (dict(v_cache=torch.zeros(5, 2, 8, 64)), "values"),
    (dict(v_cache=torch.zeros(5, 16, 2, 64).transpose(1, 2)), "values"), (dict(k_cache=torch.zeros(6, 2, 16, 64)), "6 pages"),
    (dict(block_table=torch.zeros(2, 1, dtype=torch.int32)), "block table"), (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), "block table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), "block table"), (dict(out=torch.zeros(3, 128)), "out"),
    (dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), "out"),
])
def test_attention_shared_refuses(launches, kw, words):
    with pytest.raises(ops.KernelError, match=words):
        attend(**kw)
    assert not launches


def verify(**kw):
    a = dict(logits=torch.zeros(9, 11), start=torch.zeros(3, dtype=torch.int32), n_drafts=torch.zeros(3, dtype=torch.int32),
             drafts=torch.zeros(3, 2, dtype=torch.int32), temperature=torch.ones(3), uniform=torch.zeros(3, 2), noise=torch.ones(3, 11))
    return ops.verify_drafts(**{**a, **kw})


def test_verify_drafts_takes_what_it_is_made_for(launches):
    tokens, counts, logprobs = verify()
    assert tokens.shape == (3, 3) and counts.shape == (3,) and logprobs.shape == (3, 3) and launches == ["hb_verify_drafts"]
    verify(draft_probs=torch.zeros(3, 2, 11, dtype=torch.bfloat16), logits=torch.zeros(9, 16)[:, 2:13], noise=torch.ones(3, 16)[:, :11])
    none = torch.zeros(0, dtype=torch.int32)
    del launches[:]
    assert verify(start=none, n_drafts=none, drafts=torch.zeros(0, 2, dtype=torch.int32), temperature=torch.ones(0), uniform=torch.zeros(0, 2),
                  noise=torch.ones(0, 11))[0].shape == (0, 3) and not launches


@pytest.mark.parametrize("kw,words", [
    (dict(logits=torch.zeros(9, 11, dtype=torch.float16)), "float16"), (dict(logits=torch.zeros(11, 9).t()), "logits"), (dict(logits=torch.zeros(9)), "logits"),
    (dict(start=torch.zeros(2, dtype=torch.int32)), "start"), (dict(start=torch.zeros(3, dtype=torch.int64)), "start"),
    (dict(n_drafts=torch.zeros(3)), "n_drafts"), (dict(drafts=torch.zeros(3, 2, dtype=torch.int64)), "drafts"),
    (dict(drafts=torch.zeros(2, 3, dtype=torch.int32).t()), "drafts"), (dict(drafts=torch.zeros(3, 64, dtype=torch.int32)), "64 drafts"),
    (dict(temperature=torch.ones(3, dtype=torch.float64)), "temperature"), (dict(uniform=torch.zeros(3, 3)), "uniform"),
    (dict(noise=torch.ones(3, 10)), "noise"), (dict(noise=torch.ones(11, 3).t()), "noise"), (dict(noise=torch.ones(3, 11, dtype=torch.bfloat16)), "noise"),
    (dict(draft_probs=torch.zeros(3, 3, 11)), "draft_probs"), (dict(draft_probs=torch.zeros(3, 2, 11, dtype=torch.float16)), "draft_probs"),
    (dict(draft_probs=torch.zeros(3, 11, 2).transpose(1, 2)), "draft_probs"), (dict(logits=torch.zeros(9, 0), noise=torch.ones(3, 0)), "empty"),
])
def test_verify_drafts_refuses(launches, kw, words):
    with pytest.raises(ops.KernelError, match=words):
        verify(**kw)
    assert not launches


def test_the_operators_want_cuda_tensors():
    with pytest.raises(ops.KernelError, match="CUDA"):
        attend()
    with pytest.raises(ops.KernelError, match="CUDA"):
        verify()
