"""Requests that share pages (forked, cut back, freed in any order), the prefixes that neighbours of a step have in common, and
drafts looked up in a request's own tokens. No GPU."""
import random

import numpy as np
import pytest

from hipinfer_b200.cache import CacheError, CacheGroupSpec, CacheManager, OutOfStateSlots
from hipinfer_b200.engine.batch import shared_prefixes
from hipinfer_b200.engine.samples import DraftLookup

FULL = CacheGroupSpec("full", "full", n_layers=2, kv_heads=2, head_dim=16)
WIN = CacheGroupSpec("win", "window", n_layers=1, kv_heads=1, head_dim=32, window=40)


def test_a_fork_holds_the_whole_pages_and_goes_on_in_its_own():
    cm = CacheManager([FULL], 16, 12, 4)
    cm.add_request("a")
    cm.append("a", 37)
    assert cm.fork("a", "b").length == 32 and cm.block_table("b", 0) == [0, 1]
    assert cm.free_pages() == [9] and cm.pages_needed("b", 5) == [1]
    assert cm.append("b", 5) == [[48, 49, 50, 51, 52]] and cm.block_table("b", 0) == [0, 1, 3]
    cm.check()
    cm.free_request("a")                        # page 2 was its own, pages 0 and 1 stay with b
    assert cm.free_pages() == [9] and cm.pools[0].held() == [0, 1, 3]
    cm.check()
    cm.free_request("b")
    assert cm.free_pages() == [12]
    cm.check()


def test_fork_of_little_and_misuse():
    cm = CacheManager([FULL], 16, 4, 2)
    cm.add_request("a")
    assert cm.fork("a", "b").length == 0
    with pytest.raises(CacheError):
        cm.fork("a", "b")
    with pytest.raises(CacheError):
        cm.fork("x", "c")
    with pytest.raises(OutOfStateSlots):
        cm.fork("a", "c")
    cm.check()
    pool = cm.pools[0]
    with pytest.raises(CacheError):
        pool.share(0)
    p = pool.alloc()
    pool.share(p)
    pool.release(p)
    assert pool.free_count == 3
    pool.release(p)
    assert pool.free_count == 4
    with pytest.raises(CacheError):
        pool.release(p)


def test_truncate_gives_back_pages_and_refuses_shared_ones():
    cm = CacheManager([FULL], 16, 8, 3)
    cm.add_request("a")
    cm.append("a", 50)
    assert cm.truncate("a", 50) == 0 and cm.truncate("a", 33) == 1 and cm.block_table("a", 0) == [0, 1, 2]
    assert cm.append("a", 2) == [[33, 34]]
    cm.fork("a", "b")
    for length in (31, 17, 1, 36, -1):
        with pytest.raises(CacheError):
            cm.truncate("a", length)
        with pytest.raises(CacheError):
            cm.truncate("b", length)
    assert cm.get("a").length == 35 and cm.get("b").length == 32
    assert cm.truncate("b", 16) == 1 and cm.pools[0].holders(1) == 1          # at a page's end nothing shared is written
    assert cm.append("b", 3) == [[48, 49, 50]]
    assert cm.truncate("a", 30) == 1                                         # page 1 is a's alone now
    cm.check()
    cm.free_request("a")
    cm.free_request("b")
    assert cm.free_pages() == [8]


def test_truncate_behind_a_window():
    cm = CacheManager([FULL, WIN], 16, 8, 2)
    cm.add_request("a")
    cm.append("a", 60)
    cm.release_behind_window("a")               # the next query at 60 reads 21..: page 0 of the window group is gone
    assert cm.truncate("a", 57) == 0
    with pytest.raises(CacheError):
        cm.truncate("a", 54)                    # the query at 54 would read 15
    assert cm.get("a").length == 57
    with pytest.raises(CacheError):
        cm.fork("a", "b")                       # b would go on at 48 and read 9..
    assert not cm.has_request("b")
    cm.append("a", 7)
    cm.release_behind_window("a")
    assert cm.fork("a", "b").length == 64 and cm.block_table("b", 1)[0] == -1
    cm.check()


def test_forks_in_random_order_lose_no_page():
    rnd = random.Random(3)
    cm = CacheManager([FULL, WIN], 16, [60, 60], 12)
    live, n = [], 0
    for _ in range(3000):
        do = rnd.random()
        if do < 0.15 and len(live) < 12:
            cm.add_request(n)
            live.append(n)
            n += 1
        elif do < 0.35 and live and len(live) < 12:
            try:
                cm.fork(rnd.choice(live), n)
                live.append(n)
                n += 1
            except CacheError:
                pass
        elif do < 0.7 and live:
            rid, k = rnd.choice(live), rnd.randint(1, 40)
            if cm.can_append(rid, k):
                for table, slots in zip(cm.get(rid).tables, cm.append(rid, k)):
                    for s in slots:
                        assert s // 16 in table
                # what was written to is nobody else's
                for g, pool in enumerate(cm.pools):
                    rc = cm.get(rid)
                    for page in rc.tables[g][(rc.length - k) // 16:]:
                        assert pool.holders(page) == 1
                cm.release_behind_window(rid)
        elif do < 0.85 and live:
            rid = rnd.choice(live)
            try:
                cm.truncate(rid, rnd.randint(0, cm.get(rid).length))
            except CacheError:
                pass
        elif live:
            cm.free_request(live.pop(rnd.randrange(len(live))))
        cm.check()
    for rid in live:
        cm.free_request(rid)
    assert cm.free_pages() == [60, 60]


@pytest.mark.parametrize("tables, ctx, want", [
    ([], [], []),
    ([[0, 1]], [32], []),
    ([[0, 1, 2], [0, 1, 3]], [40, 40], [(0, 2, 32)]),
    ([[0, 1, 2], [0, 1, 2]], [40, 40], [(0, 2, 32)]),                     # (a page not filled yet is not shared)
    ([[0, 1, 2], [0, 1, 3]], [40, 16], [(0, 2, 16)]),
    ([[0, 1, 2], [0, 1, 3]], [40, 15], []),
    ([[0, 1], [2, 3], [2, 4], [5]], [30, 20, 20, 3], [(1, 2, 16)]),
    ([[0, 1], [0, 2], [3, 4], [3, 5]], [16, 16, 16, 16], [(0, 2, 16), (2, 2, 16)]),
    ([[0, 1, 2, 3], [0, 1, 2, 4], [0, 5]], [63, 63, 31], [(0, 2, 48)]),   # the third would cost two pages to win one
    ([[0, 1, 3], [0, 1, 4], [0, 1, 5], [0, 6]], [40, 40, 40, 40], [(0, 3, 32)]),
    ([[0, 1, 3], [0, 1, 4], [0, 5], [0, 6]], [40, 40, 40, 40], [(0, 2, 32), (2, 2, 16)]),
    ([[-1, 1], [-1, 1]], [40, 40], []),
    ([[], []], [0, 0], []),
])
def test_shared_prefixes(tables, ctx, want):
    assert shared_prefixes([np.asarray(t, dtype=np.int32) for t in tables], ctx, 16) == want


def test_lookup_proposes_what_followed_the_longest_tail():
    text = DraftLookup([1, 2, 3, 4, 9, 2, 3, 5, 7, 2, 3])
    assert text.propose(3) == [5, 7, 2]                     # the latest of two occurrences of (2, 3)
    assert DraftLookup([1, 2, 3, 4, 9, 2, 3, 5, 1, 2, 3]).propose(2) == [4, 9]      # three tokens count more than two
    assert DraftLookup([4, 4]).propose(4) == [4]
    assert DraftLookup([1, 2, 3]).propose(4) == [] and DraftLookup().propose(4) == [] and text.propose(0) == []


def test_lookup_shares_the_prompt_and_is_the_plain_search():
    rnd = random.Random(5)
    for _ in range(200):
        prompt = [rnd.randrange(4) for _ in range(rnd.randrange(0, 30))]
        base = DraftLookup(prompt)
        a, b = DraftLookup(base=base), DraftLookup(base=base)
        for text in (a, b):
            text.extend(rnd.randrange(4) for _ in range(rnd.randrange(0, 20)))
            want = []
            for m in (3, 2, 1):
                at = [i for i in range(m, len(text.tokens)) if text.tokens[i - m:i] == text.tokens[len(text.tokens) - m:]]
                if at and m <= len(text.tokens):
                    want = text.tokens[at[-1]:at[-1] + 5]
                    break
            assert text.propose(5) == want
        assert base.tokens == prompt
