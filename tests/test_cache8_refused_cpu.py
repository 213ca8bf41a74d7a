"""Drafts that are taken back from a cache in 8 bits (no GPU): which blocks were touched, the pages that are put back, the rows that are stored again."""
import numpy as np
import pytest

from hipinfer_b200.engine.batch import StepEntry
from hipinfer_b200.engine.runner import _KeptStep


def kept(held, n, page_size=16, pages=50):
    tables = [[np.array([10 * r + i for i in range(-(-(h + m) // page_size))], dtype=np.int32)] for r, (h, m) in enumerate(zip(held, n))]
    slots = [[[int(t[0][p // page_size]) * page_size + p % page_size for p in range(h, h + m)]] for t, h, m in zip(tables, held, n)]
    return _KeptStep([StepEntry(f"r{r}", [0] * m) for r, m in enumerate(n)], held, tables, slots, page_size, [pages], []), slots


def test_what_is_put_back_and_stored_again():
    held, n = [5, 20, 16, 30, 7, 12], [4, 5, 5, 5, 1, 8]
    step, slots = kept(held, n)
    assert list(step.copies()) == [([0, 11, 31, 40, 50], [50, 51, 53, 54, 55])]             # (request 2 begins with a block)
    # all kept; two of five; one; back to a page's end; its only one is kept; over the block's end
    lengths = [9, 22, 17, 32, 8, 18]
    assert step.damaged(lengths) == [1, 2, 5]
    assert list(step.copies(lengths)) == [([11, 50], [51, 55])]
    want = [-1] * 4 + slots[1][0][:2] + [-1] * 3 + slots[2][0][:1] + [-1] * 4 + [-1] * 5 + [-1] + slots[5][0][:6] + [-1] * 2
    assert step.accepted(lengths)[0].tolist() == want and step.accepted(lengths)[0].dtype == np.int32


@pytest.mark.parametrize("page_size", [16, 32, 8, 24])
def test_every_length_is_put_back_where_a_kept_token_shares_a_block_with_one_that_is_not(page_size):
    block = lambda p: (p // page_size, p % page_size // 16)
    for held in range(0, 50):
        for n in (1, 2, 7, 20):
            step, slots = kept([held], [n], page_size)
            for length in range(0, held + n + 1):
                gone = {block(p) for p in range(max(held, length), held + n)}
                assert bool(step.damaged([length])) == any(block(p) in gone for p in range(length))
                stored = [s for s in step.accepted([length])[0].tolist() if s >= 0]
                assert stored == (slots[0][0][:max(0, length - held)] if step.damaged([length]) else [])


def test_requests_that_have_ended_are_left_alone():
    step, _ = kept([5, 21], [3, 3])
    assert step.damaged([0, 22]) == [1] and step.accepted([0, 22])[0].tolist()[:3] == [-1] * 3
