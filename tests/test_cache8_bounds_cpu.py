"""The bounds that tests of attention over a cache in 8 bits hold results to (cache8_bounds.py): results rounded as the kernels round pass them, results that lack a page or a
key, take another block's scale or see one key more or fewer do not."""
import pytest
import torch

import cache8_bounds as bounds
import plain_cache8 as plain

HEADS, KV, PS, D = 8, 2, 16, 64


def example(held, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-(h + n) // PS) for h, n in zip(held, rows))
    order, tables, at = torch.randperm(pages, generator=g).tolist(), [], 0
    for h, n in zip(held, rows):
        tables.append(order[at:at - (-(h + n) // PS)])
        at += len(tables[-1])
    cache = []
    for _ in range(2):
        cache.append(((torch.randn(pages, KV, PS, D, generator=g) * 40).clamp(-127, 127).round().to(torch.int8), torch.rand(pages, KV, 1, generator=g) * 0.04 + 0.01))
    (k, ks), (v, vs) = cache
    return torch.randn(sum(rows), HEADS * D, generator=g).to(torch.bfloat16), (k, v, ks, vs), tables


@pytest.mark.parametrize("held, rows", [([5000], [1]), ([1023, 64], [1, 1]), ([600], [300]), ([900, 333], [60, 1]), ([0], [40])])
def test_what_passes_and_what_does_not(held, rows):
    q, cache, tables = example(held, rows)
    want, bound = bounds.attend(q, cache, tables, held, rows, HEADS)
    off = lambda x: bounds.beyond(x, want, bound)
    assert off(want) == 0 and off(want.to(torch.bfloat16)) < 0.6
    # weights rounded to 16 bits, then the result
    lo = bounds.attend(q, cache, tables, held, rows, HEADS, weights=torch.bfloat16)[0].to(torch.bfloat16)
    assert off(lo) < 0.75
    # what a row is off by where something is lost
    assert off(want * 0.95) > 1
    k, v, ks, vs = cache
    for r, n in enumerate(len(t) for t in tables):
        for page in {0, n // 3, n - 2, n - 1} & set(range(n)):
            gone = [list(t) for t in tables]
            gone[r][page] = -1
            if rows[r] > 1 or page < n - 1 or (held[r] + rows[r]) % PS > 1:
                assert off(bounds.attend(q, cache, gone, held, rows, HEADS)[0]) > 1
    assert off(bounds.attend(q, (k, v, ks, vs.mean().expand_as(vs)), tables, held, rows, HEADS)[0]) > 1
    assert off(bounds.attend(q, (k, v, ks.roll(1, 0), vs), tables, held, rows, HEADS)[0]) > 1
    assert off(bounds.attend(q, (k, v, ks, vs.roll(1, 1)), tables, held, rows, HEADS)[0]) > 1


@pytest.mark.parametrize("window", [1, 2, 16, 100])
@pytest.mark.parametrize("change", [-1, 1])
def test_a_window_that_is_off_by_one(window, change):
    held, rows = [300, 37, 0], [60, 17, 130]
    q, cache, tables = example(held, rows)
    want, bound = bounds.attend(q, cache, tables, held, rows, HEADS, window, 0.2)
    if window + change:
        assert bounds.beyond(bounds.attend(q, cache, tables, held, rows, HEADS, window + change, 0.2)[0], want, bound) > 1


def test_the_64_bit_results_are_those_of_the_plain_statement():
    held, rows = [20, 33, 5], [3, 1, 16]
    q, cache, tables = example(held, rows)
    tables[1][1] = -1
    request = [r for r, n in enumerate(rows) for _ in range(n)]
    positions = [h + i for h, n in zip(held, rows) for i in range(n)]
    for window in (0, 9):
        a = bounds.attend(q, cache, tables, held, rows, HEADS, window)[0]
        b = torch.from_numpy(plain.attend(q, cache, tables, request, positions, HEADS, window, D ** -0.5)).view(a.shape)
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
