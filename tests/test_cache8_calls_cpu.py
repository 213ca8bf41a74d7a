"""Calls of the operators of a cache in 8 bits, on the host: what a failed one says, what a GPU has no room for, how a step is split."""
import functools

import pytest

from hipinfer_b200.kernels import cache8, ops


def test_a_failed_call_s_words_are_those_of_its_library(monkeypatch):
    from types import SimpleNamespace

    from hipinfer_b200.kernels import library

    words = {"cache8": b"hb_cache8_store: sizes", "fast": b"hb_flash_prefill_tc: heads"}
    monkeypatch.setattr(library, "load", lambda name: SimpleNamespace(hb_last_error=lambda: words[name]))
    before = library.launches[0]
    for result, name in ((1, "cache8"), (-1, "fast")):
        with pytest.raises(ops.KernelError, match=words[name].decode()):
            cache8._done(result, 2)
    assert library.launches[0] == before and cache8._done(0, 1) == 0 and library.launches[0] == before + 1
    library.launches[0] = before


def test_a_gpu_without_room_for_large_clusters_takes_smaller_ones(monkeypatch):
    room = {16: 0, 15: 0, 14: 0, 13: 0, 12: 0, 11: 0, 10: 0, 9: 0}
    monkeypatch.setattr(ops, "_fn", lambda lib, name: lambda dt, code, head_dim, nt, ranks: room.get(ranks, 148 // ranks))
    cache8._clusters.cache_clear()
    try:
        clusters = functools.partial(cache8._clusters, 1, 2, 64, 1)
        assert clusters(16) == 0 and cache8._ranks(8, 8000, 8000.0, clusters) == 8
        room.update({r: 0 for r in range(2, 17)})
        cache8._clusters.cache_clear()
        assert cache8._ranks(8, 8000, 8000.0, clusters) == 1 and cache8._ranks(1, 100000, 100000.0, clusters) == 1
        room[2] = -1                                               # (an error of the call)
        cache8._clusters.cache_clear()
        with pytest.raises(ops.KernelError):
            clusters(2)
    finally:
        cache8._clusters.cache_clear()


def batch_of(held, rows, ps=16):
    from hipinfer_b200.engine.batch import StepEntry, build_step_batch

    tables = [[list(range(-(-(h + n) // ps)))] for h, n in zip(held, rows)]
    return build_step_batch([StepEntry(i, [0] * n) for i, n in enumerate(rows)], held, list(range(len(rows))), tables, [[[0] * n] for n in rows], 1, "cpu")


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("most", [1, 20, 40, 10 ** 6])
def test_portions_are_expanded_within_a_bound(monkeypatch, window, most):
    """Groups of neighbours of at most `most` pages, a single request's aside; every portion is in one group, whose tables name its pages alone."""
    cache = ops.new_cache8(4, 2, 16, 64, device="cpu")
    monkeypatch.setattr(cache8, "PORTION_BYTES", most * 4 * 2 * 16 * 64)
    held, rows = [0, 300, 40, 0, 7, 100, 160], [16, 30, 1, 333, 0, 20, 15]
    batch = batch_of(held, rows)
    groups, width = cache8._portion_groups(batch, cache, window, 16), batch.block_tables[0].shape[1]
    assert [g[0] for g in groups] == [0] + [g[1] for g in groups[:-1]] and groups[-1][1] == len(rows)
    seen = []
    for first, end in groups:
        index, places, base = cache8._pages_of_portions(batch, 16, width, window, 16, (first, end))
        there = [r for r in range(first, end) if rows[r] >= 16]
        assert there and (index.numel() <= most or len(there) == 1) and index.numel() == int((places >= 0).sum())
        assert [r for r in range(len(rows)) if (places[r] >= 0).any()] == there
        assert index.tolist() == [r * width + i for r in there for i in range(width) if places[r, i] >= 0]
        assert cache8._rows_of_group(batch, (first, end)).tolist() == [n if first <= r < end else 0 for r, n in enumerate(rows)]
        seen += index.tolist()
    assert sorted(seen) == sorted(cache8._pages_of_portions(batch, 16, width, window, 16)[0].tolist()) and (len(groups) == 1) == (len(seen) <= most)
