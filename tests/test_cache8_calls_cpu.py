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
