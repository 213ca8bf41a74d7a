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
