"""A kernel's attributes belong to a device, read off the sources of what attends over a cache in 8 bits (no GPU): they are set once on each device, not once
in a process, or the second GPU that a process uses refuses the launch."""
import os
import re

import pytest

from hipinfer_b200.kernels import library


@pytest.mark.parametrize("name", ["attention_prefill_tc.cu"] + [f for f in library.LIBRARIES["cache8"] if "cudaFuncSetAttribute" in open(os.path.join(library.CSRC, f)).read()])
def test_attributes_are_set_on_every_device(name):
    with open(os.path.join(library.CSRC, name)) as f:
        text = f.read()
    assert not re.search(r"static bool configured\s*=", text)
    blocks = text.split("static bool configured[64]")[1:]
    assert blocks and all("cudaGetDevice(" in b[:400] and "cudaFuncSetAttribute(" in b[:900] for b in blocks)
    assert text.count("cudaFuncSetAttribute(") == sum(b[:900].count("cudaFuncSetAttribute(") for b in blocks)
