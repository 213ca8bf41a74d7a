"""A kernel's attributes belong to a device, read off the sources of the `drafts` library (no GPU): they are set once on each device, not once
in a process, or the second GPU that a process uses refuses the launch."""
import os
import re

import pytest

from hipinfer_b200.kernels import library

SETTING = [f for f in library.LIBRARIES["drafts"] if "cudaFuncSetAttribute" in open(os.path.join(library.CSRC, f)).read()]


@pytest.mark.parametrize("name", SETTING)
def test_attributes_are_set_on_every_device(name):
    with open(os.path.join(library.CSRC, name)) as f:
        text = f.read()
    assert not re.search(r"static bool configured\s*=", text)
    assert len(re.findall(r"static bool configured\[\d+\]", text)) == text.count("cudaFuncSetAttribute(")
    assert text.count("cudaGetDevice(") == text.count("cudaFuncSetAttribute(")
