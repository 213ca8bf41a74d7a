"""What a kernel of a thread-block cluster may do before a barrier of the cluster, read off the sources (no GPU): shared memory of another
block may be touched only when that block is known to have started, so the first access to it, in the order of the source, has a wait at
a barrier of the cluster ahead of it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipinfer_b200", "csrc")
# (a bulk copy's or a commit's destination is called shared::cluster too; without a mapped address it is the block's own)
REMOTE = re.compile(r"\b(?:st|ld|atom|red)\.[a-z.]*shared::cluster|hb_mbar_arrive_remote\(|hb_mapa\(")
WAIT = re.compile(r"barrier\.cluster\.wait|\bhb_cluster_sync\(|\bcluster_sync\(|\bcluster_wait\(")


def kernels():
    for name in sorted(f for f in os.listdir(CSRC) if f.endswith(".cu")):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__", text):
            at = text.index("{", m.end())
            semicolon = text.find(";", m.end())
            if 0 <= semicolon < at:            # a declaration
                continue
            depth, end = 1, at + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            kernel = re.search(r"(\w+)\s*\($|(\w+)\s*\(", re.sub(r"__launch_bounds__\s*\([^)]*\)", "", text[m.end():at]))
            yield name, next(g for g in kernel.groups() if g), text[at:end]


REACHING = [(name, kernel, body) for name, kernel, body in kernels() if REMOTE.search(body)]


def test_there_are_such_kernels():
    assert {"verify_pick_kernel", "attn_masked_heads_kernel"} <= {k for _, k, _ in REACHING}


@pytest.mark.parametrize("name, kernel, body", REACHING, ids=[f"{n}:{k}" for n, k, _ in REACHING])
def test_a_neighbour_has_started_before_its_shared_memory_is_touched(name, kernel, body):
    wait = WAIT.search(body)
    assert wait and wait.start() < REMOTE.search(body).start()
