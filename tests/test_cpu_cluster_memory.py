"""The kernels that write another CTA's shared memory, read from their sources: each synchronises its cluster before the first such access (the
CTAs of a cluster are placed together, but memory of one that has not begun may not be touched) and again behind the last (nor that of
one that has ended)."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "gradients.c_b200", "csrc")
SYNC = re.compile(r"cluster_sync_all\(\)|barrier\.cluster\.wait")


def kernels(path):
    """(name, body) of every kernel of a source file, comments taken out."""
    text = re.sub(r"//[^\n]*", "", open(path).read())
    for m in re.finditer(r"__global__\s+void[^;{]*?(\w+)\s*\((?:[^()]|\([^()]*\))*\)\s*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


def access(body):
    """Places of the body at which a peer's shared memory is written or read (an address alone, formed by mapa, is none)."""
    return [m.start() for m in re.finditer(r"\b(?:st|ld|red|atom)[.\w]*\.shared::cluster", body)]


FOUND = [(os.path.basename(f), name, body) for f in sorted(glob.glob(os.path.join(CSRC, "*.cu"))) for name, body in kernels(f) if access(body)]


def test_the_kernels_are_found():
    assert {name for _, name, _ in FOUND} >= {"ns_single_kernel", "ns_tile_kernel"}


@pytest.mark.parametrize("file,name,body", FOUND, ids=[f"{f}:{n}" for f, n, _ in FOUND])
def test_cluster_runs_before_and_after_its_memory_is_shared(file, name, body):
    syncs, places = [m.start() for m in SYNC.finditer(body)], access(body)
    assert any(s < places[0] for s in syncs), f"{file}: {name} touches a peer's memory before it is known to run"
    assert any(s > places[-1] for s in syncs), f"{file}: {name} may end while its memory is being written"
