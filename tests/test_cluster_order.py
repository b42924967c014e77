"""Blocks of a cluster reach into one another's shared memory only once all of them are known to run: in every kernel that does, a
wait of the cluster's barrier comes before the first such address is made. Read from the sources, as a block that starts late
is nothing a test on the GPU could bring about."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thinksound-native_b200", "csrc")
TOUCHES = re.compile(r"\bdsmem_map\(|\bdsmem_ld4\(|\bmapa\.")
WAITS = re.compile(r"\bcluster_sync_all\(\)|\bcluster_wait\(\)")


def kernels():
    """(file, name, body without comments) of every kernel."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S))
        for m in re.finditer(r"__global__\b[^{;]*?(\w+)\s*\(const|__global__\b[^{;]*?(\w+)\s*\(", text):
            start = text.index("{", m.end())
            depth, end = 0, start
            for end in range(start, len(text)):
                depth += (text[end] == "{") - (text[end] == "}")
                if depth == 0:
                    break
            yield os.path.basename(path), m.group(1) or m.group(2), text[start:end]


FOUND = [(f, n, b) for f, n, b in kernels() if TOUCHES.search(b)]


def test_kernels_are_found():
    assert {"page_select.cu", "paged_tiles.cu", "diff_attn.cu", "gemm_2sm.cuh"} <= {f for f, _, _ in FOUND}


@pytest.mark.parametrize("file,name,body", FOUND, ids=[f"{f}-{n}" for f, n, _ in FOUND])
def test_a_wait_comes_first(file, name, body):
    wait = WAITS.search(body)
    assert wait and wait.start() < TOUCHES.search(body).start()
