"""CPU: where the kernels whose warps wait for themselves hand a wait that ran out to the status word.

One thread reads the CTA's word.  A wait of another warp may run out after that thread's own work is done, so a barrier of the whole CTA has to lie between the last wait and
the read.  Such a wait cannot be made to run out in a test without a stalled copy, so this reads the sources."""
import glob
import os
import re

import pytest

from .conftest import PKG_NAME, ROOT

READ = re.compile(r"if \(threadIdx\.x == 0 && \*?abort_(?:flag|word) != 0\)")
BARRIER = re.compile(r"__syncthreads\(\);|cluster_sync_all\(\);")


def reads():
    for path in sorted(glob.glob(os.path.join(ROOT, PKG_NAME, "csrc", "*.cu*"))):
        lines = open(path).read().split("\n")
        for i, line in enumerate(lines):
            if READ.search(line):
                yield os.path.basename(path), i + 1, lines[:i]


@pytest.mark.parametrize("path,line,before", [pytest.param(*r, id=f"{r[0]}:{r[1]}") for r in reads()])
def test_a_barrier_comes_before(path, line, before):
    for text in reversed(before):
        if BARRIER.search(text):
            return
        assert "_wait(" not in text and "bulk_wait_all" not in text, f"{path}: nothing holds thread 0 between this wait and line {line}: {text.strip()}"
    pytest.fail("no barrier")


def test_there_are_such_reads():
    assert {r[0] for r in reads()} >= {"lora.cu", "norm.cu"}
