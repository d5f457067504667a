"""What one warp of `decay_grads` reads while the others go on must not be written again before it has: read from the kernel's text, since
on a GPU only time would show it.

A warp sums dg at the end of a head.  An array that the warps write in one stretch between two of the block's barriers may be read
in the next stretch, or in a later one as long as a block's barrier still lies between the reader and the next tile's writes: stretches
of the tile loop, in turn, are the weighting (0), the products (1), and what follows the last barrier (2), behind which the next
tile's weighting (0) begins without a barrier."""
import os
import re

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
with open(os.path.join(HERE, "..", "bi-mamba2_b200", "csrc", "uni_tc.cuh")) as f:
    GRADS = next(k for k in f.read().split("__global__") if re.search(r"\bdecay_grads\(GradsParams", k))
LOOP = GRADS[GRADS.index("for (int i = 0; i < nv; ++i) {"):GRADS.index("    if (ok && warp == kIssue && elect_one()) from_chunk();")]
TAIL = LOOP.index("ok = __syncthreads_and(ok);")      # the barrier of packed tails alone, on top of the others
BARRIERS = [m.start() for m in re.finditer(r"__syncthreads_and\(ok\)", LOOP)][1:]


def stretches(pattern):
    return {sum(b < m.start() for b in BARRIERS) for m in re.finditer(pattern, LOOP)}


def test_the_loop_is_what_this_reads():
    assert len(BARRIERS) == 2 and TAIL < BARRIERS[0]


@pytest.mark.parametrize("array", ["rowsum", "colsum", "past", "future", "cross"])
def test_sums_are_read_before_they_are_written_again(array):
    writes = stretches(r"\b%s\[[^\]]+\](\[[^\]]+\])? = " % array)
    reads = stretches(r"&%s\[" % array) | (stretches(r"\? %s\[lane\]" % array) if array == "cross" else set())
    assert len(writes) == 1 and reads
    write = writes.pop()
    # the reader reaches the barrier in front of the next tile's write only once it has read, and reads behind the barrier that follows this write
    for read in reads:
        assert read > write and not (write == 0 and read == 2), (array, write, read)
