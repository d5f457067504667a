"""A wait of `decay_states` that runs out is reported whichever warp's it is, and nothing is left in flight: read from the kernel's text,
since it cannot be made to happen on a GPU without breaking the kernel.

The warps play roles and meet at mbarriers alone; one that gives up leaves its wait's number in `sh.fail`.  So the flag is looked at
behind a barrier of the whole block, when every role has ended, and before tensor memory is freed."""
import os
import re

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
with open(os.path.join(HERE, "..", "bi-mamba2_b200", "csrc", "uni_tc.cuh")) as f:
    STATES = next(k for k in f.read().split("__global__") if re.search(r"\bdecay_states\(StatesParams", k))
STATES = STATES[:STATES.index("// ---- the outputs")]
ROLES = STATES.index("if (warp == 8) {")


def test_the_report_follows_a_barrier_of_the_block():
    report = [m.start() for m in re.finditer(r"atomicExch\(a\.status, kErrDecay \+ 0x10", STATES)]
    assert len(report) == 1
    between = STATES[ROLES:report[0]]
    assert "__syncthreads();" in between
    behind = between[between.rindex("__syncthreads();"):]
    assert re.search(r"if \(sh\.fail\) \{", behind) and not re.search(r"\bok\b", behind)   # nothing but the flag decides


@pytest.mark.parametrize("call", [r"drain_mmas\(&sh\.unused\)", r"drain_loads\(sh\.full, EXACT \? 1 : 2, sh\.loads\)",
                                  r"drain_loads\(sh\.full_v, 2, sh\.loads_v\)"])
def test_what_is_in_flight_is_waited_for_before_memory_is_freed(call):
    at = re.search(call, STATES).start()
    free = STATES.index("tmem_dealloc(")
    flag = STATES.index("if (sh.fail) {")
    assert flag < at < free and "__syncthreads();" in STATES[at:free]


def test_the_role_that_loads_leaves_its_counts():
    """However it ends."""
    role = STATES[ROLES:STATES.index("} else if (warp == 9) {")]
    assert re.search(r"\n        if \(lane == 0\) \{\n            sh\.loads = loads;\n            sh\.loads_v = loads_v;\n        \}\n    $", role)
