"""The kernels of the decay attention that give up wait for what they have in flight, and say that they gave up."""
import os

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
with open(os.path.join(HERE, "..", "bi-mamba2_b200", "csrc", "uni_tc.cuh")) as f:
    BEFORE, *KERNELS = f.read().split("__global__")
LOADING = [k for k in KERNELS if "tma_load" in k]


def test_there_are_such_kernels():
    assert len(LOADING) == 3


@pytest.mark.parametrize("kernel", LOADING, ids=["states", "chunks", "grads"])
def test_a_kernel_waits_for_its_loads_and_matrix_products(kernel):
    """It cannot be made to happen on a GPU without breaking the kernel: read from its text."""
    end = kernel.index("leave nothing in flight")
    left = kernel[end:]
    assert "drain_mmas(" in left and "atomicExch(a.status" in kernel
    # every barrier that a load is asked to signal is drained
    barriers = {part.split(");")[0].rsplit("&", 1)[1].split("[")[0].strip() for part in kernel.split("tma_load")[1:]}
    for bar in barriers:
        assert bar.split(".")[-1] in left, bar
