"""C ABI of the decay attention: `saved` is written by the forward pass whenever the backward pass of the same arguments reads it."""
import ctypes

import pytest

from ssd import _cabi

ALIGN = -4                                            # BISSD_ERR_ALIGN


def args(dtype=1, o=4096, q=4096, saved=4096, kdim=64, scale=0.125):
    a = _cabi.DecayArgs(batch=1, seqlen=200, nheads=4, nkheads=2, kdim=kdim, vdim=64, dtype=dtype, g_dtype=dtype, scale=scale)
    for name, heads, width in (("q", 2, kdim), ("k", 2, kdim), ("v", 4, 64), ("g", 4, 1), ("dout", 4, 64)):
        setattr(a, name, _cabi.Tensor(4096, 200 * heads * width, heads * width, width))
    a.q.ptr = q
    a.o, a.saved = o, saved
    return a


def forward(a):
    f = ctypes.c_size_t()
    assert _cabi.load().bissd_decay_workspace_bytes(ctypes.byref(a), ctypes.byref(f), None) == 0
    # one byte too few where nothing else is refused first: no launch is reached on any machine
    return lambda less: _cabi.load().bissd_decay_forward(ctypes.byref(a), 4096, f.value - less, None)


@pytest.mark.parametrize("dtype", [1, 2], ids=["bf16", "fp16"])
@pytest.mark.parametrize("off", [2, 4, 8])
def test_an_output_that_the_tensor_cores_cannot_write_is_refused_beside_saved(dtype, off):
    """Such a pass would run on the CUDA cores, which leave `saved` as it is, and the backward pass on the tensor cores, which read it."""
    assert forward(args(dtype, o=4096 + off))(0) == ALIGN


def test_what_is_not_refused():
    """Without `saved`; and where both passes run on CUDA cores, which neither write nor read it."""
    workspace = -5                                    # BISSD_ERR_WORKSPACE, looked at first
    for a in (args(o=4098, saved=None), args(o=4098, q=4098), args(o=4100, dtype=0), args(o=4098, scale=-1.0), args(o=4098, kdim=130), args()):
        assert forward(a)(256) == workspace
    lib = _cabi.load()
    n = ctypes.c_size_t()
    assert lib.bissd_decay_saved_bytes(ctypes.byref(args()), ctypes.byref(n)) == 0 and n.value > 0
