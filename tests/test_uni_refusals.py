"""What the causal decay attention, its single-token form and the norms around a block refuse, without a GPU."""
import ctypes

import pytest
import torch

from ssd import _cabi
from ssd.block_norm import block_norm
from ssd.uni.decay_attention import decay_attention, decay_attention_step


def inputs(b=1, L=6, h=4, hk=2, n=8, p=8, dtype=torch.float32):
    return [torch.zeros(b, L, hk, n, dtype=dtype), torch.zeros(b, L, hk, n, dtype=dtype), torch.zeros(b, L, h, p, dtype=dtype),
            torch.zeros(b, L, h, dtype=dtype)]


@pytest.mark.parametrize("change,says", [
    (lambda a: a.__setitem__(1, a[1][:, :5]), "q's shape"),
    (lambda a: a.__setitem__(2, torch.zeros(1, 6, 3, 8)), "multiple of q's"),
    (lambda a: a.__setitem__(2, torch.zeros(1, 7, 4, 8)), "batch and sequence"),
    (lambda a: a.__setitem__(2, torch.zeros(1, 6, 4, 257)), "1 to 256"),
    (lambda a: a.__setitem__(2, torch.zeros(1, 6, 4, 8, dtype=torch.bfloat16)), "one type"),
    (lambda a: a.__setitem__(3, torch.zeros(1, 6, 2)), "one value for each token"),
    (lambda a: a.__setitem__(3, torch.zeros(4, dtype=torch.bfloat16)), "g must be float32"),
    (lambda a: a.__setitem__(0, torch.zeros(6, 2, 8)), "dimensions"),
], ids=range(8))
def test_attention_refuses(change, says):
    a = inputs()
    change(a)
    with pytest.raises(ValueError, match=says):
        decay_attention(*a)


def test_attention_refuses_states_and_boundaries():
    a = inputs(b=2)
    for state in (torch.zeros(2, 4, 8, 9), torch.zeros(1, 4, 8, 8), torch.zeros(2, 4, 8, 8, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="initial_state"):
            decay_attention(*a, initial_state=state)
    with pytest.raises(ValueError, match="one row"):
        decay_attention(*a, cu_seqlens=torch.tensor([0, 6]))
    for cu in (torch.tensor([0.0, 6.0]), torch.tensor([0]), torch.tensor([[0, 6]])):
        with pytest.raises(ValueError, match="cu_seqlens"):
            decay_attention(*inputs(), cu_seqlens=cu)
    with pytest.raises(ValueError, match="initial_state"):   # one state for each of the two packed sequences
        decay_attention(*inputs(), cu_seqlens=torch.tensor([0, 3, 6]), initial_state=torch.zeros(1, 4, 8, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        decay_attention(*inputs())


def test_step_refuses():
    q, v, g, state = torch.zeros(3, 2, 8), torch.zeros(3, 4, 8), torch.zeros(3, 4), torch.zeros(3, 4, 8, 8)
    with pytest.raises(ValueError, match="only 2 states"):
        decay_attention_step(state[:2], q, q, v, g)
    with pytest.raises(ValueError, match="float32"):
        decay_attention_step(state.bfloat16(), q, q, v, g)
    with pytest.raises(ValueError, match="contiguous"):
        decay_attention_step(state.transpose(2, 3), q, q, v, g)
    with pytest.raises(ValueError, match="contiguous"):      # one state for all requests: they would overwrite it
        decay_attention_step(state[:1].expand(3, -1, -1, -1), q, q, v, g)
    with pytest.raises(ValueError, match="slots"):
        decay_attention_step(state, q, q, v, g, slots=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no gradient"):
        decay_attention_step(state, q.requires_grad_(True), q, v, g)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        decay_attention_step(state, q, q, v, g)


def test_block_norm_refuses():
    x, w = torch.zeros(2, 3, 16), torch.zeros(16)
    for kw, says in ((dict(residual=x[:, :2]), "residual"), (dict(residual=x.half()), "residual"), (dict(gate=torch.zeros(2, 3, 1)), "gate"),
                     (dict(gate=torch.zeros(3, 1, 16)), "gate"), (dict(gate=torch.zeros(2, 3, 16).half()), "gate"),
                     (dict(post_weight=torch.zeros(15)), "weights"), (dict(pre_weight=w.double()), "weights"),
                     (dict(scale=torch.zeros(())), "scale"), (dict(gate=x, gate_activation="relu"), "gate_activation")):
        with pytest.raises(ValueError, match=says):
            block_norm(x, **{"residual": x, **kw})
    h = x.bfloat16()
    with pytest.raises(ValueError, match="one type"):
        block_norm(h, h, post_weight=w, pre_weight=w.bfloat16())
    with pytest.raises(ValueError, match="8192"):
        block_norm(torch.zeros(1, 8193), torch.zeros(1, 8193))
    with pytest.raises(RuntimeError, match="CUDA"):
        block_norm(x, x)


def test_c_entry_points_refuse_before_any_launch():
    lib = _cabi.load()
    a = _cabi.DecayArgs(batch=1, seqlen=6, nheads=4, nkheads=2, kdim=8, vdim=8)
    f, b = ctypes.c_size_t(), ctypes.c_size_t()
    sizes = lambda: lib.bissd_decay_workspace_bytes(ctypes.byref(a), ctypes.byref(f), ctypes.byref(b))
    assert sizes() == 0 and 0 < f.value < b.value and f.value % 256 == 0 and b.value % 256 == 0
    assert lib.bissd_decay_forward(ctypes.byref(a), 4096, 1 << 30, None) == -1                # NULL tensors
    for name in ("q", "k", "v", "g", "dout"):
        setattr(a, name, _cabi.Tensor(4096, 48, 8, 8))
    a.o = a.dq = a.dk = a.dv = 4096
    assert lib.bissd_decay_forward(ctypes.byref(a), 4096, f.value - 1, None) == -5            # workspace
    assert lib.bissd_decay_backward(ctypes.byref(a), 4096, b.value - 1, None) == -5
    assert lib.bissd_decay_forward(ctypes.byref(a), 4096 + 16, f.value, None) == -4
    for field, value, rc in (("nkheads", 3, -2), ("kdim", 257, -2), ("vdim", 0, -2), ("nseq", -1, -2), ("dtype", 5, -3), ("g_dtype", -1, -3)):
        kept = getattr(a, field)
        setattr(a, field, value)
        assert sizes() == rc, field
        setattr(a, field, kept)
    a.nseq = 2
    assert lib.bissd_decay_forward(ctypes.byref(a), 4096, 1 << 30, None) == -1                # no boundaries
    assert lib.bissd_decay_workspace_bytes(None, None, None) == -1
    s = _cabi.DecayStepArgs(batch=2, nheads=4, nkheads=2, kdim=8, vdim=8, nslots=1, slot_stride=256, state=4096)
    for name in ("q", "k", "v", "g", "o"):
        setattr(s, name, _cabi.Tensor(4096, 48, 0, 8))
    assert lib.bissd_decay_step(ctypes.byref(s), None) == -2                                  # two requests, one state
    s.nslots, s.slot_stride = 2, 255
    assert lib.bissd_decay_step(ctypes.byref(s), None) == -2                                  # states that overlap
    s.slot_stride, s.state = 256, 4097
    assert lib.bissd_decay_step(ctypes.byref(s), None) == -4
    n = _cabi.BlockNormArgs(rows=4, width=16, x=4096, residual=4096, r=4096, pre_weight=4096)
    assert lib.bissd_block_norm_forward(ctypes.byref(n), None) == -1                          # nowhere for the normed rows
    n.normed, n.gate_rows = 4096, 3
    assert lib.bissd_block_norm_forward(ctypes.byref(n), None) == -2
    n.gate_rows, n.r_dtype = 2, 1
    assert lib.bissd_block_norm_forward(ctypes.byref(n), None) == -3
    n.r_dtype, n.width = 0, 8193
    assert lib.bissd_block_norm_forward(ctypes.byref(n), None) == -2
    n.width, n.dnormed = 16, 4096
    assert lib.bissd_block_norm_backward(ctypes.byref(n), 4096, 0, None) == -1                # nothing kept by the forward pass


def test_struct_layout_matches_the_header(tmp_path):
    import os
    import subprocess

    from conftest import ROOT
    c = tmp_path / "t.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "bissd.h"\nint main(void) { printf("%zu %zu %zu %zu %zu %zu",'
                 'sizeof(bissd_decay_args), offsetof(bissd_decay_args, dout), sizeof(bissd_decay_step_args),'
                 'offsetof(bissd_decay_step_args, slots), sizeof(bissd_block_norm_args), offsetof(bissd_block_norm_args, dpre)); return 0; }')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "t")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "t")]).split()]
    assert got == [ctypes.sizeof(_cabi.DecayArgs), _cabi.DecayArgs.dout.offset, ctypes.sizeof(_cabi.DecayStepArgs),
                   _cabi.DecayStepArgs.slots.offset, ctypes.sizeof(_cabi.BlockNormArgs), _cabi.BlockNormArgs.dpre.offset]
