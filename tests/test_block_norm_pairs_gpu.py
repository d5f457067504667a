"""Norms around a block where pairs of channels are all that lies aligned: even widths, addresses and strides of two elements.  Checks and
tolerances are test_block_norm_gpu's, which see."""
import pytest
import torch

import test_block_norm_gpu as norms

pytestmark = pytest.mark.gpu

CASES = [
    ((3, 17, 2), torch.bfloat16, False, "full", "silu", "vector", True, True, torch.float32),
    ((5, 9, 34), torch.bfloat16, True, "row", "sigmoid", "vector", True, True, torch.float32),
    ((4, 30, 1020), torch.float16, False, "full", "sigmoid", 0.5, True, True, torch.float32),
    ((2, 7, 250), torch.float32, False, "full", "silu", "vector", True, True, torch.float32),
    ((300, 2062), torch.bfloat16, True, "full", "sigmoid", "vector", True, True, torch.float32),
    ((2, 9, 4236), torch.bfloat16, True, "full", "sigmoid", "vector", False, True, torch.float32),
    ((2, 5, 8190), torch.float16, True, "row", "silu", "vector", True, True, torch.float32),
    ((2, 5, 8190), torch.float32, False, "full", None, 1.0, True, False, torch.float32),
]


@pytest.mark.parametrize("case", CASES, ids=["x".join(map(str, c[0])) for c in CASES])
def test_even_widths(case):
    norms.test_forward_and_backward_match_the_definition(case)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_addresses_and_strides_of_pairs(dtype):
    """The same bits as of rows that lie aligned: a thread has the same eight channels."""
    from ssd.block_norm import block_norm
    gen = torch.Generator("cuda").manual_seed(1)
    x, res = (torch.randn(40, 512, device="cuda", generator=gen).to(dtype) for _ in range(2))
    w = torch.rand(512, device="cuda", generator=gen)
    want = block_norm(x, res, post_weight=w, pre_weight=w)
    for at, stride in ((2, 512), (2, 518), (0, 514)):
        store = torch.empty(at + 40 * stride, dtype=dtype, device="cuda")
        moved = store[at:].as_strided((40, 512), (stride, 1), store.storage_offset() + at).copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(block_norm(moved, res, post_weight=w, pre_weight=w), want))
