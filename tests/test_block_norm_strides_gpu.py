"""Norms around a block on rows that lie further apart than the kernels' 32-bit strides reach."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_rows_far_apart():
    from ssd.block_norm import block_norm
    x = torch.empty((1 << 30) + 1024, dtype=torch.bfloat16, device="cuda")
    far = x.as_strided((2, 1024), (1 << 30, 1))
    near = torch.randn(2, 1024, device="cuda").bfloat16()
    far.copy_(near)
    w = torch.rand(1024, device="cuda")
    want = block_norm(near, near, post_weight=w, pre_weight=w)
    for args in ((far, near), (near, far), (far, far)):
        assert all(torch.equal(a, b) for a, b in zip(block_norm(*args, post_weight=w, pre_weight=w), want))
    one = block_norm(far[1:], far[1:], post_weight=w, pre_weight=w)
    assert all(torch.equal(a, b[1:]) for a, b in zip(one, want))
