"""Arguments beyond what the kernels count in 32 bits: refused, or brought inside.  The refusals need no GPU."""
import pytest
import torch


def test_too_many_rows_and_tokens():
    from ssd.block_norm import block_norm
    from ssd.uni.decay_attention import decay_attention
    many = torch.zeros(1, 1).expand(1 << 30, 1)
    with pytest.raises(ValueError, match="rows"):
        block_norm(many, many)
    q = torch.zeros(1, 1, 1, 1).expand(1, 1 << 23, 1, 1)
    with pytest.raises(ValueError, match="tokens"):
        decay_attention(q, q, q, torch.zeros(1))


@pytest.mark.gpu
def test_boundaries_of_64_bits():
    """What lies outside is taken as the nearest that does not, also where 32 bits would see something else."""
    from ssd.uni.decay_attention import decay_attention
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 200, 2, 64, generator=gen).bfloat16().cuda() for _ in range(3))
    g = -torch.rand(1, 200, 2, generator=gen).bfloat16().cuda()
    far = torch.tensor([-(1 << 32) + 7, 40, (1 << 32) + 60], device="cuda")
    near = torch.tensor([0, 40, 200], dtype=torch.int32, device="cuda")
    a = decay_attention(q, k, v, g, return_final_state=True, cu_seqlens=far)
    b = decay_attention(q, k, v, g, return_final_state=True, cu_seqlens=near)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
