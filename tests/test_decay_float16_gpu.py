"""The causal decay attention in float16 on the tensor cores, where sizes that other tests give to bfloat16 alone go another way, and at
the small end of the type's range.  Tolerances are test_decay_attention_gpu's, which see."""
import pytest
import torch

from oracle.decay_oracle import decay_attention_reference
from test_decay_attention_gpu import bound, check, distance, make, wide

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("size", [(1, 300, 32, 1, 64, 64), (2, 260, 24, 2, 128, 64), (1, 2100, 1, 1, 128, 80), (1, 3001, 2, 1, 64, 64)], ids=str)
def test_shared_heads_and_long_rows(size):
    """Several blocks a head of q and k; states walked in several segments."""
    b, L, h, hk, n, p = size
    q, k, v, g, init = make(F16, b, L, h, hk, n, p, initial=True, seed=L)
    g = (g.float() / 50).to(g.dtype) if L > 1000 else g
    gen = torch.Generator().manual_seed(2)
    check(F16, (q, k, v, g, init), torch.randn(b, L, h, p, generator=gen).to(F16), torch.randn(b, h, n, p, generator=gen))


@pytest.mark.parametrize("g_dtype", [F16, torch.float32], ids=["fp16", "fp32"])
def test_packed_with_decays_of_either_type(g_dtype):
    bounds = [0, 5, 6, 6, 134, 390, 400]
    tensors = make(F16, 1, 407, 4, 2, 64, 64, initial=True, seqs=6, seed=3, g_dtype=g_dtype)
    gen = torch.Generator().manual_seed(9)
    check(F16, tensors, torch.randn(1, 407, 4, 64, generator=gen).to(F16), torch.randn(6, 4, 64, 64, generator=gen), bounds)


@pytest.mark.parametrize("L", [300, 2100])
@pytest.mark.parametrize("exponent", [-14, -20])
def test_states_of_small_values(L, exponent):
    """v at and below float16's smallest normal number (2^-14): the states are float32's all the same."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = make(F16, 1, L, 2, 1, 64, 64, seed=L)
    v = (v.float() * 2.0 ** exponent).to(F16)
    g = (g.float() / 50).to(F16)
    _, final = decay_attention(*(t.cuda() for t in (q, k, v, g)), return_final_state=True)
    want = decay_attention_reference(*(wide(t) for t in (q, k, v, g)))[1]
    sizes = decay_attention_reference(*(wide(t).abs() for t in (q, k, v)), wide(g))[1]
    assert distance(final, want) <= bound(F16, L + 128, want, sizes, "state")
