"""Thousands of packed sequences, many without a token: more than one block's scan covers at a time.  Tolerances are
test_decay_attention_gpu's, which see."""
import pytest
import torch

from test_decay_attention_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("seqs", [1023, 1024, 1025, 2500])
def test_more_sequences_than_threads(dtype, seqs):
    gen = torch.Generator().manual_seed(seqs)
    lengths = torch.randint(0, 3, (seqs,), generator=gen)
    lengths[seqs // 2] = 140                          # one that ends inside its second chunk
    bounds = [4] + (4 + lengths.cumsum(0)).tolist()
    L = bounds[-1] + 3
    tensors = make(dtype, 1, L, 2, 1, 16, 16, initial=True, seqs=seqs, seed=seqs)
    check(dtype, tensors, torch.randn(1, L, 2, 16, generator=gen).to(dtype), torch.randn(seqs, 2, 16, 16, generator=gen), bounds)
