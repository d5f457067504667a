"""The decays' gradient on the tensor cores: a token's own pair is not in it, and costs it no digits however large it is.

Tolerances (2-norms), with A what the definition gives for the inputs' absolute values, in which no own pair counts; n = seqlen + kdim +
vdim.  In one chunk without states nothing of it is rounded to 16 bits: (n^(1/2) + 8) 2^-24 |A| for sums of products as in
test_decay_attention_gpu, and 2^-18 |A| for the pairs' weights, whose exponents are sums of decays below 2^8, with the hardware's 2^x within
2^-22 (an exponent of 2^5, a rounding of 2^-19; pairs whose weight is below 2^-32 are nothing beside the others).  Over several chunks states of 16
bits stand between tokens: test_decay_attention_gpu's bound."""
import pytest
import torch

from oracle.decay_oracle import decay_attention_reference
from test_decay_attention_gpu import bound, make, wide

pytestmark = pytest.mark.gpu


def case(dtype, L, rate, own, n=64, p=64, seed=1):
    q, k, v, _, _ = make(dtype, 1, L, 4, 2, n, p, seed=L)
    gen = torch.Generator().manual_seed(seed)
    g = -rate * (0.5 + torch.rand(1, L, 4, generator=gen))
    dout = torch.randn(1, L, 4, p, generator=gen).to(dtype)
    return (q, q.clone(), v, g, v.clone()) if own else (q, k, v, g, dout)


def gradients(q, k, v, g, dout, bounds=None):
    from ssd.uni.decay_attention import decay_attention
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g)]
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    got = torch.autograd.grad(decay_attention(*leaves, cu_seqlens=cu), leaves, dout.cuda())[3]

    def definition(size):
        refs = [(wide(t) if i == 3 else size(wide(t))).requires_grad_(True) for i, t in enumerate((q, k, v, g))]
        return torch.autograd.grad(decay_attention_reference(*refs, bounds=bounds)[0], refs, size(wide(dout)))[3]

    return got.double().cpu(), definition(lambda t: t), definition(torch.abs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("own", [False, True], ids=["random", "large-own-pairs"])
@pytest.mark.parametrize("rate", [0.005, 0.2, 3.0, 12.0])
@pytest.mark.parametrize("size", [(60, 64, 64), (128, 64, 64), (127, 128, 80)], ids=str)
def test_one_chunk(dtype, size, rate, own):
    L, n, p = size
    got, want, sizes = gradients(*case(dtype, L, rate, own, n, p))
    off, most = float((got - want).norm()), (((L + n + p) ** 0.5 + 8) * 2.0 ** -24 + 2.0 ** -18) * float(sizes.norm())
    print("%.2e / %.2e, %.2e of the gradient" % (off, most, off / float(want.norm())))
    assert off <= most


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("own", [False, True], ids=["random", "large-own-pairs"])
@pytest.mark.parametrize("rate", [0.2, 3.0, 12.0])
@pytest.mark.parametrize("bounds", [None, [3, 131, 131, 259, 300]], ids=["row", "packed"])
def test_several_chunks(dtype, rate, own, bounds):
    got, want, sizes = gradients(*case(dtype, 310, rate, own), bounds)
    off, most = float((got - want).norm()), bound(dtype, 310 + 128, want, sizes, "decay")
    print("%.2e / %.2e, %.2e of the gradient" % (off, most, off / float(want.norm())))
    assert off <= most
