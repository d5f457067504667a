"""The decays' gradient on CUDA cores: a token's own pair is not in it, and costs it no digits however large it is.

Tolerance (2-norms), with A what the definition gives for the inputs' absolute values, in which no own pair counts: as
test_decay_attention_gpu's for fp32, (n^(1/2) + 8) 2^-24 |A|, n = seqlen + kdim + vdim.  Each value of it is a product of q (or k) with a
gradient, kdim terms, whose own terms are sums over the tokens and vdim, and is summed over the tokens that follow: n roundings in a row.
For large own pairs the inputs are made so that q.k of a token with itself, and v.dout with itself, are about N and P, and
other pairs' about N^(1/2) and P^(1/2)."""
import pytest
import torch

from oracle.decay_oracle import decay_attention_reference
from test_decay_attention_gpu import make, wide

pytestmark = pytest.mark.gpu


def gradient(tensors, dout, bounds=None, dfinal=None):
    from ssd.uni.decay_attention import decay_attention
    leaves = [None if t is None else t.cuda().requires_grad_(True) for t in tensors]
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    out, final = decay_attention(*leaves[:4], initial_state=leaves[4], return_final_state=True, cu_seqlens=cu)
    outs, gos = ([out], [dout.cuda()]) if dfinal is None else ([out, final], [dout.cuda(), dfinal.cuda()])
    return torch.autograd.grad(outs, leaves[:4], gos)


def definition(tensors, dout, size, bounds=None, dfinal=None):
    leaves = [None if t is None else (wide(t) if i == 3 else size(wide(t))).requires_grad_(True) for i, t in enumerate(tensors)]
    out, final = decay_attention_reference(*leaves[:4], initial_state=leaves[4], bounds=bounds)
    outs, gos = ([out], [size(wide(dout))]) if dfinal is None else ([out, final], [size(wide(dout)), size(wide(dfinal))])
    return torch.autograd.grad(outs, leaves[:4], gos, allow_unused=True)


@pytest.mark.parametrize("own", [False, True], ids=["random", "large-own-pairs"])
@pytest.mark.parametrize("rate", [0.005, 0.2, 3.0, 12.0])
@pytest.mark.parametrize("size", [(1, 90, 2, 1, 32, 48), (2, 400, 4, 2, 64, 64), (1, 700, 3, 3, 112, 128), (1, 130, 2, 2, 200, 33)], ids=str)
def test_digits(size, rate, own):
    """Also where decays are so strong that a token's own pair is nearly all there is."""
    b, L, h, hk, n, p = size
    q, k, v, _, init = make(torch.float32, b, L, h, hk, n, p, initial=True, seed=L)
    gen = torch.Generator().manual_seed(1)
    g = -rate * (0.5 + torch.rand(b, L, h, generator=gen))
    dout, dfinal = torch.randn(b, L, h, p, generator=gen), torch.randn(b, h, n, p, generator=gen)
    if own:
        k, dout = q.clone(), v.clone()
    tensors = (q, k, v, g, init)
    got = gradient(tensors, dout, dfinal=dfinal)
    want, sizes = (definition(tensors, dout, f, dfinal=dfinal) for f in (lambda t: t, torch.abs))
    most = ((L + n + p) ** 0.5 + 8) * 2.0 ** -24
    for name, a, w, s in zip(("dq", "dk", "dv", "dg"), got, want, sizes):
        off = float((a.double().cpu() - w).norm())
        print(name, "%.2e / %.2e, %.2e of the gradient" % (off, most * float(s.norm()), off / float(w.norm())))
        assert off <= most * float(s.norm()), name


@pytest.mark.parametrize("bounds", [[0, 5, 6, 6, 134, 390, 400], [3, 131, 131, 259, 300]], ids=str)
def test_packed(bounds):
    L = bounds[-1] + 7
    tensors = make(torch.float32, 1, L, 4, 2, 64, 64, seed=len(bounds))
    tensors = (tensors[0], tensors[0].clone(), *tensors[2:])
    dout = tensors[2].clone()
    got = gradient(tensors, dout, bounds)
    want, sizes = (definition(tensors, dout, f, bounds) for f in (lambda t: t, torch.abs))
    for name, a, w, s in zip(("dq", "dk", "dv", "dg"), got, want, sizes):
        assert float((a.double().cpu() - w).norm()) <= ((L + 128) ** 0.5 + 8) * 2.0 ** -24 * float(s.norm()), name
    outside = [*range(bounds[0]), *range(bounds[-1], L)]
    assert all(not t[:, outside].any() for t in got)


@pytest.mark.parametrize("size", [(1, 60, 2, 1, 7, 5), (1, 300, 2, 1, 96, 40)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_16_bits_on_cuda_cores(dtype, size):
    """Sizes and scales that the tensor cores do not take: sums of fp32 here too, and half a step for the result's rounding."""
    from ssd.uni.decay_attention import decay_attention
    b, L, h, hk, n, p = size
    q, _, v, g, _ = make(dtype, b, L, h, hk, n, p, seed=L, g_dtype=torch.float32)
    k, dout, scale = q.clone(), v.clone(), -0.25      # a negative scale is not the tensor cores'
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g)]
    dg = torch.autograd.grad(decay_attention(*leaves, scale=scale), leaves, dout.cuda())[3]
    refs = [wide(t).requires_grad_(True) for t in (q, k, v, g)]
    want = torch.autograd.grad(decay_attention_reference(*refs, scale=scale)[0], refs, wide(dout))[3]
    refs = [(wide(t) if i == 3 else wide(t).abs()).requires_grad_(True) for i, t in enumerate((q, k, v, g))]
    sizes = torch.autograd.grad(decay_attention_reference(*refs, scale=-scale)[0], refs, wide(dout).abs())[3]
    assert float((dg.double().cpu() - want).norm()) <= ((L + n + p) ** 0.5 + 8) * 2.0 ** -24 * float(sizes.norm())
