"""The causal decay attention where many heads share q and k, with other scales and types than the usual, and from the gradients that
an expression hands in.  Tolerances are test_decay_attention_gpu's, which see."""
import pytest
import torch

from test_decay_attention_gpu import check, make, off, tolerance, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [(1, 300, 32, 1, 64, 64), (2, 260, 24, 2, 128, 64), (1, 200, 20, 2, 64, 128)], ids=str)
def test_many_heads_share_q_and_k(size):
    """Few rows: several blocks walk the heads of one q and k, and their parts of dq and dk are summed."""
    b, L, h, hk, n, p = size
    tensors = make(torch.bfloat16, b, L, h, hk, n, p, initial=True, seed=L)
    gen = torch.Generator().manual_seed(2)
    check(torch.bfloat16, tensors, torch.randn(b, L, h, p, generator=gen).to(torch.bfloat16), torch.randn(b, h, n, p, generator=gen))


def test_one_block_walks_many_heads():
    """Rows enough that one block takes all sixteen heads of a q and k: against the CUDA cores' results for the same values in fp32,
    themselves good to fp32's tolerance."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(torch.bfloat16, 4, 4096, 64, 4, 64, 64, seed=1))
    dout = torch.randn(v.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    results = []
    for dtype in (torch.bfloat16, torch.float32):
        leaves = [t.to(dtype).requires_grad_(True) for t in (q, k, v, g)]
        out = decay_attention(*leaves)
        results.append([out, *torch.autograd.grad(out, leaves, dout.to(dtype))])
    n = 4096 + 128
    for i, (got, want) in enumerate(zip(*results)):
        kind = "decay" if i == 4 else "out"
        assert off(got, wide(want)) <= tolerance(torch.bfloat16, n, kind) + tolerance(torch.float32, n), i
        for head in (0, 7, 8, 15, 63):                # each head by itself: a head's tables are made in turns
            if i in (0, 3, 4):
                assert off(got[:, :, head], wide(want[:, :, head])) <= tolerance(torch.bfloat16, n, kind) + tolerance(torch.float32, n), (i, head)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 0.03125, -0.25, 0.0])
def test_a_scale_of_ones_own(dtype, scale):
    tensors = make(dtype, 1, 270, 4, 2, 64, 64, initial=True, seed=4)
    gen = torch.Generator().manual_seed(2)
    check(dtype, tensors, torch.randn(1, 270, 4, 64, generator=gen).to(dtype), torch.randn(1, 4, 64, 64, generator=gen), scale=scale)


@pytest.mark.parametrize("decay", ["token", "head"])
def test_decays_of_32_bits(decay):
    """The decays of bf16 tensors may be fp32, and their gradient then is."""
    tensors = make(torch.bfloat16, 2, 330, 4, 1, 64, 64, decay, seed=6, g_dtype=torch.float32)
    assert tensors[3].dtype == torch.float32
    check(torch.bfloat16, tensors, torch.randn(2, 330, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_gradients_that_an_expression_hands_in(dtype):
    """Broadcast, transposed and cut at an odd address: the same bits as from a tensor of its own."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(dtype, 2, 200, 4, 2, 64, 64, seed=9))
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    dout = torch.randn(2, 4, 200, 64, device="cuda").to(dtype).transpose(1, 2)
    odd = torch.empty(dout.numel() + 1, dtype=dtype, device="cuda")[1:].view(2, 200, 4, 64).copy_(dout)
    one = torch.randn(64, device="cuda").to(dtype)

    def grads(d):
        return torch.autograd.grad(decay_attention(*leaves), leaves, d)

    want = grads(dout.contiguous())
    for d in (dout, odd):
        assert all(torch.equal(a, b) for a, b in zip(grads(d), want))
    assert all(torch.equal(a, b) for a, b in zip(grads(one.expand(v.shape)), grads(one.expand(v.shape).contiguous())))


def test_two_calls_at_once():
    """Two streams, forward and backward: no scratch is shared."""
    from ssd.uni.decay_attention import decay_attention
    cases = [[t.cuda().requires_grad_(True) for t in make(torch.bfloat16, 1, 3000, 4, 2, 64, 64, seed=i)[:4]] for i in (1, 2)]
    douts = [torch.randn_like(c[2]) for c in cases]

    def one(c, d):
        out = decay_attention(*c)
        return [out.detach(), *torch.autograd.grad(out, c, d)]

    want = [one(c, d) for c, d in zip(cases, douts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for c, d, s in zip(cases, douts, streams):
            with torch.cuda.stream(s):
                got.append(one(c, d))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
