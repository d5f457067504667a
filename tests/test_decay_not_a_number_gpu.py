"""A log decay that is no number makes no number of what comes after it in its sequence, on either kind of core; nothing else changes."""
import pytest
import torch

from test_decay_attention_gpu import make

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
NAN = float("nan")


@TYPES
@pytest.mark.parametrize("at", [100, 180, 249])
def test_outputs_and_states(dtype, at):
    """One sequence of three, 100 ... 249, two chunks of it: its outputs from the token on and its final state."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, init = (t.cuda() for t in make(dtype, 1, 400, 4, 2, 64, 64, initial=True, seqs=3, seed=6))
    cu = torch.tensor([0, 100, 250, 400], dtype=torch.int32, device="cuda")
    call = lambda: decay_attention(q, k, v, g, initial_state=init, return_final_state=True, cu_seqlens=cu)
    want = call()
    g[:, at, 2] = NAN
    out, final = call()
    assert bool(out[:, at:250, 2].isnan().all()) and bool(final[1, 2].isnan().all())
    for a, z, i in ((0, 100, 0), (250, 400, 2)):
        assert torch.equal(out[:, a:z], want[0][:, a:z]) and torch.equal(final[i], want[1][i])
    others = [0, 1, 3]                                # heads
    assert torch.equal(out[:, :, others], want[0][:, :, others]) and torch.equal(final[:, others], want[1][:, others])


@TYPES
@pytest.mark.parametrize("L", [200, 2100])
def test_rows_of_a_batch(dtype, L):
    """Also where a row is walked in several segments: the states behind it."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(dtype, 2, L, 2, 1, 64, 64, seed=L))
    want = decay_attention(q, k, v, g, return_final_state=True)
    g[1, 40, 0] = NAN
    out, final = decay_attention(q, k, v, g, return_final_state=True)
    assert bool(out[1, 40:, 0].isnan().all()) and bool(final[1, 0].isnan().all())
    assert torch.equal(out[0], want[0][0]) and torch.equal(out[1, :, 1], want[0][1, :, 1])
    assert torch.equal(final[0], want[1][0]) and torch.equal(final[1, 1], want[1][1, 1])


@TYPES
def test_gradients(dtype):
    """dg of the token itself, and dk and dv of the tokens before it, whose outputs behind it are no numbers; other sequences' none."""
    from ssd.uni.decay_attention import decay_attention
    tensors = [t.cuda() for t in make(dtype, 1, 400, 2, 2, 64, 64, seed=6)[:4]]
    cu = torch.tensor([0, 100, 250, 400], dtype=torch.int32, device="cuda")
    dout = torch.randn_like(tensors[2])

    def grads():
        leaves = [t.clone().requires_grad_(True) for t in tensors]
        return torch.autograd.grad(decay_attention(*leaves, cu_seqlens=cu), leaves, dout)

    want = grads()
    tensors[3][:, 150, 1] = NAN
    got = grads()
    for a, z in ((0, 100), (250, 400)):
        assert all(torch.equal(x[:, a:z], y[:, a:z]) for x, y in zip(got, want))
    assert all(torch.equal(x[:, :, 0], y[:, :, 0]) for x, y in zip(got, want))
    dq, dk, dv, dg = (t[0, :, 1] for t in got)
    assert bool(dq[150:250].isnan().all()) and bool(dk[100:150].isnan().all()) and bool(dv[100:150].isnan().all()) and bool(dg[150].isnan())


@TYPES
def test_single_tokens(dtype):
    from ssd.uni.decay_attention import decay_attention_step
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 2, 64, generator=gen).to(dtype).cuda() for _ in range(3))
    state, g = torch.randn(2, 2, 64, 64, generator=gen).cuda(), torch.full((2, 2), -0.5, device="cuda").to(dtype)
    g[1, 0] = NAN
    out = decay_attention_step(state, q, k, v, g)
    assert bool(out[1, 0].isnan().all()) and bool(state[1, 0].isnan().all())
    assert bool(out[0].isfinite().all()) and bool(out[1, 1].isfinite().all()) and bool(state[0].isfinite().all())
