"""Pairs of tokens behind many strong decays of the same chunk: what came before takes no digits from their weights.

Tokens from FIRST on hardly decay; those before empty the state, or nearly.  Inputs are unit vectors chosen so that each result
is one pair's weight w_ts = scale e^{g_{s+1} + ... + g_t}, alone: |result - w| <= (eps / 2 + 2^-18) w.  Half a step for the rounding to the
tensors' type - once: a weight that has been rounded already is not rounded again - and 2^-18 for the exponent: it is a sum of at most
27 fp32 decays, in powers of two below 1 (27 roundings of 2^-24 of it), and the hardware's 2^x is within 2^-22.  The decays' gradient is a sum of
n^2 pairs at most, fp32 throughout: (n^(1/2) + 8) roundings of the sum of the terms' sizes, rows and columns."""
import math

import pytest
import torch

from test_decay_attention_gpu import make, check

pytestmark = pytest.mark.gpu
FIRST, L = 100, 128                                   # one chunk: no state of 16 bits stands between two tokens
N = 64
CASES = [(dtype, before, every) for dtype in (torch.float16, torch.bfloat16) for before in (-math.inf, -100.0, -20.0) for every in (1, 2)]
ID = lambda c: "%s-%g-%d" % (str(c[0])[6:], c[1], c[2])


def decays(before, every):
    g = torch.full((1, L, 1), -0.001)
    g[:, 1:FIRST + 1:every] = before
    g[:, FIRST + 1:] -= 0.0005 * torch.rand(1, L - FIRST - 1, 1, generator=torch.Generator().manual_seed(1))
    return g


def weights(g):
    """w[t, s] in 64 bits for s, t from FIRST + 1 on, zero above the diagonal; scale 1."""
    c = torch.cumsum(g[0, FIRST + 1:, 0].double(), 0)
    return torch.exp(c[:, None] - c[None, :]).tril()


def units(n=L - FIRST - 1):
    """(1, L, 1, N): unit vector s of token FIRST + 1 + s, zeros before; and the same first unit vector for all of them."""
    own, one = torch.zeros(1, L, 1, N), torch.zeros(1, L, 1, N)
    own[0, FIRST + 1:, 0, :n] = torch.eye(n)
    one[0, FIRST + 1:, 0, 0] = 1
    return own, one


def near(got, want, dtype):
    n = want.shape[0]
    got = got[0, FIRST + 1:, 0, :n].double().cpu()
    worst = ((got - want).abs() / want.clamp_min(1e-30)).where(want > 0, got.abs()).max().item()
    assert worst <= torch.finfo(dtype).eps / 2 + 2.0 ** -18, worst


@pytest.mark.parametrize("case", CASES, ids=ID)
def test_weights_of_outputs(case):
    from ssd.uni.decay_attention import decay_attention
    dtype, before, every = case
    g, (own, one) = decays(before, every), units()
    out = decay_attention(one.to(dtype).cuda(), one.to(dtype).cuda(), own.to(dtype).cuda(), g.cuda(), scale=1.0)
    near(out, weights(g), dtype)


@pytest.mark.parametrize("case", CASES, ids=ID)
@pytest.mark.parametrize("what", ["dq", "dk", "dv", "dg"])
def test_weights_of_gradients(case, what):
    from ssd.uni.decay_attention import decay_attention
    dtype, before, every = case
    g, (own, one) = decays(before, every), units()
    q, k, v, dout = one, one, one, one                # dq_t[s] = w_ts where k has unit vectors, and so on
    if what == "dq":
        k = own
    elif what == "dk":
        q = own
    elif what == "dv":
        dout = own
    leaves = [t.to(dtype).cuda().requires_grad_(True) for t in (q, k, v)] + [g.cuda().requires_grad_(True)]
    grads = torch.autograd.grad(decay_attention(*leaves, scale=1.0), leaves, dout.to(dtype).cuda())
    w = weights(g)
    if what in ("dq", "dk", "dv"):
        near(grads["qkv".index(what[1])], w if what == "dq" else w.T, dtype)
        return
    n = w.shape[0]
    want = torch.stack([w[t:, :t].sum() for t in range(n)])       # every pair s < t <= t'
    got = grads[3][0, FIRST + 1:, 0].double().cpu()
    most = (n ** 0.5 + 8) * 2.0 ** -24 * 2 * w.sum() + 2.0 ** -18 * want
    assert bool(((got - want).abs() <= most).all()), ((got - want).abs() / most).max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_against_the_definition(dtype):
    """Resets all over a row and a packed one, everything random (a pair that crosses one has no weight at all)."""
    q, k, v, g, _ = make(dtype, 1, 300, 2, 1, 64, 64, seed=3, g_dtype=torch.float32)
    g = -0.002 * torch.rand(g.shape, generator=torch.Generator().manual_seed(2))
    g[:, 1:110:2] = -1e4
    g[:, 130:230:3] = -120.0
    gen = torch.Generator().manual_seed(4)
    dout = torch.randn(1, 300, 2, 64, generator=gen).to(dtype)
    check(dtype, (q, k, v, g, None), dout)
    check(dtype, (q, k, v, g, None), dout, bounds=[3, 120, 121, 299])
