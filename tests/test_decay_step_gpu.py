"""One token of every request against the definition in 64 bits.  Tolerances (2-norms), of what the definition gives for the inputs'
absolute values, so that they hold whatever cancels: states 4 2^-24 (a product, a decay, a sum and the decay's own exponential),
outputs (kdim + 4) 2^-24 and, in 16 bits, half a step for their rounding."""
import pytest
import torch

from oracle.decay_oracle import decay_attention_reference, decay_step_reference
from test_decay_attention_gpu import distance, off, wide

pytestmark = pytest.mark.gpu


def make(dtype, b, h, hk, n, p, pool, per_head=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    g = -torch.rand(h, generator=gen) if per_head else -torch.rand(b, h, generator=gen)
    return r(pool, h, n, p), r(b, hk, n).to(dtype), r(b, hk, n).to(dtype), r(b, h, p).to(dtype), g if per_head else g.to(dtype)


def check(dtype, out, state, want, states, sizes, size_states, times=1):
    """`times`: tokens one after another in one state."""
    to, ts = tolerances(dtype, states.shape[2])
    eps = times * to * float(sizes.norm()), times * ts * float(size_states.norm())
    assert out.dtype == dtype and distance(out, want) <= eps[0] and distance(state, states) <= eps[1]


def both(state, q, k, v, g, slots):
    """The definition of the inputs, and of their absolute values."""
    args = [wide(t) for t in (state, q, k, v, g)]
    return *decay_step_reference(*args, slots=slots), *decay_step_reference(*(t.abs() for t in args[:4]), args[4], slots=slots)


def tolerances(dtype, n):
    return (n + 4) * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2), 4 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (1, 8, 8, 64, 64), (5, 6, 2, 128, 64), (3, 4, 1, 96, 80), (2, 3, 3, 256, 256), (4, 2, 1, 33, 7),
                                  (2, 2, 2, 130, 33)], ids=str)
@pytest.mark.parametrize("how", ["plain", "slots", "head"])
def test_step_matches_the_definition(dtype, size, how):
    from ssd.uni.decay_attention import decay_attention_step
    b, h, hk, n, p = size
    pool = b + 3 if how == "slots" else b
    state, q, k, v, g = make(dtype, b, h, hk, n, p, pool, how == "head", seed=n + p)
    slots = torch.randperm(pool, generator=torch.Generator().manual_seed(1))[:b].to(torch.int32) if how == "slots" else None
    dev = state.cuda()
    out = decay_attention_step(dev, q.cuda(), k.cuda(), v.cuda(), g.cuda(), slots=None if slots is None else slots.cuda())
    check(dtype, out, dev, *both(state, q, k, v, g, slots))
    if slots is not None:                             # states of nobody are left as they were
        rest = [i for i in range(pool) if i not in slots.tolist()]
        assert torch.equal(dev[rest].cpu(), state[rest])


@pytest.mark.parametrize("many", [False, True])
def test_rows_of_padding_and_tokens_of_one_sequence(many):
    """A slot outside the pool is padding; requests with one slot are its tokens, in order."""
    from ssd.uni.decay_attention import decay_attention_step
    slots = torch.tensor([2, -1, 0, 2, 7, 1, 2, 0, -5, 10 ** 9], dtype=torch.int32)
    if many:                                          # further apart than a block looks at once
        slots = torch.cat([slots, torch.full((600,), -1, dtype=torch.int32), torch.tensor([1, 2, 2], dtype=torch.int32)])
    state, q, k, v, g = make(torch.float32, len(slots), 3, 1, 64, 64, 5)
    dev = state.cuda()
    out = decay_attention_step(dev, q.cuda(), k.cuda(), v.cuda(), g.cuda(), slots=slots.cuda())
    check(torch.float32, out, dev, *both(state, q, k, v, g, slots), times=6)
    assert not out[1].any() and not out[8].any() and not out[9].any() and torch.equal(dev[[3, 4]].cpu(), state[[3, 4]])
    assert torch.equal(decay_attention_step(state.cuda(), q.cuda(), k.cuda(), v.cuda(), g.cuda(), slots=slots.long().cuda()), out)


def test_a_pool_of_several_layers_and_strided_tokens():
    """States inside a larger cache, q, k and v as slices of a projection, addresses that no 16-byte access fits."""
    from ssd.uni.decay_attention import decay_attention_step
    state, q, k, v, g = (t.cuda() for t in make(torch.bfloat16, 4, 2, 2, 64, 32, 4))
    a = state.clone()
    want = decay_attention_step(a, q, k, v, g)
    cache = torch.zeros(4, 3, 2, 64, 32, device="cuda")
    cache[:, 1] = state
    wide_ = torch.cat([t.reshape(4, -1) for t in (q, k, v)] + [g], 1)
    q2, k2, v2, g2 = wide_.split([128, 128, 64, 2], 1)
    got = decay_attention_step(cache[:, 1], q2.unflatten(1, (2, 64)), k2.unflatten(1, (2, 64)), v2.unflatten(1, (2, 32)), g2)
    assert torch.equal(got, want) and torch.equal(cache[:, 1], a) and not cache[:, 0].any() and not cache[:, 2].any()
    odd = torch.zeros(state.numel() + 1, device="cuda")[1:].view_as(state).copy_(state)
    # one column a lane instead of four: the sums over rows are taken in another order
    assert off(decay_attention_step(odd, q, k, v, g), wide(want)) <= 2 * tolerances(torch.bfloat16, 64)[0]
    assert torch.equal(odd, a)


def test_offsets_past_32_bits():
    """States behind the first 2^31 elements of the pool."""
    from ssd.uni.decay_attention import decay_attention_step
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of device memory")
    h, n, p = 16, 128, 128
    pool = (1 << 31) // (h * n * p) + 3
    state, q, k, v, g = make(torch.bfloat16, 2, h, 1, n, p, 2)
    big = torch.zeros(pool, h, n, p, device="cuda")
    slots = torch.tensor([pool - 1, 1], dtype=torch.int32)
    big[slots.long().cuda()] = state.cuda()
    out = decay_attention_step(big, q.cuda(), k.cuda(), v.cuda(), g.cuda(), slots=slots.cuda())
    check(torch.bfloat16, out, big[slots.long().cuda()], *both(state, q, k, v, g, None))
    assert not big[2:pool - 1].any()


def test_single_tokens_go_on_from_a_prompt():
    """A prompt, then single tokens, against the whole sequence at once."""
    from ssd.uni.decay_attention import decay_attention, decay_attention_step
    from test_decay_attention_gpu import make as whole, tolerance
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, g, _ = whole(dtype, 2, 140, 4, 2, 64, 64, seed=4)
        want, final = decay_attention_reference(*(wide(t) for t in (q, k, v, g)))
        dev = [t.cuda() for t in (q, k, v, g)]
        out, state = decay_attention(*(t[:, :131] for t in dev), return_final_state=True)
        rows = [out] + [decay_attention_step(state, *(t[:, i] for t in dev))[:, None] for i in range(131, 140)]
        n = 140 + 128
        assert off(torch.cat(rows, 1), want) <= tolerance(dtype, n) and off(state, final) <= tolerance(dtype, n, "state")


def test_captured_step_and_version():
    from ssd.uni.decay_attention import decay_attention_step
    state, q, k, v, g = (t.cuda() for t in make(torch.bfloat16, 3, 2, 1, 64, 64, 3))
    a = state.clone()
    want = [decay_attention_step(a, q, k, v, g) for _ in range(3)][-1]
    version = state._version
    start, graph = state.clone(), torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = decay_attention_step(state, q, k, v, g)
    assert state._version > version
    state.copy_(start)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(state, a)
