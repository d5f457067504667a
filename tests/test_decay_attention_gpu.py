"""The causal decay attention against its definition, token by token in 64 bits (oracle/decay_oracle.py).

Tolerances, for the 2-norm of the difference, with A what the definition gives for the inputs' absolute values (the sum of the
terms' sizes), n = seqlen + kdim + vdim, u = 2^-24 and h = eps / 2 (half a step) of a 16-bit type:
  fp32      each of n roundings in a row is off by at most u A and as often one way as the other: (n^(1/2) + 8) u |A|
  16 bits   and h for the result's own rounding, and h for each 16-bit operand that the tensor cores are given in place of a 32-bit
            one: the weighted pair and the state for outputs, dq, dk and dv (3 h); the decay's gradient sums products of two such
            results and crosses two states (5 h).  These errors are of single terms, of mixed signs: of the larger of |result| and
            |A| / n^(1/2)
            (On CUDA cores a token's own pair is subtracted from itself on the way to dg: it counts in dg's A.)
  states    as fp32, whatever the inputs are; on the tensor cores a term is the sum of two 16-bit halves, off by at most
            eps^2 / 4 = 2^-16 of itself in bf16
Where there is no A at hand, |A| = 1.25 n^(1/2) |result|, as for terms of random signs: 2 n u of the result covers fp32's part.
"""
import pytest
import torch

from oracle.decay_oracle import decay_attention_reference

pytestmark = pytest.mark.gpu


def off(got, want):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    norm = float(want.norm())
    return float((got - want).norm()) / norm if norm else float(got.norm())


def tolerance(dtype, n, kind="out"):
    """Of the result's 2-norm."""
    fp32 = 2 * n * 2.0 ** -24
    if kind == "state":
        return fp32 + (0 if dtype == torch.float32 else 2.0 ** -16)
    return fp32 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (5 if kind == "decay" else 3))


def bound(dtype, n, want, sizes, kind="out"):
    """Of the difference's 2-norm; `sizes`: A."""
    a = float(sizes.detach().norm())
    typical = max(float(want.detach().norm()), a / n ** 0.5)
    fp32 = (n ** 0.5 + 8) * 2.0 ** -24 * a
    if kind == "state":
        return fp32 + (0 if dtype == torch.float32 else 2.0 ** -16 * typical)
    return fp32 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (5 if kind == "decay" else 3) * typical)


def distance(got, want):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    return float((got - want).norm())


def make(dtype, b, L, h, hk, n, p, decay="token", initial=False, seqs=None, seed=0, g_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    q, k, v = r(b, L, hk, n).to(dtype), r(b, L, hk, n).to(dtype), r(b, L, h, p).to(dtype)
    rate = torch.exp(torch.rand(h, generator=gen) * 2.7)
    g = -rate * torch.nn.functional.softplus(r(b, L, h) - 3) if decay == "token" else -rate / 50
    g = g.to(g_dtype or (dtype if decay == "token" else torch.float32))
    init = r(seqs or b, h, n, p) if initial else None
    return q, k, v, g, init


def wide(t):
    return None if t is None else t.detach().double().cpu()


def check(dtype, tensors, dout=None, dfinal=None, bounds=None, scale=None, cu=None, strided=False):
    """Forward, and with dout backward, against the oracle."""
    from ssd.uni.decay_attention import decay_attention
    dev = [None if t is None else t.cuda() for t in tensors]
    if strided:                                       # slices of one wider tensor, as a projection's output is split
        q, k, v, g = dev[:4]
        b, L = q.shape[:2]
        parts = [t.reshape(b, L, -1) for t in (q, k, v)]
        both = torch.cat(parts + [torch.zeros(b, L, 8, dtype=q.dtype, device="cuda")], -1)
        views = both.split([t.shape[-1] for t in parts] + [8], -1)
        dev[:3] = [w.unflatten(-1, t.shape[2:]) for w, t in zip(views, (q, k, v))]
    leaves = [t.detach().requires_grad_(dout is not None) if t is not None else None for t in dev]
    if cu is None and bounds is not None:
        cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    out, final = decay_attention(*leaves[:4], scale=scale, initial_state=leaves[4], return_final_state=True, cu_seqlens=cu)
    had = [i for i, t in enumerate(leaves) if t is not None]
    got = []
    if dout is not None:
        outs, gos = ([out], [dout.cuda()]) if dfinal is None else ([out, final], [dout.cuda(), dfinal.cuda()])
        got = torch.autograd.grad(outs, [leaves[i] for i in had], gos)

    def oracle(size):
        ref = [None if t is None else size(wide(t)) if i != 3 else wide(t) for i, t in enumerate(tensors)]
        ref = [None if t is None else t.requires_grad_(dout is not None) for t in ref]
        o, f = decay_attention_reference(*ref[:4], scale=scale, initial_state=ref[4], bounds=bounds)
        if dout is None:
            return [o, f]
        outs, gos = ([o], [size(wide(dout))]) if dfinal is None else ([o, f], [size(wide(dout)), size(wide(dfinal))])
        g = torch.autograd.grad(outs, [ref[i] for i in had], gos, allow_unused=True)
        return [o, f] + [torch.zeros_like(ref[i]) if t is None else t for i, t in zip(had, g)]

    want, sizes = oracle(lambda t: t), oracle(torch.abs)
    q, k, v = tensors[:3]
    if dout is not None:
        heads = torch.arange(v.shape[2]) * q.shape[2] // v.shape[2]
        own = (wide(q) * wide(k)).abs().sum(-1)[..., heads] * (wide(v) * wide(dout)).abs().sum(-1) * (q.shape[3] ** -0.5 if scale is None else scale)
        sizes[2 + had.index(3)] = sizes[2 + had.index(3)] + (own if tensors[3].dim() == 3 else own.sum((0, 1)))
    n = q.shape[1] + q.shape[3] + v.shape[3]
    assert out.dtype == v.dtype and final.dtype == torch.float32 and all(t.dtype == leaves[i].dtype for i, t in zip(had, got))
    names = ["out", "final"] + [["dq", "dk", "dv", "dg", "dinitial"][i] for i in had]
    kinds = {"final": "state", "dinitial": "state", "dg": "decay"}
    errors = {m: (distance(a, w), bound(dtype, n, w, z, kinds.get(m, "out"))) for m, a, w, z in zip(names, [out, final, *got], want, sizes)}
    print({m: "%.2e / %.2e" % e for m, e in errors.items()})
    for name, (e, most) in errors.items():
        assert e <= most, (name, e, most, errors)


SIZES = [
    # batch, seqlen, heads, kv_heads, kdim, vdim, decay, initial
    (1, 1, 1, 1, 1, 1, "token", False),
    (2, 1, 4, 2, 64, 64, "token", True),
    (1, 2, 3, 1, 7, 5, "head", True),
    (2, 65, 6, 3, 16, 32, "token", False),
    (1, 127, 2, 2, 64, 64, "token", True),
    (1, 128, 4, 1, 128, 64, "token", False),
    (2, 129, 2, 1, 128, 128, "head", True),
    (1, 300, 4, 4, 80, 48, "token", True),
    (1, 257, 2, 1, 24, 130, "token", False),
    (1, 70, 2, 2, 256, 256, "token", True),
    (3, 520, 3, 1, 64, 128, "token", True),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES, ids=["x".join(map(str, s[:6])) for s in SIZES])
def test_forward_and_backward_match_the_definition(dtype, size):
    b, L, h, hk, n, p, decay, initial = size
    tensors = make(dtype, b, L, h, hk, n, p, decay, initial, seed=L + n)
    gen = torch.Generator().manual_seed(5)
    dout = torch.randn(b, L, h, p, generator=gen).to(dtype)
    check(dtype, tensors, dout, torch.randn(b, h, n, p, generator=gen) if initial else None)


@pytest.mark.parametrize("size", [(1, 3001, 2, 1, 64, 64), (1, 2100, 1, 1, 128, 80)], ids=str)
def test_long_rows_in_several_segments(size):
    """Few heads and many chunks: the states of a row are walked in segments of several chunks each."""
    b, L, h, hk, n, p = size
    gen = torch.Generator().manual_seed(3)
    q, k, v, g, init = make(torch.bfloat16, b, L, h, hk, n, p, initial=True, seed=L)
    g = (g.float() / 50).to(g.dtype)                  # a state outlives its segment
    check(torch.bfloat16, (q, k, v, g, init), torch.randn(b, L, h, p, generator=gen).to(torch.bfloat16), torch.randn(b, h, n, p, generator=gen))
    bounds = [5, 1300, 1301, 2000, L]
    init = torch.randn(4, h, n, p, generator=gen)
    check(torch.bfloat16, (q, k, v, g, init), torch.randn(b, L, h, p, generator=gen).to(torch.bfloat16), torch.randn(4, h, n, p, generator=gen), bounds)


PACKED = [[0, 5, 6, 6, 134, 390, 400], [3, 131, 131, 259, 300], [0, 0, 0], [0, 1, 2, 3, 4], [10, 700]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("bounds", PACKED, ids=[str(i) for i in range(len(PACKED))])
def test_packed_sequences(dtype, bounds):
    """Empty sequences, ones that end inside a tile, tokens before the first and behind the last."""
    L, seqs = bounds[-1] + 7, len(bounds) - 1
    tensors = make(dtype, 1, L, 4, 2, 64, 64, initial=True, seqs=seqs, seed=len(bounds))
    gen = torch.Generator().manual_seed(9)
    check(dtype, tensors, torch.randn(1, L, 4, 64, generator=gen).to(dtype), torch.randn(seqs, 4, 64, 64, generator=gen), bounds)


def test_packed_boundaries_that_make_no_sense():
    """Boundaries outside the tokens or running backwards are taken as the nearest that are not; nothing is read outside."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(torch.bfloat16, 1, 200, 2, 1, 64, 64))
    bad = torch.tensor([-50, 40, 20, 90, 10 ** 9, 300], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 40, 40, 90, 200, 200], dtype=torch.int32, device="cuda")
    a = decay_attention(q, k, v, g, return_final_state=True, cu_seqlens=bad)
    b = decay_attention(q, k, v, g, return_final_state=True, cu_seqlens=good.long())
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_slices_of_a_projection(dtype):
    tensors = make(dtype, 2, 150, 4, 2, 64, 64, seed=3)
    check(dtype, tensors, torch.randn(2, 150, 4, 64, generator=torch.Generator().manual_seed(1)).to(dtype), strided=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_odd_strides_and_offsets(dtype):
    """An inner stride of two, an address that no 16-byte access fits, a batch that repeats one row."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(dtype, 2, 140, 2, 2, 64, 64, seed=4))
    want = decay_attention(q, k, v, g)
    q2 = torch.stack([q, q], -1)[..., 0]
    k2 = torch.empty(k.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(k).copy_(k)
    assert torch.equal(decay_attention(q2, k2, v, g.transpose(1, 2).contiguous().transpose(1, 2)), want)
    one = decay_attention(q[:1], k[:1], v[:1], g[:1])
    many = decay_attention(q[:1].expand(3, -1, -1, -1), k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), g[:1].expand(3, -1, -1))
    assert all(torch.equal(many[i], one[0]) for i in range(3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_decay_of_minus_infinity_empties_the_state(dtype):
    """What came before is gone, and every gradient that crosses is zero."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = make(dtype, 1, 300, 2, 1, 64, 64, seed=8)
    for cut in (130, 200):
        g[:, cut] = -float("inf")
    dout = torch.randn(1, 300, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    dev = [t.cuda().requires_grad_(True) for t in (q, k, v, g)]
    out = decay_attention(*dev)
    grads = torch.autograd.grad(out, dev, dout.cuda())
    n = 300 + 128
    for a, z in ((0, 130), (130, 200), (200, 300)):
        part = [t[:, a:z].double().requires_grad_(True) for t in (q, k, v, g)]
        with torch.no_grad():
            part[3][:, 0] = 0 if a == 0 else -1.0             # multiplies an empty state
        want, _ = decay_attention_reference(*part)
        assert off(out[:, a:z], want) <= tolerance(dtype, n)
        exp = torch.autograd.grad(want, part, dout[:, a:z].double())
        for i, (got, e) in enumerate(zip(grads, exp)):
            assert off(got[:, a:z], e) <= tolerance(dtype, n, "decay" if i == 3 else "out"), (i, a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_strong_and_no_decay(dtype):
    """From no decay at all to states that are gone at the next token."""
    for g0 in (0.0, -0.001, -30.0, -200.0):
        q, k, v, g, _ = make(dtype, 1, 280, 2, 1, 64, 64, decay="head", seed=2)
        g = torch.full_like(g, g0)
        check(dtype, (q, k, v, g, None), torch.randn(1, 280, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype))


def test_infinities_of_one_sequence_stay_there():
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(torch.bfloat16, 1, 400, 2, 2, 64, 64, seed=6))
    cu = torch.tensor([0, 100, 250, 400], dtype=torch.int32, device="cuda")
    want = decay_attention(q, k, v, g, return_final_state=True, cu_seqlens=cu)
    for t, value in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        t[:, 100:250] = value
    got = decay_attention(q, k, v, g, return_final_state=True, cu_seqlens=cu)
    for a, z, i in ((0, 100, 0), (250, 400, 2)):
        assert torch.equal(got[0][:, a:z], want[0][:, a:z]) and torch.equal(got[1][i], want[1][i])
    dout = torch.ones_like(v)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    grads = torch.autograd.grad(decay_attention(*leaves, cu_seqlens=cu), leaves, dout)
    assert all(bool(torch.isfinite(t[:, a:z]).all()) for t in grads for a, z in ((0, 100), (250, 400)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_sequence_in_two_calls(dtype):
    """The final state of one call is the initial state of the next, at any place, and gradients go through both."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(dtype, 2, 333, 4, 2, 64, 64, seed=7))
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    whole, final = decay_attention(*leaves, return_final_state=True)
    dout, dfinal = torch.randn_like(whole), torch.randn_like(final)
    grads = torch.autograd.grad([whole, final], leaves, [dout, dfinal])
    n = 333 + 128
    for cut in (1, 128, 200, 332):
        o1, s1 = decay_attention(*(t[:, :cut] for t in leaves), return_final_state=True)
        o2, s2 = decay_attention(*(t[:, cut:] for t in leaves), initial_state=s1, return_final_state=True)
        both = torch.cat([o1, o2], 1)
        assert off(both, wide(whole)) <= 2 * tolerance(dtype, n) and off(s2, wide(final)) <= 2 * tolerance(dtype, n, "state")
        again = torch.autograd.grad([both, s2], leaves, [dout, dfinal])
        for i, (a, b) in enumerate(zip(again, grads)):
            assert off(a, wide(b)) <= 2 * tolerance(dtype, n, "decay" if i == 3 else "out"), (cut, i)


def test_gradients_against_differences():
    """fp32: the slope along a direction, from two forward passes half a step apart on either side.  With a step of 2^-6 the
    difference's own error is of the step's square (2^-12) and of the sums' rounding over the step (n 2^-24 / 2^-6): below 2^-9
    of the larger of the slope and the norms' product over the root of the size, here with n = 200 + 64."""
    from ssd.uni.decay_attention import decay_attention
    gen = torch.Generator().manual_seed(11)
    q, k, v, g, init = (t.cuda() for t in make(torch.float32, 1, 200, 2, 1, 32, 32, initial=True, seed=1))
    dout = torch.randn(1, 200, 2, 32, generator=gen).cuda()
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, init)]
    grads = torch.autograd.grad(decay_attention(*leaves[:4], initial_state=init), leaves, dout)
    h = 2.0 ** -6
    for i in range(5):
        d = torch.randn(leaves[i].shape, generator=gen).cuda() * (0.1 if i == 3 else 1)
        with torch.no_grad():
            ends = []
            for sign in (0.5, -0.5):
                moved = [t + sign * h * d if j == i else t for j, t in enumerate(leaves)]
                ends.append(float((decay_attention(*moved[:4], initial_state=moved[4]).double() * dout).sum()))
        slope, want = (ends[0] - ends[1]) / h, float((grads[i].double() * d).sum())
        size = max(abs(want), float(grads[i].double().norm() * d.double().norm()) / grads[i].numel() ** 0.5)
        assert abs(slope - want) <= 2.0 ** -9 * size, (i, slope, want, size)


def test_nothing_to_do():
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, init = (t.cuda() for t in make(torch.bfloat16, 2, 4, 2, 1, 64, 64, initial=True))
    leaves = [t.requires_grad_(True) for t in (q[:, :0], k[:, :0], v[:, :0], g[:, :0], init)]
    out, final = decay_attention(*leaves[:4], initial_state=init, return_final_state=True)
    assert out.shape == (2, 0, 2, 64) and torch.equal(final, init)
    grads = torch.autograd.grad(final.sum(), leaves)
    assert torch.equal(grads[4], torch.ones_like(init)) and grads[0].shape == leaves[0].shape
    out, final = decay_attention(q[:0], k[:0], v[:0], g[:0], return_final_state=True)
    assert out.shape[0] == 0 and final.shape[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_same_bits_on_any_stream_in_a_graph_and_again(dtype):
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(dtype, 2, 700, 4, 1, 64, 64, seed=5))
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    dout = torch.randn_like(v)

    def both():
        out, final = decay_attention(*leaves, return_final_state=True)
        return [out.detach(), final.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = both()
    assert all(torch.equal(a, b) for a, b in zip(both(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():                             # two captured calls, replayed in turn, with new inputs
        with torch.cuda.stream(side):
            decay_attention(q, k, v, g)
        side.synchronize()
        graphs = []
        from ssd.bi import ssd_combined                # the status word's synchronising read cannot be captured
        import ssd.uni.decay_attention as module
        kept, module.CHECK_STATUS = module.CHECK_STATUS, False
        try:
            for _ in range(2):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    o = decay_attention(q, k, v, g, return_final_state=True)
                graphs.append((graph, o))
        finally:
            module.CHECK_STATUS = kept
        assert ssd_combined.CHECK_STATUS == kept
        for (graph, o) in graphs + graphs[::-1]:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
        v.neg_()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1][0], -want[0])


def test_a_row_does_not_depend_on_the_others():
    """A sequence's results are the same alone, in a batch and packed (decays, gradients and states included)."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(torch.bfloat16, 3, 200, 4, 2, 128, 64, seed=12))
    out, final = decay_attention(q, k, v, g, return_final_state=True)
    for i in range(3):
        o, f = decay_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], g[i:i + 1], return_final_state=True)
        assert torch.equal(o[0], out[i]) and torch.equal(f[0], final[i])


def test_a_thread_that_has_made_no_cuda_call():
    """With all memory at hand, the first call of a new thread that reaches CUDA is the building of a tensor map."""
    import threading
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda() for t in make(torch.bfloat16, 1, 200, 2, 1, 64, 64))
    with torch.no_grad():
        decay_attention(q, k, v, g)
        torch.cuda.synchronize()
        got = []
        thread = threading.Thread(target=lambda: got.append(decay_attention(q, k, v, g)))
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert got and torch.equal(got[0], decay_attention(q, k, v, g))


def test_no_second_derivative():
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = (None if t is None else t.cuda().requires_grad_(True) for t in make(torch.float32, 1, 8, 1, 1, 8, 8))
    out = decay_attention(q, k, v, g)
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.grad(out.sum(), q, create_graph=True)
