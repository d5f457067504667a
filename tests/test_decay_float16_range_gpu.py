"""float16 tensors whose results are in the type's range while what lies between is not: states, weighted pairs or their gradients beyond
65504.  Such a head of a sequence is computed in float32 throughout; the others keep their bits.

Tolerances (2-norms) are test_decay_attention_gpu's for fp16: a pass in which nothing leaves the range stays on the tensor cores (a single chunk's
backward pass has no state but the initial one, for instance), and what is done again is nearer - fp32's part of the same, with half a step for the
result's rounding where that has three or five; 2^-25 absolute where a result is below the normal numbers.
"""
import pytest
import torch

from oracle.decay_oracle import decay_attention_reference
from test_decay_attention_gpu import bound, make, wide

pytestmark = pytest.mark.gpu
F16 = torch.float16
# sizes of q, k, v, dout, initial state, its gradient; what leaves the range
KINDS = {
    "states": (2e-3, 300, 300, 1e-3, 1, 1e-3),
    "pairs": (400, 400, 0.01, 0.01, 1, 1e-3),
    "pairs-of-gradients": (0.01, 0.01, 400, 400, 1, 1e-3),
    "state-in": (1e-3, 0.1, 0.1, 1e-3, 1e6, 1e-3),
    "states-of-gradients": (300, 1e-3, 1e-3, 300, 1e-3, 1e-3),
    "gradient-in": (0.1, 1e-3, 1e-3, 0.1, 1, 1e6),
}


def tensors(kind, b, L, h, hk, n, p, decay="token", seqs=None, seed=1):
    q, k, v, g, init = make(F16, b, L, h, hk, n, p, decay, True, seqs, seed, torch.float32)
    gen = torch.Generator().manual_seed(seed)
    dout, dfinal = torch.randn(b, L, h, p, generator=gen), torch.randn(init.shape, generator=gen)
    s = KINDS[kind]
    t = [(x.float() * f).to(F16) for x, f in zip((q, k, v, dout), s)]
    return t[0], t[1], t[2], g, init * s[4], t[3], dfinal * s[5]


def results(q, k, v, g, init, dout, dfinal, bounds=None):
    from ssd.uni.decay_attention import decay_attention
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g, init)]
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    out, final = decay_attention(*leaves[:4], initial_state=leaves[4], return_final_state=True, cu_seqlens=cu)
    return [out, final, *torch.autograd.grad([out, final], leaves, [dout.cuda(), dfinal.cuda()])]


def definition(size, q, k, v, g, init, dout, dfinal, bounds=None):
    refs = [(wide(t) if i == 3 else size(wide(t))).requires_grad_(True) for i, t in enumerate((q, k, v, g, init))]
    out, final = decay_attention_reference(*refs[:4], initial_state=refs[4], bounds=bounds)
    return [out, final, *torch.autograd.grad([out, final], refs, [size(wide(dout)), size(wide(dfinal))])]


def check(case, bounds=None):
    got, n = results(*case, bounds), case[0].shape[1] + case[0].shape[3] + case[2].shape[3]
    want, sizes = definition(lambda t: t, *case, bounds), definition(torch.abs, *case, bounds)
    for name, a, w, s in zip(("out", "final", "dq", "dk", "dv", "dg", "dinitial"), got, want, sizes):
        w, s = w.detach(), s.detach()
        beyond = w.abs() > 66000 if a.dtype == F16 else torch.zeros_like(w, dtype=torch.bool)   # where the definition's result itself is out of range
        a = a.detach().double().cpu()
        assert bool((a.isinf() == beyond)[(w.abs() - 65500).abs() > 500].all()) and not a.isnan().any(), name
        assert torch.equal(a[beyond].sign(), w[beyond].sign()) and float(beyond.double().mean()) < 1e-3, name
        if beyond.any():                              # what is near the border may lie on either side of it
            a, w = a.masked_fill(w.abs() > 65000, 0), w.masked_fill(w.abs() > 65000, 0)
        kind = {"final": "state", "dinitial": "state", "dg": "decay"}.get(name, "out")
        off, most = float((a - w).norm()), bound(F16, n, w, s, kind) + 2.0 ** -25 * w.numel() ** 0.5
        print(name, "%.2e / %.2e of %.2e" % (off, most, float(w.norm())))
        assert off <= most, name


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [(1, 60, 2, 1, 64, 64), (2, 300, 4, 2, 64, 64), (1, 260, 3, 3, 128, 80), (1, 2100, 1, 1, 64, 64)], ids=str)
def test_out_of_range_between(size, kind):
    check(tensors(kind, *size))


@pytest.mark.parametrize("kind", KINDS)
def test_one_decay_for_each_head(kind):
    check(tensors(kind, 2, 200, 4, 1, 64, 64, "head"))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bounds", [[0, 5, 6, 6, 134, 390, 400], [3, 131, 131, 259, 300]], ids=str)
def test_packed(kind, bounds):
    case = tensors(kind, 1, bounds[-1] + 7, 4, 2, 64, 64, seqs=len(bounds) - 1)
    check(case, bounds)


@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("kind", KINDS)
def test_only_one_sequence_and_head(kind, decay):
    """The others' bits are what they are without it."""
    bounds = [2, 100, 250, 400]
    small = tensors("states", 1, 405, 4, 4, 64, 64, decay, 3)
    ordinary = [t / f if t is not small[3] else t for t, f in zip(small, (2e-3, 300, 300, 1, 1, 1e-3, 1e-3))]
    ordinary = [t.to(F16) if i in (0, 1, 2, 5) else t for i, t in enumerate(ordinary)]
    large = [t.clone() for t in ordinary]
    for a, f in zip((0, 1, 2, 5, 4, 6), KINDS[kind]):
        part = large[a][:, 100:250, 1] if a not in (4, 6) else large[a][1, 1]
        part.copy_((part.float() * f).to(part.dtype))
    want, got = results(*ordinary, bounds), results(*large, bounds)
    assert all(bool(t.isfinite().all()) for t in got)
    rest = [0, 2, 3]
    for i, (a, b) in enumerate(zip(got, want)):
        if i in (1, 6):
            assert torch.equal(a[:, rest], b[:, rest]) and torch.equal(a[[0, 2]], b[[0, 2]]), i
        elif a.dim() == 1:
            assert torch.equal(a[rest], b[rest]), i
        else:
            assert torch.equal(a[:, :, rest], b[:, :, rest]) and torch.equal(a[:, :100], b[:, :100]) and torch.equal(a[:, 250:], b[:, 250:]), i
    exact, sizes = definition(lambda t: t, *large, bounds), definition(torch.abs, *large, bounds)
    for i, part, dtype in ((0, (slice(None), slice(100, 250), 1), F16), (1, (1, 1), torch.float32)):
        w = exact[i][part].detach()
        assert float((got[i][part].detach().double().cpu() - w).norm()) <= bound(dtype, 150 + 128, w, sizes[i][part])


def test_only_the_final_state():
    """Decays above 0, which let the weights of a chunk's rows grow: nothing but the state behind it leaves the range."""
    from ssd.uni.decay_attention import decay_attention
    q, k, v, g, _ = make(F16, 2, 100, 2, 1, 64, 64, seed=1, g_dtype=torch.float32)
    q, v, g = torch.zeros_like(q), (v.float() * 300).to(F16), torch.full_like(g, 0.06)
    out, final = decay_attention(*(t.cuda() for t in (q, k, v, g)), return_final_state=True)
    want = decay_attention_reference(*(wide(t) for t in (q, k, v, g)))[1]
    sizes = decay_attention_reference(*(wide(t).abs() for t in (q, k, v)), wide(g))[1]
    assert not out.any() and float((final.double().cpu() - want).norm()) <= bound(torch.float32, 228, want, sizes)


def test_a_captured_call_on_changing_inputs():
    """What is out of range may change from replay to replay."""
    from ssd.uni import decay_attention as module
    kept, module.CHECK_STATUS = module.CHECK_STATUS, False
    try:
        case = [t.cuda() for t in tensors("states", 2, 300, 4, 2, 64, 64)[:4]]
        ordinary = [t / f if i < 3 else t for i, (t, f) in enumerate(zip(case, (2e-3, 300, 300, 1)))]
        dout = torch.randn(2, 300, 4, 64, device="cuda").to(F16) * 1e-3
        leaves = [t.clone().requires_grad_(True) for t in case]

        def both():
            out, final = module.decay_attention(*leaves, return_final_state=True)
            return [out, final, *torch.autograd.grad(out, leaves, dout)]

        want = []
        for inputs in (case, ordinary):
            with torch.no_grad():
                for a, b in zip(leaves, inputs):
                    a.copy_(b)
            want.append([t.detach().clone() for t in both()])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        with torch.cuda.stream(side):
            both()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = both()
        for which in (0, 1, 1, 0, 1):
            with torch.no_grad():
                for a, b in zip(leaves, (case, ordinary)[which]):
                    a.detach().copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert all(bool(a.isfinite().all()) and torch.equal(a, b) for a, b in zip(got, want[which])), which
    finally:
        module.CHECK_STATUS = kept


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_inputs_that_are_no_numbers(value):
    """They reach what the definition lets them reach: a row of v the outputs from its token on, a row of dout the gradients up to it."""
    L, at, n = 300, 150, 300 + 128
    q, k, v, g, _ = make(F16, 1, L, 2, 2, 64, 64, seed=4, g_dtype=torch.float32)
    dout = torch.randn(v.shape, generator=torch.Generator().manual_seed(3)).to(F16)
    refs = [wide(t).requires_grad_(True) for t in (q, k, v, g)]
    o = decay_attention_reference(*refs)[0]
    exp = torch.autograd.grad(o, refs, wide(dout))
    o = o.detach()
    sizes = [wide(t).abs() if i < 3 else wide(t) for i, t in enumerate((q, k, v, g))]
    sizes = [t.requires_grad_(True) for t in sizes]
    so = decay_attention_reference(*sizes)[0]
    sg = torch.autograd.grad(so, sizes, wide(dout).abs())
    from ssd.uni.decay_attention import decay_attention
    bad = v.clone()
    bad[:, at, 0] = value
    out = decay_attention(*(t.cuda() for t in (q, k, bad, g))).double().cpu()
    assert not out[:, at:, 0].isfinite().any()
    assert float((out[:, :at] - o[:, :at]).norm()) <= bound(F16, n, o[:, :at], so[:, :at])
    assert float((out[:, :, 1] - o[:, :, 1]).norm()) <= bound(F16, n, o[:, :, 1], so[:, :, 1])
    bad = dout.clone()
    bad[:, at, 0] = value
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g)]
    grads = torch.autograd.grad(decay_attention(*leaves), leaves, bad.cuda())
    for i, (a, w, s) in enumerate(zip(grads, exp, sg)):
        a, kind = a.double().cpu(), "decay" if i == 3 else "out"
        assert not a[:, at, 0].isfinite().any()
        assert float((a[:, at + 1:] - w[:, at + 1:]).norm()) <= bound(F16, n, w[:, at + 1:], s[:, at + 1:], kind), i
        assert float((a[:, :, 1] - w[:, :, 1]).norm()) <= bound(F16, n, w[:, :, 1], s[:, :, 1], kind), i
