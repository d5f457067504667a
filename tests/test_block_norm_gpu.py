"""The norms around a block against their definition in 64 bits.  Tolerances (2-norms): sums of squares or products over n = width
(rows for the gradients of weights, rows of one entry for a shared gate) terms, the hardware's sigmoid (8 2^-24) and a dozen
roundings: (n^(1/2) + 24) 2^-24; half a step more for results in 16 bits.  A gradient's fp32 part counts from what it would be if
the rows' sizes were constants, where that is more: the part that is subtracted for them may leave little of it."""
import pytest
import torch

from oracle.decay_oracle import block_norm_reference
from test_decay_attention_gpu import distance, off, wide

pytestmark = pytest.mark.gpu

CASES = [
    # shape, dtype, residual fp32, gate, activation, scale, post, pre, weights' dtype
    ((2, 33, 1024), torch.bfloat16, False, "full", "sigmoid", "vector", True, True, torch.float32),
    ((3, 50, 2048), torch.bfloat16, True, "row", None, 0.5, True, True, torch.float32),
    ((1, 1, 64), torch.bfloat16, False, None, None, 1.0, True, True, torch.bfloat16),
    ((7, 1), torch.float32, False, None, None, "vector", True, True, torch.float32),
    ((5, 9, 33), torch.float16, True, "full", "silu", 2.0, False, True, torch.float16),
    ((4, 1, 100), torch.float32, False, "row", "silu", "vector", True, False, torch.float32),
    ((3, 11, 264), torch.float16, False, "row", "sigmoid", "vector", False, True, torch.float32),
    ((2, 5, 8192), torch.bfloat16, True, "full", "silu", "vector", True, True, torch.float32),
    ((2, 3, 8191), torch.bfloat16, False, "all", "sigmoid", "vector", True, True, torch.float32),
    ((700, 4104), torch.float32, False, "full", None, 1.0, True, True, torch.float32),
    ((2, 300, 96), torch.bfloat16, False, None, None, 1.0, False, False, torch.float32),
    ((40, 77, 512), torch.bfloat16, False, "row", "sigmoid", "vector", True, True, torch.float32),
]


def make(case, seed=0):
    shape, dtype, wide_residual, gate, act, scale, post, pre, wd = case
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    d = shape[-1]
    rows = {"full": shape, "row": (shape[0],) + (1,) * (len(shape) - 2) + (d,), "all": (1,) * (len(shape) - 1) + (d,)}
    rdt = torch.float32 if wide_residual else dtype
    t = dict(x=(2 * r(*shape)).to(dtype), residual=r(*shape).to(rdt), gate=r(*rows[gate]).to(dtype) if gate else None,
             scale=(0.5 + 0.3 * r(d)).to(wd) if scale == "vector" else scale, post_weight=(1 + 0.2 * r(d)).to(wd) if post else None,
             pre_weight=(1 + 0.2 * r(d)).to(wd) if pre else None)
    return t, act, (r(*shape).to(rdt), r(*shape).to(dtype) if pre else None)


def tol(dtype, n):
    return (n ** 0.5 + 24) * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("case", CASES, ids=["x".join(map(str, c[0])) for c in CASES])
def test_forward_and_backward_match_the_definition(case):
    from ssd.block_norm import block_norm
    t, act, (dout, dnormed) = make(case, seed=sum(case[0]))
    tensor = lambda v: isinstance(v, torch.Tensor)
    dev = {n: v.cuda().requires_grad_(True) if tensor(v) else v for n, v in t.items()}
    ref = {n: wide(v).requires_grad_(True) if tensor(v) else v for n, v in t.items()}
    got, want = block_norm(**dev, gate_activation=act), block_norm_reference(**ref, gate_activation=act)
    if dnormed is None:
        got, want = (got,), (want,)
    d = case[0][-1]
    for a, b, like in zip(got, want, (t["residual"], t["x"])):
        assert a.dtype == like.dtype and off(a, b) <= tol(a.dtype, d), off(a, b)
    with torch.no_grad():                             # the same numbers without a graph
        again = block_norm(**dev, gate_activation=act)
    assert all(torch.equal(a, b) for a, b in zip(again if dnormed is not None else (again,), got))
    names = [n for n, v in dev.items() if tensor(v)]
    gos = [dout, dnormed][:len(got)]
    grads = torch.autograd.grad(got, [dev[n] for n in names], [g.cuda() for g in gos])
    exp = torch.autograd.grad(want, [ref[n] for n in names], [wide(g) for g in gos])
    fixed = block_norm_reference(**ref, gate_activation=act, fixed=True)
    sizes = torch.autograd.grad(fixed, [ref[n] for n in names], [wide(g) for g in gos])
    rows = t["x"].numel() // d
    for n, a, b, z in zip(names, grads, exp, sizes):
        terms = rows + d if t[n].dim() == 1 or t[n].numel() < t["x"].numel() else 2 * d
        most = tol(torch.float32, terms) * max(float(b.norm()), float(z.norm())) + tol(a.dtype, terms) * float(b.norm())
        assert a.dtype == t[n].dtype and distance(a, b) <= most, (n, distance(a, b), most)


def test_only_some_gradients_are_wanted_or_given():
    from ssd.block_norm import block_norm
    t, act, (dout, dnormed) = make(CASES[0], seed=3)
    dev = {n: v.cuda() for n, v in t.items()}
    for n in ("x", "scale"):
        dev[n].requires_grad_(True)
    ref = {n: wide(v).requires_grad_(n in ("x", "scale")) for n, v in t.items()}
    got, want = block_norm(**dev, gate_activation=act), block_norm_reference(**ref, gate_activation=act)
    for i, go in ((0, dout), (1, dnormed)):           # one of the two results is used
        grads = torch.autograd.grad(got[i], [dev["x"], dev["scale"]], go.cuda(), retain_graph=True)
        exp = torch.autograd.grad(want[i], [ref["x"], ref["scale"]], wide(go), retain_graph=True)
        for a, b in zip(grads, exp):
            assert off(a, b) <= tol(a.dtype, 66 + 1024)


def test_strided_rows_and_addresses():
    """x, residual and gate as slices of wider rows; an address that no 16-byte access fits."""
    from ssd.block_norm import block_norm
    t, act, (dout, dnormed) = make(CASES[0], seed=1)
    dev = {n: v.cuda() for n, v in t.items()}
    want = block_norm(**dev, gate_activation=act)
    both = torch.cat([dev["x"], dev["gate"], dev["residual"]], -1)
    x, gate, residual = both.split(1024, -1)
    got = block_norm(x, residual, gate, dev["scale"], dev["post_weight"], dev["pre_weight"], act)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.empty(dev["x"].numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(dev["x"]).copy_(dev["x"])
    for a, b in zip(block_norm(x, residual, gate, dev["scale"], dev["post_weight"], dev["pre_weight"], act), want):
        assert off(a, wide(b)) <= 2 * tol(torch.bfloat16, 1024)
    x = x.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
    out, _ = block_norm(x, residual, gate, dev["scale"], dev["post_weight"], dev["pre_weight"], act)
    assert torch.equal(out, want[0]) or off(out, wide(want[0])) <= 2 * tol(torch.bfloat16, 1024)
    assert torch.autograd.grad(out.float().sum(), x)[0].shape == x.shape


def test_rows_of_infinities_stay_alone_and_nothing_to_do():
    from ssd.block_norm import block_norm
    t, act, _ = make(CASES[1], seed=2)
    dev = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in t.items()}
    want = block_norm(**dev, gate_activation=act)
    dev["x"][1, 7] = float("nan")
    dev["residual"][2, 9] = float("inf")
    got = block_norm(**dev, gate_activation=act)
    keep = torch.ones(3, 50, dtype=torch.bool)
    keep[1, 7] = keep[2, 9] = False
    assert all(torch.equal(a[keep.cuda()], b[keep.cuda()]) for a, b in zip(got, want))
    zero = torch.zeros(2, 4, 64, device="cuda")       # eps keeps a row of zeros finite
    w = torch.ones(64, device="cuda")
    x = zero.clone().requires_grad_(True)
    out, normed = block_norm(x, zero, post_weight=w, pre_weight=w)
    assert not out.any() and not normed.any() and bool(torch.isfinite(torch.autograd.grad(normed.sum(), x)[0]).all())
    empty = torch.zeros(0, 4, 64, device="cuda", requires_grad=True)
    w.requires_grad_(True)
    out, normed = block_norm(empty, empty, post_weight=w, pre_weight=w)
    assert out.shape == empty.shape and not torch.autograd.grad(normed.sum(), w)[0].any()


def test_same_bits_in_a_graph_and_on_a_stream():
    from ssd.block_norm import block_norm
    t, act, gos = make(CASES[11], seed=4)
    dev = {n: v.cuda().requires_grad_(True) for n, v in t.items()}
    names = list(dev)

    def both():
        got = block_norm(**dev, gate_activation=act)
        return [*(a.detach() for a in got), *torch.autograd.grad(got, [dev[n] for n in names], [g.cuda() for g in gos])]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=side):
        out = block_norm(**dev, gate_activation=act)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
