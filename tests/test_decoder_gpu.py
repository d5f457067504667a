"""The causal mixer, the residual block and the decoder: a training step against the definitions in 64 bits, prompts and single tokens
against the whole sequence, a block around the bidirectional layer.

Tolerances (of 2-norms).  fp32: each of two blocks is a chain of sums over at most n = 256 + 300 + 64 terms, 2 n 2^-24 of its result as in
test_decay_attention_gpu.py; products with the projections come from the library's fp32 GEMM (as exact); the chain's length (gate,
mixer, two norms, twice) multiplies that by 16.  bf16, a sequence at once against the same in pieces: both round at the same places
but for the states, the chunks and the order of sums: half a step for each of the four roundings (q.k pairs, state, output, projection) of
each of two blocks and two ways: 16 half steps."""
import pytest
import torch

from oracle.decay_oracle import block_norm_reference, decay_attention_reference
from test_decay_attention_gpu import off, wide

pytestmark = pytest.mark.gpu


def decoder(dtype, **kw):
    from ssd.modules import DecayDecoder
    torch.manual_seed(0)
    net = DecayDecoder(256, 2, d_state=64, headdim=64, ngroups=2, device="cuda", dtype=dtype, **kw)
    with torch.no_grad():
        for p in net.parameters():
            p.add_(0.1 * torch.randn_like(p)) if p.dim() == 1 else None
    return net


def reference(net, params, x):
    """DecayDecoder.forward from the definitions, on the CPU in 64 bits."""
    P = lambda name: params[name]
    u = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * P("norm.weight")
    residual = x
    for i in range(len(net.blocks)):
        pre = f"blocks.{i}."
        m = net.blocks[i].mixer
        qk = m.ngroups * m.d_state
        q, k, v, dt = torch.split(u @ P(pre + "mixer.in_proj.weight").T, [qk, qk, m.d_inner, m.nheads], dim=-1)
        g = -torch.exp(P(pre + "mixer.A_log")) * torch.nn.functional.softplus(dt + P(pre + "mixer.dt_bias"))
        heads = lambda t, n: t.unflatten(-1, (n, -1))
        o, _ = decay_attention_reference(heads(q, m.ngroups), heads(k, m.ngroups), heads(v, m.nheads), g)
        y = o.flatten(-2) @ P(pre + "mixer.out_proj.weight").T
        residual, u = block_norm_reference(y, residual, u @ P(pre + "gate_proj.weight").T, P(pre + "scale"), P(pre + "post_weight"),
                                           P(pre + "next_weight"), net.blocks[i].gate_activation)
    return u


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_a_training_step(act):
    net = decoder(torch.float32, gate_activation=act)
    gen = torch.Generator().manual_seed(1)
    x, dout = torch.randn(2, 70, 256, generator=gen), torch.randn(2, 70, 256, generator=gen)
    out = net(x.cuda())
    names, params = zip(*net.named_parameters())
    grads = torch.autograd.grad(out, params, dout.cuda())
    ref = {n: wide(p).requires_grad_(True) for n, p in zip(names, params)}
    want = reference(net, ref, x.double())
    exp = torch.autograd.grad(want, [ref[n] for n in names], dout.double())
    tol = 16 * 2 * (256 + 70 + 64) * 2.0 ** -24
    assert off(out, want) <= tol
    for n, a, b in zip(names, grads, exp):
        assert off(a, b) <= tol, (n, off(a, b), tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_prompts_then_single_tokens(dtype):
    """Packed prompts fill a pool of states; the tokens after them come one by one, in another order of requests, with rows of padding."""
    net = decoder(dtype)
    tol = 16 * 2 * (256 + 300 + 64) * 2.0 ** -24 if dtype == torch.float32 else 16 * torch.finfo(dtype).eps / 2
    gen = torch.Generator().manual_seed(2)
    lengths, more = [1, 130, 300], 4
    x = [torch.randn(1, n + more, 256, generator=gen).to(dtype).cuda() for n in lengths]
    with torch.no_grad():
        want = [net(t) for t in x]
        cu = torch.tensor([0, 1, 131, 431], dtype=torch.int32, device="cuda")
        out, finals = net(torch.cat([t[:, :n] for t, n in zip(x, lengths)], 1), return_final_states=True, cu_seqlens=cu)
        for i, (a, b) in enumerate(zip([0, 1, 131], [1, 131, 431])):
            assert off(out[0, a:b], wide(want[i][0, :lengths[i]])) <= tol
        states = net.init_states(6)
        place = torch.tensor([4, 0, 3])
        for pool, final in zip(states, finals):
            pool[place.cuda()] = final
        slots = torch.tensor([3, -1, 4, 0], dtype=torch.int32, device="cuda")   # requests 2, none, 0, 1
        for j in range(more):
            rows = [x[2][0, lengths[2] + j], torch.zeros_like(x[0][0, 0]), x[0][0, lengths[0] + j], x[1][0, lengths[1] + j]]
            got = net.step(torch.stack(rows), states, slots)
            for row, i in ((0, 2), (2, 0), (3, 1)):
                assert off(got[row], wide(want[i][0, lengths[i] + j])) <= tol
        assert all(not pool[[1, 2, 5]].any() for pool in states)


def test_a_captured_token():
    """A token of the whole decoder as a graph, replayed over states that go on."""
    net = decoder(torch.bfloat16)
    x = torch.randn(3, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        a = net.init_states(3)
        want = [net.step(x, a).clone() for _ in range(3)]
        b = net.init_states(3)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            net.step(x, net.init_states(3))
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = net.step(x, b)
        for w in want:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("what", ["attention", "norm"])
def test_a_captured_backward_pass(what):
    """While an eager graph of the same leaves lives on another stream PyTorch cannot capture a backward pass: refused before the
    capture is spoilt, the eager graph still good.  Without it, captured gradients are the eager ones."""
    from ssd.block_norm import block_norm
    from ssd.uni import decay_attention as module
    kept, module.CHECK_STATUS = module.CHECK_STATUS, False
    try:
        gen = torch.Generator(device="cuda").manual_seed(1)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
        if what == "attention":
            leaves = [r(1, 200, 1, 64), r(1, 200, 1, 64), r(1, 200, 4, 64), -r(1, 200, 4).abs()]
            call, dout = (lambda: module.decay_attention(*leaves)), r(1, 200, 4, 64)
        else:
            leaves = [r(1, 200, 256), r(1, 200, 256), torch.ones(256, device="cuda")]
            call, dout = (lambda: block_norm(leaves[0], leaves[1], post_weight=leaves[2], pre_weight=leaves[2])[1]), r(1, 200, 256)
        leaves = [t.requires_grad_(True) for t in leaves]
        eager = call()
        want = torch.autograd.grad(eager, leaves, dout, retain_graph=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph, stream=side):
                call()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, leaves, dout), want))
        del eager
        with torch.cuda.stream(side):
            torch.autograd.grad(call(), leaves, dout)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(call(), leaves, dout)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        module.CHECK_STATUS = kept


def test_a_block_around_the_bidirectional_layer():
    from ssd.modules import BiMamba2, Block
    torch.manual_seed(0)
    mixer = BiMamba2(128, d_state=64, headdim=64, device="cuda", dtype=torch.bfloat16)
    block = Block(128, mixer, device="cuda", dtype=torch.bfloat16)
    u = torch.randn(2, 200, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    residual = torch.randn(2, 200, 128, device="cuda", requires_grad=True)
    out, normed = block(u, residual)
    assert out.dtype == torch.float32 and normed.dtype == torch.bfloat16
    y, gate = mixer(u), block.gate_proj(u)
    want = block_norm_reference(wide(y), wide(residual), wide(gate), wide(block.scale), wide(block.post_weight), wide(block.next_weight), "sigmoid")
    assert off(out, want[0]) <= (128 ** 0.5 + 24) * 2.0 ** -24 and off(normed, want[1]) <= 2.0 ** -8 + 40 * 2.0 ** -24
    grads = torch.autograd.grad([out.sum(), normed.float().sum()], [u, residual, *block.parameters()], allow_unused=True)
    assert all(g is None or bool(torch.isfinite(g).all()) for g in grads) and sum(g is not None for g in grads) >= 10
