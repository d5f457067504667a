"""A residual block around a mixer that returns more than its output: the rest comes back behind the block's own results.  Stand-ins for the
operators: no GPU."""
import pytest
import torch

from ssd import modules


@pytest.fixture(autouse=True)
def operators(monkeypatch):
    def attention(q, k, v, g, scale=None, initial_state=None, return_final_state=False, cu_seqlens=None):
        return (v, torch.ones(v.shape[0], v.shape[2], q.shape[3], v.shape[3])) if return_final_state else v

    monkeypatch.setattr(modules, "decay_attention", attention)
    monkeypatch.setattr(modules, "block_norm", lambda y, residual, **kw: (residual + y, 2 * y))


def test_a_mixer_with_states():
    mixer = modules.DecayAttention(64, d_state=16, headdim=16)
    block = modules.Block(64, mixer)
    u, residual = torch.randn(2, 5, 64), torch.randn(2, 5, 64)
    plain = block(u, residual)
    out = block(u, residual, return_final_state=True)
    assert len(plain) == 2 and len(out) == 3 and out[2].shape == (2, 4, 16, 16)
    assert torch.equal(out[0], plain[0]) and torch.equal(out[1], plain[1])


@pytest.mark.parametrize("kind", [tuple, list])
def test_any_mixer(kind):
    class Mixer(torch.nn.Module):
        def forward(self, u, extra):
            return kind([u, extra, 7])

    block = modules.Block(8, Mixer(), gate_activation=None)
    u = torch.randn(1, 3, 8)
    out, normed, extra, seven = block(u, u, extra="cache")
    assert torch.equal(out, 2 * u) and torch.equal(normed, 2 * u) and extra == "cache" and seven == 7
