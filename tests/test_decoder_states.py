"""Final states of the decoder and of a block: made and held only where they are asked for, and handed on where they are.  Stand-ins for the
operators: no GPU."""
import pytest
import torch

from ssd import modules


@pytest.fixture
def asked(monkeypatch):
    """What decay_attention is asked for, a call an entry; the stand-ins return v, and states of ones."""
    calls = []

    def attention(q, k, v, g, scale=None, initial_state=None, return_final_state=False, cu_seqlens=None):
        calls.append(dict(initial_state=initial_state, return_final_state=return_final_state, cu_seqlens=cu_seqlens))
        return (v, torch.ones(v.shape[0], v.shape[2], q.shape[3], v.shape[3])) if return_final_state else v

    monkeypatch.setattr(modules, "decay_attention", attention)
    monkeypatch.setattr(modules, "block_norm", lambda y, residual, **kw: (residual + y.float(), y))
    return calls


def decoder(layers=3):
    net = modules.DecayDecoder(256, layers, d_state=16, headdim=64)
    net.norm = torch.nn.Identity()
    return net


def test_a_training_step_asks_for_no_states(asked):
    out = decoder()(torch.randn(2, 5, 256))
    assert out.shape == (2, 5, 256) and [c["return_final_state"] for c in asked] == [False] * 3


def test_states_that_are_asked_for(asked):
    starts = [torch.full((2, 4, 16, 64), float(i)) for i in range(3)]
    out, finals = decoder()(torch.randn(2, 5, 256), starts, True)
    assert out.shape == (2, 5, 256) and len(finals) == 3 and all(f.shape == (2, 4, 16, 64) for f in finals)
    assert all(c["return_final_state"] and c["initial_state"] is s for c, s in zip(asked, starts))


def test_states_that_are_only_given(asked):
    starts = [torch.zeros(2, 4, 16, 64)] * 2
    decoder(2)(torch.randn(2, 5, 256), starts)
    assert [c["return_final_state"] for c in asked] == [False] * 2 and all(c["initial_state"] is starts[0] for c in asked)
