"""Forward-mode derivatives are not defined for the causal decay attention, its single-token form and the norms around a block: an input that
carries a tangent is refused, not answered without one."""
import pytest
import torch
from torch.autograd import forward_ad

from ssd.block_norm import block_norm
from ssd.uni.decay_attention import decay_attention, decay_attention_step


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("which", range(5), ids=["q", "k", "v", "g", "initial_state"])
@pytest.mark.parametrize("grad", [False, True], ids=["", "and a gradient"])
def test_attention(which, grad):
    a = [torch.zeros(1, 6, 2, 8), torch.zeros(1, 6, 2, 8), torch.zeros(1, 6, 4, 8), torch.zeros(1, 6, 4), torch.zeros(1, 4, 8, 8)]
    if grad:
        a[(which + 1) % 4].requires_grad_(True)
    with forward_ad.dual_level():
        a[which] = dual(a[which])
        with pytest.raises(RuntimeError, match="tangent"):
            decay_attention(*a[:4], initial_state=a[4])


@pytest.mark.parametrize("which", range(5), ids=["state", "q", "k", "v", "g"])
def test_step(which):
    a = [torch.zeros(3, 4, 8, 8), torch.zeros(3, 2, 8), torch.zeros(3, 2, 8), torch.zeros(3, 4, 8), torch.zeros(3, 4)]
    with forward_ad.dual_level(), torch.no_grad():
        with torch.enable_grad():
            a[which] = dual(a[which])
        with pytest.raises(RuntimeError, match="tangent"):
            decay_attention_step(*a)


@pytest.mark.parametrize("which", range(6), ids=["x", "residual", "gate", "scale", "post_weight", "pre_weight"])
def test_block_norm(which):
    x, w = torch.zeros(2, 3, 16), torch.zeros(16)
    a = [x, x.clone(), x.clone(), w, w.clone(), w.clone()]
    with forward_ad.dual_level():
        a[which] = dual(a[which])
        with pytest.raises(RuntimeError, match="tangent"):
            block_norm(a[0], a[1], gate=a[2], scale=a[3], post_weight=a[4], pre_weight=a[5])


def test_a_tangent_that_is_over_is_none():
    """Behind the level, and on a value taken out of it, the usual answer: no implementation without a GPU."""
    x = torch.zeros(2, 3, 16)
    with forward_ad.dual_level():
        d = dual(x)
        primal = forward_ad.unpack_dual(d).primal
        with pytest.raises(RuntimeError, match="CUDA"):
            block_norm(primal, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        block_norm(d, x)
