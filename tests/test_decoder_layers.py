"""What the layers around the causal decay attention hand to it, with stand-ins for the operators: no GPU."""
import pytest
import torch

from ssd import modules


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_log_decays_stay_in_32_bits(dtype):
    """-exp(A_log) softplus(dt + dt_bias), each within fp32's roundings (five, of 2^-24) of what 64 bits give for the same projection."""
    torch.manual_seed(0)
    mixer = modules.DecayAttention(64, d_state=16, headdim=16, ngroups=2, dtype=dtype)
    with torch.no_grad():
        mixer.A_log.normal_()
    u = torch.randn(2, 5, 64).to(dtype)
    q, k, v, g = mixer._project(u)
    assert g.dtype == torch.float32 and q.dtype == k.dtype == v.dtype == dtype
    dt = mixer.in_proj(u)[..., -4:].double()
    want = -torch.exp(mixer.A_log.double()) * torch.nn.functional.softplus(dt + mixer.dt_bias.double())
    # softplus(x) = log(1 + e^x) of a sum x that is rounded itself: 2^-24 |x| of x, at most as much of the result's size and 2^-24 |x| e^x / (1 + e^x)
    most = 2.0 ** -24 * (5 * want.abs() + torch.exp(mixer.A_log.double()) * (dt + mixer.dt_bias.double()).abs())
    assert bool(((g.double() - want).abs() <= most).all())
