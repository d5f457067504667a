"""The norms before and after a block of a residual network, fused with the block's gate and residual scale.

    n = rms(x) * post_weight                          (x itself without post_weight)
    out = residual + scale * act(gate) * n
    normed = rms(out) * pre_weight                    rms(t) = t / sqrt(mean(t^2) + eps)

x is what a block returned, `out` the residual stream after it and `normed` the next block's input: one pass over the rows
instead of one for each norm, the gate and the sum.  It stands beside the gated RMSNorm inside BiMamba2 (ssd.bi.layernorm_gated) and
runs on libbissd's kernels (csrc/block_norm.cuh); there is no CPU path.  Wrong arguments raise ValueError, tensors off the GPU
and forward-mode derivatives RuntimeError.
"""
from ssd import _cabi

_ACT = {None: 0, "sigmoid": 1, "silu": 2}
_ops = None


def block_norm(x, residual, gate=None, scale=1.0, post_weight=None, pre_weight=None, gate_activation=None, eps=1e-5):
    """Returns (out, normed), or out alone without pre_weight.

    x: (..., width), width 1 to 8192 and fewer than 2^30 rows, float32, bfloat16 or float16; residual: x's shape, x's type or float32.
    gate: of x's type, x's shape or one row for each entry of the first dimension - (batch, 1, width) beside (batch, seqlen, width),
        or one row for all.  gate_activation: None, "sigmoid" or "silu".
    scale: a number or (width) values; post_weight, pre_weight: (width).  Those given are of one type, float32 or x's.

    out has residual's type, normed x's; the norm of out is taken before out is rounded.  Differentiable once with respect to every
    tensor; sums over rows are float32 in a fixed order.
    """
    global _ops
    if _ops is None:
        _ops = _cabi.torch_ops()
    if gate_activation not in _ACT:
        raise ValueError(f"block_norm: gate_activation must be None, 'sigmoid' or 'silu', not {gate_activation!r}")
    number = isinstance(scale, (int, float))
    return _ops.block_norm(x, residual, gate, None if number else scale, float(scale) if number else 1.0, post_weight, pre_weight,
                           _ACT[gate_activation], eps)
