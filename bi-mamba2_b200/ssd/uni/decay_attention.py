"""Causal linear attention with a decay for each head: the one-directional sibling of the bidirectional scan.

    S_t = exp(g_t) S_{t-1} + k_t v_t^T          o_t = scale * S_t^T q_t

The scan's terms in other letters: q = C, k = B, v = dt * x, g = dt * A, the state kept as (dstate, headdim).  The reference
keeps a causal path beside its bidirectional one (src/ssd/uni/); these are a decoder's two forms of it:

  decay_attention         whole sequences, forward and backward, with the state they start from and the one they end in
  decay_attention_step    one token of every request, the states updated in place

Both run on libbissd's kernels (csrc/uni_*.cuh); there is no CPU path.  Wrong arguments raise ValueError, tensors off the GPU and
forward-mode derivatives RuntimeError.
"""
from ssd import _cabi
from ssd.bi.ssd_combined import CHECK_STATUS

_ops = None


def _native():
    global _ops
    if _ops is None:
        _ops = _cabi.torch_ops()
    return _ops


def decay_attention(q, k, v, g, scale=None, initial_state=None, return_final_state=False, cu_seqlens=None):
    """Outputs of whole sequences, and with return_final_state the states after them.

    q, k: (batch, seqlen, kv_heads, kdim); v: (batch, seqlen, heads, vdim), heads a multiple of kv_heads: head h reads head
        h * kv_heads // heads of q and k.  float32, bfloat16 or float16, all the same; head sizes 1 to 256; any strides (a copy
        is made where the innermost dimension is not contiguous or 16-bit rows are not 16-byte aligned).
    g: log decays (batch, seqlen, heads), or (heads) where they are the same for all tokens; of q's type or float32.  They are meant
        to be at most 0; -inf empties the state before the token.
    scale: kdim ** -0.5 by default.
    initial_state: (batch, heads, kdim, vdim) float32, zeros by default.  final states have that shape and type.
    cu_seqlens: (n + 1) int32 (or int64, which costs a conversion) on the GPU: with batch 1, sequence i is the tokens cu_seqlens[i]
        up to cu_seqlens[i + 1], and there are n states.  Sequences may be empty.  Boundaries are taken to 0 ... seqlen and never back;
        tokens of no sequence have zeros for outputs and gradients.

    On the tensor cores (16-bit types, kdim up to 128, head sizes that are multiples of 8, scale > 0) the state that enters a chunk of 128
    tokens of a sequence, the products scale * q.k of its pairs, rows of v weighted by decays and their gradients' like are rounded to the tensors'
    type on the way.  In float16 a head of a sequence for which any of these, or an input, is out of range (65504) is computed again on the CUDA
    cores, in float32 throughout and many times slower; those below 2^-14, where float16 has fewer bits, are off by up to 2^-25 each (small q and k
    beside a large v, a small scale, small gradients: float32 tensors, of which nothing is rounded on the way, are the choice there).  In
    bfloat16 a value of v, in the backward pass also of q, k or a gradient, that is not finite reaches all 128 tokens of its chunk, also those
    before it; other sequences never.  The states handed in and out are float32 throughout.  How a call is split over the GPU follows its
    sizes: the last bits of a row may depend on the number of rows.

    A call has at most 2^23 - 1 tokens.

    Differentiable once with respect to q, k, v, g and initial_state.  Returns the output (like v), or (output, final states).
    Gradients of one q, k or g that several heads or tokens share are summed in float32 in a fixed order, as everything is.
    """
    return _native().decay_attention(q, k, v, g, scale, initial_state, return_final_state, cu_seqlens, CHECK_STATUS)


def decay_attention_step(state, q, k, v, g, scale=None, slots=None):
    """One token of every request: updates the requests' states in place and returns the outputs (batch, heads, vdim).

    state: (slots, heads, kdim, vdim) float32, each slot contiguous, as decay_attention's final states are.
    q, k: (batch, kv_heads, kdim); v: (batch, heads, vdim); g: (batch, heads) or (heads); types and scale as decay_attention's.
    slots: (batch) int32 (or int64, which costs a conversion): the state of each request; without it request i has state i.  A slot
        outside the pool marks a row of padding: zeros are returned for it and no state changes.  Requests with the same slot are
        tokens of one sequence, taken in the order of their rows.

    No gradient is defined: raises RuntimeError where autograd would want one.
    """
    return _native().decay_step(state, q, k, v, g, scale, slots)
