"""The causal decay attention and the norms around a block from their definitions, token by token in 64 bits on the CPU."""
import torch


def decay_attention_reference(q, k, v, g, scale=None, initial_state=None, bounds=None):
    """q, k (b, L, hk, N), v (b, L, H, P), g (b, L, H) or (H): (o, final states), differentiable.  `bounds`: boundaries of packed
    sequences (b = 1); tokens outside have zeros."""
    h, n, p = v.shape[2], q.shape[3], v.shape[3]
    scale = n ** -0.5 if scale is None else scale
    heads = torch.arange(h) * q.shape[2] // h
    g = g.expand(*q.shape[:2], h) if g.dim() == 1 else g
    spans = [(b, 0, q.shape[1]) for b in range(q.shape[0])] if bounds is None else [(0, a, z) for a, z in zip(bounds[:-1], bounds[1:])]
    rows = {}
    finals = []
    for i, (b, a, z) in enumerate(spans):
        s = torch.zeros(h, n, p, dtype=torch.float64) if initial_state is None else initial_state[i]
        for t in range(a, z):
            s = torch.exp(g[b, t])[:, None, None] * s + k[b, t][heads][:, :, None] * v[b, t][:, None, :]
            rows[b, t] = scale * torch.einsum("hn,hnp->hp", q[b, t][heads], s)
        finals.append(s)
    zero = 0 * v.sum() + torch.zeros(h, p, dtype=torch.float64)
    out = torch.stack([torch.stack([rows.get((b, t), zero) for t in range(q.shape[1])]) for b in range(q.shape[0])])
    return out, torch.stack(finals)


def decay_step_reference(state, q, k, v, g, scale=None, slots=None):
    """One token of every request, one request after another; returns (o, states)."""
    state = state.clone()
    h, n = v.shape[1], q.shape[2]
    scale = n ** -0.5 if scale is None else scale
    heads = torch.arange(h) * q.shape[1] // h
    out = torch.zeros_like(v)
    for i in range(q.shape[0]):
        at = i if slots is None else int(slots[i])
        if not 0 <= at < state.shape[0]:
            continue
        gi = g if g.dim() == 1 else g[i]
        state[at] = torch.exp(gi)[:, None, None] * state[at] + k[i][heads][:, :, None] * v[i][:, None, :]
        out[i] = scale * torch.einsum("hn,hnp->hp", q[i][heads], state[at])
    return out, state


def block_norm_reference(x, residual, gate=None, scale=1.0, post_weight=None, pre_weight=None, gate_activation=None, eps=1e-5, fixed=False):
    """fixed: the rows' sizes count as constants, so that gradients are without the part that is subtracted for them."""
    def rms(t):
        size = torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps)
        return t / (size.detach() if fixed else size)

    n = x if post_weight is None else rms(x) * post_weight
    if gate is not None:
        act = {None: lambda a: a, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[gate_activation]
        n = act(gate) * n
    out = residual + scale * n
    return out if pre_weight is None else (out, rms(out) * pre_weight)
