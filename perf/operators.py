"""Causal linear attention with a decay for each head, its single-token form, and the norms around a residual block, as
cases that can be timed and compared.

A case is a dict of plain values.  `kind` names the call:

  prompt    `decay_attention` without gradients: the outputs of a prompt and the state that single tokens go on from
  train     `decay_attention` forward and backward
  step      `decay_attention_step`: one token of every request, states updated in place
  norm      `block_norm` without gradients
  norm_train  `block_norm` forward and backward

Attention cases have dtype, batch, seqlen (tokens of each row; with `packed` sequences in one row instead, of lengths up to
seqlen), heads, kv_heads (heads of q and k, each shared by heads / kv_heads heads of v), kdim,
vdim, decay ("token": a log decay for each token and head, in the activations' type, or "head": one for each head in fp32)
and initial (an initial state is given).  Norm cases have dtype, batch, seqlen, width, gate ("full": as large as x, "row":
one row for each batch entry, "none"), act (of the gate), scale ("channel" or a number), post (norm after the block) and
wide_residual (the residual stream in fp32).
"""
import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CHUNK = 64                                           # of the plain form
_EPS = 1e-5


def _attn(name, kind, dtype, batch, seqlen, heads, kv_heads, kdim, vdim, decay="token", packed=0, initial=False):
    case = dict(kind=kind, dtype=dtype, batch=batch, seqlen=seqlen, heads=heads, kv_heads=kv_heads, kdim=kdim, vdim=vdim,
                decay=decay, packed=packed, initial=initial)
    return dict(case, name=name) if name else case


def _step(name, dtype, batch, heads, kv_heads, kdim, vdim, slots):
    case = dict(kind="step", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, kdim=kdim, vdim=vdim, slots=slots)
    return dict(case, name=name) if name else case


def _norm(name, kind, dtype, batch, seqlen, width, gate, act, scale, post, wide_residual):
    case = dict(kind=kind, dtype=dtype, batch=batch, seqlen=seqlen, width=width, gate=gate, act=act, scale=scale, post=post,
                wide_residual=wide_residual)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one request generating: eight heads; latency is all there is
        _step("step_one_request", "bf16", 1, 8, 8, 64, 64, 0),
        # a server's batch of requests, states at shuffled places of a pool, q and k shared by all heads
        _step("step_batch_slots", "bf16", 64, 24, 1, 128, 64, 96),
        # many requests with wide heads
        _step("step_wide_heads", "bf16", 128, 16, 2, 128, 128, 0),
        # the smallest fp32 prompt, odd length, small heads
        _attn("prompt_fp32_small", "prompt", "fp32", 1, 253, 4, 1, 16, 32),
        # one short prompt
        _attn("prompt_short", "prompt", "bf16", 1, 384, 8, 2, 64, 64),
        # prompts of several requests packed into one row, from one token to thousands
        _attn("prompt_packed", "prompt", "bf16", 1, 2048, 24, 1, 128, 64, packed=13),
        # one long document, eight groups, going on from a state
        _attn("prompt_long", "prompt", "bf16", 1, 65536, 32, 8, 128, 64, initial=True),
        # training step of a 24-head layer: the sizes of this repository's default benchmark
        _attn("train_24_heads", "train", "bf16", 8, 2048, 24, 1, 128, 64),
        # training step on rows of odd length, wide heads that share nothing, one decay for each head
        _attn("train_wide_heads", "train", "bf16", 3, 1021, 16, 16, 128, 128, decay="head"),
        # the norms around a block while one token is generated
        _norm("norm_one_token", "norm", "bf16", 1, 1, 1024, "none", "none", 1.0, True, False),
        # the norms around a block in training: gate as wide as the block's output, scale for each channel
        _norm("norm_train_gated", "norm_train", "bf16", 16, 4096, 1024, "full", "sigmoid", "channel", True, False),
        # a block conditioned by one gate for each row of the batch, residual stream in fp32, odd lengths
        _norm("norm_train_row_gate", "norm_train", "bf16", 3, 1777, 2048, "row", "none", 0.5, True, True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["prompt", "train", "step", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind.startswith("norm"):
        width = rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 8, 1024)])
        rows = _log(rng, 1, max(1, min(65536, (1 << 25) // width)))
        batch = rng.randint(1, min(rows, 16))
        return _norm(None, kind, dtype, batch, max(1, rows // batch), width, rng.choice(["full", "row", "none"]),
                     rng.choice(["none", "sigmoid", "silu"]), rng.choice(["channel", 1.0, 0.25]), rng.random() < 0.7,
                     rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.randint(1, 32 // kv_heads)
    kdim, vdim = 16 * rng.randint(1, 8), 16 * rng.randint(1, 8)
    if kind == "step":
        batch = _log(rng, 1, 256)
        return _step(None, dtype, batch, heads, kv_heads, kdim, vdim, rng.choice([0, batch + rng.randint(0, 64)]))
    most = (1 << 31) if dtype == "bf16" else 1 << 28   # kdim * vdim * heads * tokens: CUDA cores do the other types
    tokens = _log(rng, 1, max(1, min(32768, most // (kdim * vdim * heads))))
    batch = rng.randint(1, min(tokens, 8))
    packed = rng.choice([0, 0, rng.randint(2, 24)])
    if packed:
        batch, tokens = 1, min(tokens, 4096)
    return _attn(None, kind, dtype, batch, max(1, tokens // batch), heads, kv_heads, kdim, vdim,
                 rng.choice(["token", "token", "head"]), packed, rng.random() < 0.3)


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Lengths of the packed sequences, a case's own: over their logarithm, one of them a single token."""
    u = torch.rand(case["packed"], generator=torch.Generator().manual_seed(case["seqlen"] * 64 + case["packed"]))
    n = torch.exp(u * math.log(case["seqlen"])).round().long().clamp(1, case["seqlen"])
    n[0], n[-1] = case["seqlen"], 1
    return n


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(to)

    if case["kind"].startswith("norm"):
        b, l, d = case["batch"], case["seqlen"], case["width"]
        wide = torch.float32 if case["wide_residual"] else dtype
        s = dict(case=case, x=normal(b, l, d, std=2.0), residual=normal(b, l, d, to=wide), gate=None, post=None,
                 pre=1 + normal(d, std=0.2, to=torch.float32), scale=case["scale"])
        if case["gate"] != "none":
            s["gate"] = normal(b, l if case["gate"] == "full" else 1, d)
        if case["post"]:
            s["post"] = 1 + normal(d, std=0.2, to=torch.float32)
        if case["scale"] == "channel":
            s["scale"] = 0.3 + normal(d, std=0.1, to=torch.float32)
        if case["kind"] == "norm_train":
            s["dout"], s["dnormed"] = normal(b, l, d, to=wide), normal(b, l, d)
            s["leaves"] = [t.requires_grad_(True) for t in (s["x"], s["residual"], s["gate"], s["scale"], s["post"], s["pre"])
                           if isinstance(t, torch.Tensor)]
        return s

    h, hk, n, p = case["heads"], case["kv_heads"], case["kdim"], case["vdim"]
    step = case["kind"] == "step"
    lead, seqs, s = (case["batch"],), case["batch"], dict(case=case, cu=None, initial=None, slots=None)
    if not step:
        lead = (case["batch"], case["seqlen"])
        if case["packed"]:
            lengths = _lengths(case)
            seqs, lead = len(lengths), (1, int(lengths.sum()))
            ends = torch.cumsum(lengths, 0)
            s["cu"] = torch.cat([torch.zeros(1, dtype=torch.long), ends]).to(torch.int32).to(dev)
            # for the plain form: the place of every token in rows padded to the longest sequence
            row = torch.repeat_interleave(torch.arange(seqs), lengths)
            s["at"] = (row * case["seqlen"] + torch.arange(lead[1]) - (ends - lengths)[row]).to(dev)
    s["q"], s["k"], s["v"] = normal(*lead, hk, n), normal(*lead, hk, n), normal(*lead, h, p)
    rate = torch.exp(torch.rand(h, generator=gen, device=dev) * math.log(16.0))
    if step or case["decay"] == "token":               # steps of a layer whose decay follows its input
        s["g"] = (-rate * torch.nn.functional.softplus(normal(*lead, h, to=torch.float32) - 4)).to(dtype)
    else:
        s["g"] = -rate / 100
    if step:
        pool = max(case["slots"], seqs)
        s["state"] = normal(pool, h, n, p, to=torch.float32)
        if case["slots"]:
            s["slots"] = torch.randperm(pool, generator=gen, device=dev)[:seqs].to(torch.int32)
    if case.get("initial"):
        s["initial"] = normal(seqs, h, n, p, to=torch.float32)
    if case["kind"] == "train":
        s["dout"] = normal(*lead, h, p)
        s["leaves"] = [t.requires_grad_(True) for t in (s["q"], s["k"], s["v"])]
        if case["decay"] == "token":
            s["leaves"].append(s["g"].requires_grad_(True))
        if s["initial"] is not None:
            s["leaves"].append(s["initial"].requires_grad_(True))
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------


def _shared(t, heads):
    return t.repeat_interleave(heads // t.shape[-2], dim=-2) if t.shape[-2] != heads else t


def _plain_attention(q, k, v, g, initial, at, seqs, longest):
    """Chunks of _CHUNK tokens: products inside a chunk, and a state that enters it.  In 32 bits; sums of decays in 64."""
    dtype, tokens = q.dtype, q.shape[:2]
    h, p, n = v.shape[2], v.shape[3], q.shape[3]
    g = g.expand(*tokens, h) if g.dim() == 1 else g
    q, k, v, g = q.float() * n ** -0.5, k.float(), v.float(), g.double()
    if at is not None:                                # packed: rows padded to the longest sequence
        rows = lambda t: t.new_zeros(seqs * longest, *t.shape[2:]).index_copy(0, at, t[0]).unflatten(0, (seqs, longest))
        q, k, v, g = rows(q), rows(k), rows(v), rows(g)
    b, l = q.shape[:2]
    pad = -l % _CHUNK
    q, k, v, g = (torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, pad)).unflatten(1, (-1, _CHUNK)) for t in (q, k, v, g))
    c = torch.cumsum(g, 2)                            # (b, chunks, _CHUNK, h)
    last = c[:, :, -1]
    ct = c.permute(0, 1, 3, 2)
    below = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((ct[..., :, None] - ct[..., None, :]).masked_fill(~below, -math.inf).float())
    hk = q.shape[3]
    weights = torch.einsum("bctgn,bcsgn->bcgts", q, k).repeat_interleave(h // hk, dim=2) * decay
    out = torch.einsum("bchts,bcshp->bcthp", weights, v)
    local = torch.einsum("bcshn,bcshp->bchnp", _shared(k, h), v * torch.exp((last[:, :, None] - c).float())[..., None])
    # the state that enters chunk z, and the one after the last: local states of the chunks before it, decayed over those between
    total = torch.cat([torch.zeros_like(last[:, :1]), torch.cumsum(last, 1)], 1).permute(0, 2, 1)      # (b, h, chunks + 1)
    nc = last.shape[1]
    before = torch.ones(nc + 1, nc, dtype=torch.bool, device=q.device).tril(-1)
    between = torch.exp((total[..., :, None] - total[..., None, 1:]).masked_fill(~before, -math.inf).float())
    states = torch.einsum("bhzc,bchnp->bzhnp", between, local)
    if initial is not None:
        states = states + torch.exp(total.float()).permute(0, 2, 1)[..., None, None] * initial[:, None]
    out = out + torch.einsum("bcthn,bchnp->bcthp", _shared(q, h) * torch.exp(c.float())[..., None], states[:, :-1])
    out = out.flatten(1, 2)[:, :l]
    if at is not None:
        out = out.flatten(0, 1).index_select(0, at)[None]
    return out.to(dtype), states[:, -1]


def _plain_step(s):
    case, state = s["case"], s["state"]
    h, n = case["heads"], case["kdim"]
    rows = torch.arange(case["batch"], device=state.device) if s["slots"] is None else s["slots"].long()
    k, q = _shared(s["k"], h).float(), _shared(s["q"], h).float()
    new = state[rows] * torch.exp(s["g"].float())[..., None, None] + k[..., :, None] * s["v"].float()[..., None, :]
    state[rows] = new
    return (torch.einsum("bhn,bhnp->bhp", q, new) * n ** -0.5).to(s["v"].dtype)


def _plain_norm(s):
    x, residual = s["x"].float(), s["residual"].float()
    if s["post"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * s["post"]
    if s["gate"] is not None:
        a, act = s["gate"].float(), s["case"]["act"]
        x = x * (a if act == "none" else torch.sigmoid(a) if act == "sigmoid" else a * torch.sigmoid(a))
    out = residual + s["scale"] * x
    normed = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + _EPS) * s["pre"]
    return out.to(s["residual"].dtype), normed.to(s["x"].dtype)


# ---- one pass --------------------------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _package():
    at = os.path.abspath("bi-mamba2_b200")             # the package's folder is no importable name: it is put on the path
    if at not in sys.path:
        sys.path.insert(0, at)
    from ssd.block_norm import block_norm
    from ssd.uni.decay_attention import decay_attention, decay_attention_step
    return decay_attention, decay_attention_step, block_norm


def _attention(s, finals):
    if own:
        return _package()[0](s["q"], s["k"], s["v"], s["g"], initial_state=s["initial"], return_final_state=finals,
                             cu_seqlens=s["cu"])
    case = s["case"]
    out, state = _plain_attention(s["q"], s["k"], s["v"], s["g"], s["initial"], s.get("at"), case["packed"], case["seqlen"])
    return (out, state) if finals else out


def _norms(s):
    if own:
        act = s["case"]["act"]
        return _package()[2](s["x"], s["residual"], gate=s["gate"], gate_activation=None if act == "none" else act,
                             scale=s["scale"], post_weight=s["post"], pre_weight=s["pre"], eps=_EPS)
    return _plain_norm(s)


def run(s):
    kind = s["case"]["kind"]
    if kind == "step":
        with torch.no_grad():
            out = _package()[1](s["state"], s["q"], s["k"], s["v"], s["g"], slots=s["slots"]) if own else _plain_step(s)
        return {"out": out, "state": s["state"]}
    if kind == "prompt":
        with torch.no_grad():
            out, state = _attention(s, True)
        return {"out": out, "state": state}
    if kind == "norm":
        with torch.no_grad():
            out, normed = _norms(s)
        return {"out": out, "normed": normed}
    if kind == "train":
        out = _attention(s, False)
        return {"out": out.detach(), "grads": list(torch.autograd.grad(out, s["leaves"], s["dout"]))}
    out, normed = _norms(s)
    grads = torch.autograd.grad([out, normed], s["leaves"], [s["dout"], s["dnormed"]])
    return {"out": out.detach(), "normed": normed.detach(), "grads": list(grads)}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"].startswith("norm"):
        rows, d = case["batch"] * case["seqlen"], case["width"]
        wide = 4 if case["wide_residual"] else size
        gate = {"full": rows, "row": case["batch"], "none": 0}[case["gate"]] * d * size
        forward = rows * d * (2 * size + 2 * wide) + gate
        if case["kind"] == "norm":
            return {"bytes": forward, "flops": 12 * rows * d}
        # x, residual, gate and the two gradients in; three gradients out
        return {"bytes": forward + rows * d * (3 * size + 3 * wide) + 2 * gate, "flops": 42 * rows * d}
    h, hk, n, p = case["heads"], case["kv_heads"], case["kdim"], case["vdim"]
    if case["kind"] == "step":
        b = case["batch"]
        return {"bytes": b * (8 * h * n * p + size * (2 * hk * n + 2 * h * p + h)), "flops": 5 * b * h * n * p}
    tokens = int(_lengths(case).sum()) if case["packed"] else case["batch"] * case["seqlen"]
    seqs = case["packed"] or case["batch"]
    states = seqs * h * n * p * 4
    decays = tokens * h * size if case["decay"] == "token" else 4 * h
    forward = tokens * size * (2 * hk * n + 2 * h * p) + decays + (states if case["initial"] else 0)
    if case["kind"] == "prompt":
        return {"bytes": forward + states, "flops": 4 * tokens * h * n * p}
    backward = tokens * size * (4 * hk * n + 3 * h * p) + 2 * decays + (2 * states if case["initial"] else 0)
    return {"bytes": forward + backward, "flops": 14 * tokens * h * n * p}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------


def _exact_sequence(q, k, v, g, initial, dout):
    """One sequence of one head.  q, k (l, n), v (l, p), g (l): every pair of tokens, a block of rows at a time."""
    l, c = q.shape[0], torch.cumsum(g, 0)
    out, dq, dk, dv, flow = torch.empty_like(v), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(c)
    scale, at = q.shape[1] ** -0.5, torch.arange(l, device=q.device)
    start = 0.0 if initial is None else initial
    dstart = None
    for r0 in range(0, l, 2048):
        r = slice(r0, min(l, r0 + 2048))
        e = r.stop
        w = torch.where(at[r, None] >= at[None, :e], torch.exp(torch.clamp(c[r, None] - c[None, :e], max=60.0)), 0.0) * scale
        pair = q[r] @ k[:e].T
        out[r] = (w * pair) @ v[:e]
        if initial is not None:
            enter = scale * torch.exp(c[r])[:, None]
            out[r] += enter * (q[r] @ start)
        if dout is not None:
            dpair = w * (dout[r] @ v[:e].T)
            dq[r] = dpair @ k[:e]
            dk[:e] += dpair.T @ q[r]
            dv[:e] += (w * pair).T @ dout[r]
            moved = dpair * pair
            flow[r] += moved.sum(1)
            flow[:e] -= moved.sum(0)
            if initial is not None:
                dq[r] += enter * (dout[r] @ start.T)
                flow[r] += ((enter * (q[r] @ start)) * dout[r]).sum(1)
                part = (enter * q[r]).T @ dout[r]
                dstart = part if dstart is None else dstart + part
    final = (k * torch.exp(c[-1] - c)[:, None]).T @ v + torch.exp(c[-1]) * start
    dg = torch.flip(torch.cumsum(torch.flip(flow, [0]), 0), [0])
    return out, final, dq, dk, dv, dg, dstart


def _exact_attention(case, s):
    h, hk, dev = case["heads"], case["kv_heads"], s["q"].device
    bounds = s["cu"].tolist() if s["cu"] is not None else None
    spans = [(0, a, z) for a, z in zip(bounds[:-1], bounds[1:])] if bounds else [(b, 0, case["seqlen"]) for b in range(case["batch"])]
    wide = lambda t: None if t is None else t.detach().double()
    q, k, v, g, dout, initial = (wide(s.get(x)) for x in ("q", "k", "v", "g", "dout", "initial"))
    g = g.expand(*q.shape[:2], h) if g.dim() == 1 else g
    out, dq, dk, dv, dg = (torch.zeros_like(t) for t in (v, q, k, v, g))
    final = torch.zeros(len(spans), h, case["kdim"], case["vdim"], dtype=torch.double, device=dev)
    dstart = torch.zeros_like(final)
    for i, (b, a, z) in enumerate(spans):
        for j in range(h):
            m = j * hk // h
            r = _exact_sequence(q[b, a:z, m], k[b, a:z, m], v[b, a:z, j], g[b, a:z, j], None if initial is None else initial[i, j],
                                None if dout is None else dout[b, a:z, j])
            out[b, a:z, j], final[i, j] = r[0], r[1]
            if dout is not None:
                dq[b, a:z, m] += r[2]
                dk[b, a:z, m] += r[3]
                dv[b, a:z, j], dg[b, a:z, j] = r[4], r[5]
                if initial is not None:
                    dstart[i, j] = r[6]
    if case["kind"] == "prompt":
        return {"out": out, "state": final}
    grads = [dq, dk, dv] + ([dg] if case["decay"] == "token" else []) + ([dstart] if initial is not None else [])
    return {"out": out, "grads": grads}


def _exact_norm(case, s):
    wide = lambda t: t.detach().double() if isinstance(t, torch.Tensor) else t
    x, r, gate, scale, post, pre = (wide(s[n]) for n in ("x", "residual", "gate", "scale", "post", "pre"))
    rms = lambda t: torch.sqrt(t.pow(2).sum(-1, keepdim=True) / t.shape[-1] + _EPS)
    unit, sx = (x / rms(x), rms(x)) if post is not None else (x, None)
    n = unit * post if post is not None else x
    sig = torch.sigmoid(gate) if gate is not None else None
    a, da = {"none": (gate, 1.0), "sigmoid": (sig, None), "silu": (None, None)}[case["act"]] if gate is not None else (1.0, 0.0)
    if gate is not None and case["act"] == "sigmoid":
        da = sig * (1 - sig)
    if gate is not None and case["act"] == "silu":
        a, da = gate * sig, sig * (1 + gate * (1 - sig))
    out = r + scale * a * n
    so = rms(out)
    if case["kind"] == "norm":
        return {"out": out, "normed": out / so * pre}
    back = lambda d, u, size: (d - u * (d * u).mean(-1, keepdim=True)) / size
    dn, u = wide(s["dnormed"]), out / so
    dr = wide(s["dout"]) + back(dn * pre, u, so)
    grads = [scale * a * dr, dr]
    if post is not None:
        grads[0] = back(grads[0] * post, unit, sx)
    if gate is not None:
        dgate = dr * scale * n * da
        grads.append(dgate if case["gate"] == "full" else dgate.sum(1, keepdim=True))
    if isinstance(scale, torch.Tensor):
        grads.append((dr * a * n).sum((0, 1)))
    if post is not None:
        grads.append((scale * a * dr * unit).sum((0, 1)))
    grads.append((dn * u).sum((0, 1)))
    return {"out": out, "normed": u * pre, "grads": grads}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("norm"):
        return _exact_norm(case, s)
    if case["kind"] != "step":
        return _exact_attention(case, s)
    state, h = s["state"].double(), case["heads"]
    rows = list(range(case["batch"])) if s["slots"] is None else s["slots"].tolist()
    heads = torch.arange(h, device=state.device) * case["kv_heads"] // h
    q, k, v, g = (s[x].double() for x in ("q", "k", "v", "g"))
    out = torch.empty_like(v)
    for i, r in enumerate(rows):
        state[r] = torch.exp(g[i])[:, None, None] * state[r] + k[i][heads][:, :, None] * v[i][:, None, :]
        out[i] = (q[i][heads][:, None, :] @ state[r])[:, 0] * case["kdim"] ** -0.5
    return {"out": out, "state": state}
