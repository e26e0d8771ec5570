"""Operators of packed and multi-modal decoder training whose speed is tracked: attention under document and prefix masks with
capped or distance-biased scores, rotary positions with several axes, layer norm.  Each forward and backward.

Sizes are those of the model configurations (llama-tiny 4/2 heads of 64, llama-small 8/2 of 128, llama3-1b 32/8 of 64,
llama3-8b 32/8 of 128), of ``bench.py`` (one sequence of 8192) and ``bench_diloco.py`` (sequences of 2048), and 3 x 1000
tokens for what is a multiple of nothing.

``run`` computes an operator in its plain form, in 32 bits from elementary operations, or with ``own`` by the package's
kernels.  ``exact`` is the definition in 64 bits, written row by row and head by head.
"""

import math

import torch

own = False

ROPE_THETA = 500000.0
EPS = 1e-5


def listed():
    return [
        # a debugging-size model's forward pass over a few short documents: launches count, not the chip
        _attention("attn-tiny", 1, 256, 4, 2, 64, mean=60),
        # a training step of the 8B model on one packed sequence of the benchmark's length, documents of a thousand tokens
        _attention("attn-8b-packed-train", 1, 8192, 32, 8, 128, mean=1000, train=True),
        # a training step of the 1B model at the DiLoCo benchmark's length: capped scores, documents and a padded tail
        _attention("attn-1b-capped-train", 4, 2048, 32, 8, 64, mean=700, cap=50.0, pad=True, train=True),
        # a small model on ragged rows whose documents open with a prompt that is seen in both directions
        _attention("attn-small-prefix-train", 3, 1000, 8, 2, 128, mean=400, prefix=True, pad=True, train=True),
        # evaluation on a long context with linear distance biases, 16384 tokens in few documents
        _attention("attn-long-bias", 1, 16384, 8, 2, 128, mean=9000, slopes=True),
        # evaluation with capped scores and a sliding window of 1024
        _attention("attn-8b-capped-window", 2, 4096, 32, 8, 128, mean=2500, cap=30.0, window=1024),
        # a debugging-size model's packed QKV of one short image-and-text row: latency
        _rope("rope-tiny", 256, 6, 8, 64, axes=3),
        # the 8B model's packed QKV (32 + 8 of 48 heads rotated), time/height/width positions, forward
        _rope("rope-8b-image", 8192, 40, 48, 128, axes=3),
        # two-axis (height, width) positions of a vision tower, gradients of 3 x 1000 patches rotated back, half-split pairs, fp32
        _rope("rope-small-patches-bwd", 3000, 10, 12, 128, axes=2, half=True, backward=True, dtype="float32"),
        # a block's norm of the 8B width on a full step's tokens, with the residual sum
        _norm("norm-8b-fwd", 8192, 4096, res=True),
        # the same width of the 1B model backwards, with the residual's gradient and those of weight and bias
        _norm("norm-1b-bwd", 8192, 2048, res=True, backward=True),
        # a small model's rows, fp32, backwards without a residual
        _norm("norm-small-bwd", 750, 1024, backward=True, dtype="float32"),
    ]


def _attention(name, batch, seq, heads, kv_heads, dim, mean, causal=True, prefix=False, window=0, cap=0.0, slopes=False, pad=False,
               train=False):
    return {"name": name, "op": "attention", "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim, "mean": mean,
            "causal": causal, "prefix": prefix, "window": window, "cap": cap, "slopes": slopes, "pad": pad, "train": train}


def _rope(name, tokens, rotated, heads, dim, axes, half=False, backward=False, dtype="bfloat16"):
    return {"name": name, "op": "rope", "tokens": tokens, "rotated": rotated, "heads": heads, "dim": dim, "axes": axes, "half": half,
            "backward": backward, "dtype": dtype}


def _norm(name, rows, width, res=False, bias=True, backward=False, dtype="bfloat16"):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "res": res, "bias": bias, "backward": backward, "dtype": dtype}


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "rope", "norm"))
    if op == "attention":
        kv_heads, rep = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4))
        heads = kv_heads * rep
        seq = _log(rng, 1, min(8192, int(16384 / math.sqrt(heads))))
        batch = min(_log(rng, 1, 16), max(1, 4 * 8192 * 8192 // (heads * seq * seq)), max(1, 16384 // seq))
        causal = rng.random() < 0.85
        case = _attention("", batch, seq, heads, kv_heads, rng.choice((64, 128)), mean=_log(rng, 1 + seq // 50, 2 * seq), causal=causal,
                          prefix=causal and rng.random() < 0.4, window=_log(rng, 1, 2 * seq) if causal and rng.random() < 0.3 else 0,
                          cap=rng.choice((0.0, 0.0, 15.0, 50.0)), slopes=rng.random() < 0.3, pad=rng.random() < 0.4,
                          train=rng.random() < 0.6)
    elif op == "rope":
        dim = rng.choice((32, 64, 80, 128, 256))
        rotated = rng.randint(1, 40)
        heads = rotated + rng.randint(0, 8)
        tokens = _log(rng, 1, min(32768, (1 << 26) // (heads * dim)))
        case = _rope("", tokens, rotated, heads, dim, axes=rng.randint(1, 4), half=rng.random() < 0.5, backward=rng.random() < 0.5,
                     dtype=rng.choice(("bfloat16", "float32")))
    else:
        width = 8 * _log(rng, 8, 2048)
        rows = _log(rng, 1, min(32768, (1 << 25) // width))
        case = _norm("", rows, width, res=rng.random() < 0.5, bias=rng.random() < 0.7, backward=rng.random() < 0.6,
                     dtype=rng.choice(("bfloat16", "float32")))
    del case["name"]
    return case


def _layout(case, seed):
    """Documents of a packed batch: ids [batch, seq] (negative: padding) and flags of the leading tokens of each."""
    g = torch.Generator().manual_seed(seed)
    B, S = case["batch"], case["seq"]
    cuts = torch.rand(B, S, generator=g) < 1.0 / case["mean"]
    ids = cuts.cumsum(1)
    if case["pad"]:
        tail = (torch.rand(B, 1, generator=g) * 0.3 * S).long()
        ids = ids.masked_fill(torch.arange(S) >= S - tail, -1)
    at = torch.arange(S).expand(B, S)
    first = torch.ones(B, S, dtype=torch.bool)
    first[:, 1:] = ids[:, 1:] != ids[:, :-1]
    start = torch.where(first, at, 0).cummax(1).values
    lead = (torch.rand(B, S, generator=g) * 0.5 * case["mean"]).long().gather(1, start)  # one length a document
    prefix = (at - start < lead) & (ids >= 0)
    return ids.to(torch.int32), prefix


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, std=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)

    if case["op"] == "attention":
        B, S, H, G, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        ids, prefix = _layout(case, seed)
        state = {"case": case, "qkv": normal(B * S, (H + 2 * G) * D), "documents": ids.cuda(),
                 "prefix": prefix.cuda() if case["prefix"] else None, "slopes": None}
        # queries and keys of a trained model are far from orthogonal: scores of a few units, some near a cap
        state["qkv"][:, : H * D] *= 2
        if case["slopes"]:
            state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
        if case["train"]:
            state["d_out"] = normal(B * S, H * D)
        return state
    if case["op"] == "rope":
        T, dim, axes = case["tokens"], case["dim"], case["axes"]
        # images of a grid of patches between runs of text: three slow counters
        at = torch.arange(T, device="cuda")
        start = int(torch.randint(0, 100000, (1,), device="cuda", generator=g))
        steps = [torch.div(at, 24 ** (axes - 1 - a), rounding_mode="floor") % (24 if a else 1 << 20) for a in range(axes)]
        positions = torch.stack(steps).to(torch.int32) + start
        half = dim // 2
        inv_freq = ROPE_THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        axis = (torch.arange(half, device="cuda") * axes // half).to(torch.int32)  # sections of equal length
        return {"case": case, "buf": normal(T, case["heads"] * dim, dtype=getattr(torch, case["dtype"])), "positions": positions,
                "inv_freq": inv_freq, "axis": axis}
    T, D, dtype = case["rows"], case["width"], getattr(torch, case["dtype"])
    state = {"case": case, "x": normal(T, D, dtype=dtype, std=2.0, mean=0.3), "w": normal(D, dtype=dtype, std=0.2, mean=1.0),
             "b": normal(D, dtype=dtype, std=0.2) if case["bias"] else None, "res": normal(T, D, dtype=dtype) if case["res"] else None}
    if case["backward"]:  # what the forward pass kept
        x = state["x"].float()
        state["dy"], state["mean"] = normal(T, D, dtype=dtype), x.mean(1)
        state["rstd"] = ((x - state["mean"][:, None]).square().mean(1) + EPS).rsqrt()
    return state


def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    if case["op"] == "rope":
        return _rope_own(state) if own else _rope_plain(state)
    return _norm_own(state) if own else _norm_plain(state)


# ------------------------------------------------------------------ the package's calls


def _attention_own(state):
    from torchft_b200.ops import kernels as K

    c, qkv = state["case"], state["qkv"]
    B, S, H, G, D = (c[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    a, b = H * D, (H + G) * D
    q, k, v = qkv[:, :a], qkv[:, a:b], qkv[:, b:]
    spans = K.attention_spans(state["documents"], prefix=state["prefix"], causal=c["causal"], window=c["window"])
    out = torch.empty(B * S, a, dtype=qkv.dtype, device=qkv.device)
    how = {"spans": spans, "softcap": c["cap"], "slopes": state["slopes"], "any_length": True}
    if not c["train"]:
        K.attention_fwd(q, k, v, B, S, H, G, D, out, **how)
        return out
    lse = torch.empty(B, H, S, dtype=torch.float32, device=qkv.device)
    K.attention_fwd(q, k, v, B, S, H, G, D, out, lse, **how)
    d = torch.empty_like(qkv)
    K.attention_bwd(q, k, v, out, state["d_out"], lse, d[:, :a], d[:, a:b], d[:, b:], B, S, H, G, D, **how)
    return out, lse, d


def _rope_own(state):
    from torchft_b200.ops import kernels as K

    c = state["case"]
    return K.rope_axes_(state["buf"], state["positions"], state["inv_freq"], state["axis"], c["rotated"], c["dim"], half=c["half"],
                        backward=c["backward"])


def _norm_own(state):
    from torchft_b200.ops import kernels as K

    if state["case"]["backward"]:
        return K.layernorm_bwd(state["dy"], state["x"], state["w"], state["mean"], state["rstd"], dres=state["res"],
                               bias=state["case"]["bias"])
    return K.layernorm_fwd(state["x"], state["w"], state["b"], EPS, res=state["res"])


# ------------------------------------------------------------------ the plain forms, in 32 bits


def _seen(state):
    """[batch, 1, query, key]: whether the query sees the key."""
    c, ids = state["case"], state["documents"]
    S = c["seq"]
    at = torch.arange(S, device=ids.device)
    # the documents of a row follow one another, so equal ids are one document
    seen = (ids[:, :, None] == ids[:, None, :]) & (ids >= 0)[:, :, None]
    if c["causal"]:
        before = at[:, None] >= at[None, :]
        seen &= before | state["prefix"][:, None, :] if c["prefix"] else before  # a prefix is seen from all of its document
    if c["window"]:
        seen &= at[None, :] > at[:, None] - c["window"]
    return seen[:, None]


def _attention_plain(state):
    c, qkv = state["case"], state["qkv"]
    B, S, H, G, D = (c[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    rep, cap, scale = H // G, c["cap"], 1.0 / math.sqrt(D)
    x = qkv.float().view(B, S, H + 2 * G, D).transpose(1, 2)  # [batch, head, token, dim]
    q, k, v = x[:, :H], x[:, H : H + G].repeat_interleave(rep, 1), x[:, H + G :].repeat_interleave(rep, 1)
    s = q @ k.transpose(-1, -2)
    s *= scale
    if cap:
        s = torch.tanh(s.div_(cap))
        slope_of_cap = 1 - s * s if c["train"] else None
        s *= cap
    if c["slopes"]:
        at = torch.arange(S, device=qkv.device, dtype=torch.float32)
        s -= state["slopes"][:, None, None] * (at[:, None] - at[None, :]).abs()
    s = s.masked_fill_(~_seen(state), -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    o = p @ v
    out = o.transpose(1, 2).reshape(B * S, H * D).to(qkv.dtype)
    if not c["train"]:
        return out
    lse = (top + total.log()).squeeze(-1)
    do = state["d_out"].float().view(B, S, H, D).transpose(1, 2)
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds -= (do * o).sum(-1, keepdim=True)
    ds *= p
    if cap:
        ds *= slope_of_cap
    ds *= scale
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    dk, dv = dk.view(B, G, rep, S, D).sum(2), dv.view(B, G, rep, S, D).sum(2)
    d = torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B * S, (H + 2 * G) * D)
    return out, lse, d.to(qkv.dtype)


def _rope_plain(state):
    c, buf = state["case"], state["buf"]
    T, dim, n = c["tokens"], c["dim"], c["rotated"]
    angle = state["positions"].double()[state["axis"].long()].t() * state["inv_freq"]  # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if c["backward"]:
        sin = -sin
    x = buf[:, : n * dim].float().view(T, n, dim)
    if c["half"]:
        a, b = x[..., : dim // 2], x[..., dim // 2 :]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1)
    buf[:, : n * dim] = y.reshape(T, n * dim).to(buf.dtype)
    return buf


def _norm_plain(state):
    c, dtype = state["case"], state["x"].dtype
    x, w = state["x"].float(), state["w"].float()
    if c["backward"]:
        rstd = state["rstd"][:, None]
        xh = (x - state["mean"][:, None]) * rstd
        dy = state["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        if c["res"]:
            dx = dx + state["res"].float()
        return dx.to(dtype), (dy * xh).sum(0).to(dtype), dy.sum(0).to(dtype) if c["bias"] else None
    h = x
    if c["res"]:  # the sum is the residual stream that later passes read: the norm is that of the rounded values
        h = (x + state["res"].float()).to(dtype).float()
    mean = h.mean(1, keepdim=True)
    centred = h - mean
    rstd = (centred.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = centred * rstd * w
    if c["bias"]:
        y = y + state["b"].float()
    return y.to(dtype), mean.squeeze(1), rstd.squeeze(1), h.to(dtype)


# ------------------------------------------------------------------ what a pass cannot do without


def _spans64(case, ids, prefix):
    """(first, end) of the keys that each query of one sequence sees; an empty range for padding."""
    S = ids.numel()
    at = torch.arange(S)
    edge = torch.ones(S + 1, dtype=torch.bool)
    edge[1:S] = ids[1:] != ids[:-1]
    starts = edge.nonzero().squeeze(1)
    doc = edge[:S].cumsum(0) - 1
    first, end = starts[doc], starts[doc + 1]
    if case["causal"]:
        lead = torch.zeros(starts.numel() - 1, dtype=torch.long)
        if case["prefix"]:
            lead.index_add_(0, doc, prefix.long())
        end = torch.maximum(at + 1, first + lead[doc])
        if case["window"]:
            first = torch.maximum(first, at + 1 - case["window"])
    return torch.where(ids >= 0, first, 0), torch.where(ids >= 0, end, 0)


def work(case):
    if case["op"] == "attention":
        B, S, H, G, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
        ids, prefix = _layout(case, 0)
        pairs = 0
        for b in range(B):
            first, end = _spans64(case, ids[b], prefix[b])
            pairs += int((end - first).sum())
        packed, rows = 2 * B * S * (H + 2 * G) * D, 2 * B * S * H * D
        moved = packed + rows + 4 * B * S
        if case["train"]:
            moved += 4 * B * H * S + packed + rows  # log-sum-exp out, gradient in, gradients out
        return {"bytes": moved, "flops": pairs * H * D * (14 if case["train"] else 4)}
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rope":
        T, n, dim = case["tokens"], case["rotated"], case["dim"]
        return {"bytes": 2 * size * T * n * dim + 4 * T * case["axes"], "flops": 3 * T * n * dim}
    T, D = case["rows"], case["width"]
    if case["backward"]:
        return {"bytes": size * (T * D * (4 if case["res"] else 3) + 3 * D) + 8 * T, "flops": 12 * T * D}
    return {"bytes": size * (T * D * (4 if case["res"] else 2) + 2 * D) + 8 * T, "flops": 8 * T * D}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _attention_exact(case, seed, state)
    if case["op"] == "rope":
        T, dim, n = case["tokens"], case["dim"], case["rotated"]
        full = state["buf"].double()
        x = full[:, : n * dim].reshape(T, n, dim)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           state["inv_freq"] * state["positions"].t().double()[:, state["axis"].long()])[:, None]
        turn = turn.conj() if case["backward"] else turn
        if case["half"]:
            z = torch.complex(x[..., : dim // 2], x[..., dim // 2 :]) * turn
            y = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(x.reshape(T, n, dim // 2, 2).contiguous()) * turn
            y = torch.view_as_real(z)
        full[:, : n * dim] = y.reshape(T, n * dim)
        return full
    x, w = state["x"].double(), state["w"].double()
    D = case["width"]
    if case["backward"]:
        mean, rstd = state["mean"].double()[:, None], state["rstd"].double()[:, None]
        xh, dy = (x - mean) * rstd, state["dy"].double()
        dot1, dot2 = (dy @ w)[:, None] / D, ((dy * xh) @ w)[:, None] / D
        dx = rstd * (dy * w - dot1 - xh * dot2)
        dx = dx + state["res"].double() if case["res"] else dx
        return dx, torch.einsum("td,td->d", dy, xh), dy.sum(0) if case["bias"] else None
    h = (x + state["res"].double()).to(state["x"].dtype).double() if case["res"] else x
    var, mean = torch.var_mean(h, 1, correction=0)
    rstd = 1 / torch.sqrt(var + EPS)
    y = (h - mean[:, None]) * rstd[:, None] * w
    return y + state["b"].double() if case["bias"] else y, mean, rstd, h


def _attention_exact(case, seed, state):
    B, S, H, G, D = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim"))
    if B * H * S * S > 40 * 8192 * 8192:
        return None
    ids, prefix = _layout(case, seed)
    x = state["qkv"].view(B, S, H + 2 * G, D)
    out = torch.zeros(B, S, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, S), -math.inf, dtype=torch.float64, device="cuda")
    grad = torch.zeros(B, S, H + 2 * G, D, dtype=torch.float64, device="cuda")
    at = torch.arange(S, device="cuda")
    far = (at[:, None] - at[None, :]).abs().double()
    for b in range(B):
        first, end = (t.cuda()[:, None] for t in _spans64(case, ids[b], prefix[b]))
        seen = (at >= first) & (at < end)
        some = seen.any(1, keepdim=True)
        for h in range(H):
            kv = H + h // (H // G)
            q, k, v = x[b, :, h].double(), x[b, :, kv].double(), x[b, :, kv + G].double()
            s = q @ k.t() / math.sqrt(D)
            if case["cap"]:
                t = torch.tanh(s / case["cap"])
                s = case["cap"] * t
            if case["slopes"]:
                s = s - float(state["slopes"][h]) * far
            s = s.masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(some, torch.exp(s - norm), 0.0)
            o = p @ v
            out[b, :, h], lse[b, h] = o, norm[:, 0]
            if case["train"]:
                do = state["d_out"].view(B, S, H, D)[b, :, h].double()
                ds = p * (do @ v.t() - (do * o).sum(1, keepdim=True))
                if case["cap"]:
                    ds = ds * (1 - t * t)
                ds = ds / math.sqrt(D)
                grad[b, :, h] = ds @ k
                grad[b, :, kv] += ds.t() @ q
                grad[b, :, kv + G] += p.t() @ do
    out = out.view(B * S, H * D)
    return (out, lse, grad.view(B * S, (H + 2 * G) * D)) if case["train"] else out
