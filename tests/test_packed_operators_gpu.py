"""Attention under masks and changed scores, rotary positions with several axes and layer norm on the GPU, against plain 64-bit forms.

Bounds count roundings: u = 2^-8 is half a step of bf16.  P is rounded before P V, the output once more; dS before dS K and dS^T Q, and its
delta is that of the rounded output.  What the fp32 sums and the exponentials add is below a twentieth of that (2e-4 of a probability where
the products of a score add up to 50), hence the factor."""
import concurrent.futures
import math

import pytest
import torch

from torchft_b200.ops import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
MORE = 1.05
TINY = 1e-6  # of what is zero


def _documents(B, S, mean, pad=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(B, S, generator=g) < 1.0 / mean).cumsum(1).to(torch.int32)
    if pad:
        ids[:, S - S // 5 :] = -1
        ids[:, S // 3 : S // 3 + 3] = -2
    prefix = (torch.rand(B, S, generator=g) < 0.9).to(torch.uint8)
    return ids.cuda(), prefix.cuda()


def _dense(q, k, v, rows, causal, cap, slopes, do=None):
    """(o, lse, bound of o, gradients, their bounds) in 64 bits; 4-D arguments."""
    B, S, H, D = q.shape
    G = k.shape[2]
    rep = H // G
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    scale = 1 / math.sqrt(D)
    s = q @ k.transpose(-1, -2) * scale
    at = torch.arange(S, device=q.device)
    f = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        s, f = cap * t, 1 - t * t
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (at[:, None] - at[None, :]).abs()
    if rows is None:
        seen = ((at[:, None] >= at[None, :]) | (not causal)).expand(B, 1, S, S)
    else:
        seen = ((at >= rows[..., 0:1]) & (at < rows[..., 1:2]))[:, None]
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse > -math.inf, lse, 0.0).unsqueeze(-1))
    o = p @ v
    e_o = U * (p @ v.abs() + o.abs())
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    if do is None:
        return back(o), lse, back(e_o)
    do = do.double().transpose(1, 2)
    delta = (do * o).sum(-1, keepdim=True)
    e_delta = (do.abs() * e_o).sum(-1, keepdim=True)
    ds = p * (do @ v.transpose(-1, -2) - delta) * f * scale
    e_ds = U * ds.abs() + p * f * scale * e_delta
    shared = lambda t: back(t.view(B, G, rep, S, D).sum(2))  # noqa: E731
    dq, dk, dv = back(ds @ k), shared(ds.transpose(-1, -2) @ q), shared(p.transpose(-1, -2) @ do)
    e_dq = back(e_ds @ k.abs()) + U * dq.abs()
    e_dk = shared(e_ds.transpose(-1, -2) @ q.abs()) + U * dk.abs()
    e_dv = U * (shared(p.transpose(-1, -2) @ do.abs()) + dv.abs())
    return back(o), lse, back(e_o), (dq, dk, dv), (e_dq, e_dk, e_dv)


def _near(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= MORE * bound + TINY)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond, worst {(off / (MORE * bound + TINY)).nan_to_num(1e9).max():.3g} of the bound"


def _packed(B, S, H, G, D, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(B * S, (H + 2 * G) * D, device="cuda", generator=g) * scale).to(torch.bfloat16)
    return qkv, torch.randn(B * S, H * D, device="cuda", generator=g).to(torch.bfloat16)


def _parts(t, H, G, D):
    return t[:, : H * D], t[:, H * D : (H + G) * D], t[:, (H + G) * D :]


def _run(qkv, do, B, S, H, G, D, **how):
    q, k, v = _parts(qkv, H, G, D)
    out = torch.full((B * S, H * D), math.nan, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((B, H, S), math.nan, dtype=torch.float32, device="cuda")
    K.attention_fwd(q, k, v, B, S, H, G, D, out, lse, **how)
    d = torch.full_like(qkv, math.nan)
    K.attention_bwd(q, k, v, out, do, lse, *_parts(d, H, G, D), B, S, H, G, D, **how)
    K.check_status(qkv.device)
    return out, lse, d


def _check(qkv, do, B, S, H, G, D, rows, got, causal=True, softcap=0.0, slopes=None):
    out, lse, d = got
    four = lambda t: t.reshape(B, S, -1, D)  # noqa: E731
    o, l, e_o, grads, bounds = _dense(*map(four, _parts(qkv, H, G, D)), rows, causal, softcap, slopes, four(do))
    _near(four(out), o, e_o, "out")
    none = l == -math.inf
    assert torch.equal(lse == -math.inf, none)
    # 2^-18: 32 roundings of sums of up to 64, and the two base-2 logarithms and exponentials
    torch.testing.assert_close(lse[~none].double(), l[~none], rtol=2.0**-18, atol=2.0**-18 * 8)
    for x, y, e, what in zip(map(four, _parts(d, H, G, D)), grads, bounds, ("dq", "dk", "dv")):
        _near(x, y, e, what)


# ------------------------------------------------------------------ spans


@pytest.mark.parametrize("S", [1, 2, 31, 32, 33, 127, 128, 129, 1000, 1023, 1024, 1025, 2500, 40001])
@pytest.mark.parametrize("causal,prefix,window", [(True, False, 0), (True, True, 0), (True, False, 1), (True, True, 70), (False, False, 0),
                                                  (True, False, 2**31 - 1)])
def test_spans(S, causal, prefix, window):
    for mean, pad in ((1, False), (3, True), (90, True), (700, False), (10**9, False)):
        ids, flags = _documents(2, S, mean, pad, seed=S + mean)
        spans = K.attention_spans(ids, prefix=flags if prefix else None, causal=causal, window=window)
        rows, positions, tiles, padded = K.ref_attention_spans(ids.cpu(), flags.cpu() if prefix else None, causal, window)
        assert torch.equal(spans.rows.cpu(), rows) and torch.equal(spans.positions.cpu(), positions)
        assert torch.equal(spans.tiles.cpu(), tiles) and torch.equal(spans.padded.cpu(), padded)


def test_spans_whole_row_flagged_and_all_padding():
    ids = torch.zeros(3, 3000, dtype=torch.int32, device="cuda")
    ids[1] = -1
    ids[2, 1500:] = -1
    flags = torch.ones(3, 3000, dtype=torch.bool, device="cuda")
    spans = K.attention_spans(ids, prefix=flags)
    for got, want in zip((spans.rows, spans.positions, spans.tiles, spans.padded), K.ref_attention_spans(ids.cpu(), flags.cpu())):
        assert torch.equal(got.cpu(), want)


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,H,G", [(1, 1, 1, 1), (2, 2, 2, 1), (1, 127, 4, 2), (2, 128, 3, 3), (1, 129, 6, 2), (2, 257, 2, 2), (1, 300, 8, 1),
                                     (3, 1000, 8, 2), (1, 1280, 3, 1)])
@pytest.mark.parametrize("mean,pad,prefix,window,causal", [(40, False, False, 0, True), (200, True, False, 0, True), (150, True, True, 0, True),
                                                           (300, False, False, 90, True), (100, True, False, 0, False),
                                                           (250, True, True, 130, True)])
def test_attention_under_documents(B, S, H, G, D, mean, pad, prefix, window, causal):
    qkv, do = _packed(B, S, H, G, D, seed=S + H)
    ids, flags = _documents(B, S, mean, pad, seed=S)
    spans = K.attention_spans(ids, prefix=flags if prefix else None, causal=causal, window=window)
    got = _run(qkv, do, B, S, H, G, D, spans=spans)
    _check(qkv, do, B, S, H, G, D, spans.rows, got)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,S,H,G", [(1, 1, 2, 1), (1, 130, 2, 1), (2, 500, 6, 2), (1, 1100, 3, 3)])
@pytest.mark.parametrize("cap,bias,docs,causal,scale", [(50.0, False, True, True, 1.0), (0.0, True, True, True, 1.0), (15.0, True, True, True, 2.0),
                                                        (5.0, False, False, True, 3.0), (20.0, True, False, False, 1.0),
                                                        (0.01, False, True, True, 1.0), (1e30, False, False, True, 1.0)])
def test_attention_with_changed_scores(B, S, H, G, D, cap, bias, docs, causal, scale):
    qkv, do = _packed(B, S, H, G, D, seed=S + H, scale=scale)
    slopes = 2.0 ** -torch.arange(1, H + 1, device="cuda", dtype=torch.float32) if bias else None
    spans = K.attention_spans(_documents(B, S, 150, docs)[0], causal=causal) if docs else None
    got = _run(qkv, do, B, S, H, G, D, spans=spans, softcap=cap, slopes=slopes, causal=causal)
    _check(qkv, do, B, S, H, G, D, spans.rows if docs else None, got, causal, cap, slopes)


@pytest.mark.parametrize("D,G", [(64, 1), (128, 2)])
def test_large_scores_under_documents(D, G):
    """The maximum moves and the output is rescaled, also from a first block in which a row saw nothing."""
    B, S, H = 1, 700, 2
    qkv, do = _packed(B, S, H, G, D, seed=5, scale=3.0)
    spans = K.attention_spans(_documents(B, S, 230)[0])
    _check(qkv, do, B, S, H, G, D, spans.rows, _run(qkv, do, B, S, H, G, D, spans=spans))


@pytest.mark.parametrize("B,S,H,G,D", [(3, 2500, 8, 8, 64), (5000, 40, 1, 1, 64), (37, 129, 10, 5, 128), (40, 300, 6, 2, 64), (1, 2000, 64, 8, 128)])
def test_more_key_blocks_than_fit_the_chip(B, S, H, G, D):
    """Sorted by their work up to 4096 of them, as they come beyond; of unequal documents, and padding that nobody sees."""
    ids, _ = _documents(B, S, 300, pad=True, seed=B)
    spans = K.attention_spans(ids)
    qkv, do = _packed(B, S, H, G, D, S)
    _check(qkv, do, B, S, H, G, D, spans.rows, _run(qkv, do, B, S, H, G, D, spans=spans))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("D,G,cap", [(64, 2, 0.0), (128, 1, 0.0), (128, 2, 30.0)])
def test_padding_may_hold_anything(bad, D, G, cap):
    B, S, H = 2, 400, 2
    qkv, do = _packed(B, S, H, G, D, seed=9)
    ids, _ = _documents(B, S, 100, pad=True)
    spans = K.attention_spans(ids)
    clean = _run(qkv, do, B, S, H, G, D, spans=spans, softcap=cap)
    dead = (ids < 0).view(-1)
    qkv[dead], do[dead] = bad, bad
    dirty = _run(qkv, do, B, S, H, G, D, spans=spans, softcap=cap)
    for x, y in zip(clean[:2], dirty[:2]):
        assert torch.equal(x, y)
    assert not dirty[0][dead].any() and not dirty[2][dead].any()
    qkv[dead], do[dead] = 0, 0
    _check(qkv, do, B, S, H, G, D, spans.rows, dirty, softcap=cap)


@pytest.mark.parametrize("D", [64, 128])
def test_no_mask_is_the_plain_attention(D):
    """One document, a prefix of none, a window that reaches everything, a cap far away: the causal attention's result within roundings."""
    B, S, H, G = 1, 640, 4, 2
    qkv, do = _packed(B, S, H, G, D, seed=3)
    ids = torch.zeros(B, S, dtype=torch.int32, device="cuda")
    for how in ({"spans": K.attention_spans(ids)}, {"spans": K.attention_spans(ids, prefix=ids.to(torch.uint8), window=S)}, {"softcap": 1e6}):
        _check(qkv, do, B, S, H, G, D, None, _run(qkv, do, B, S, H, G, D, **how))


def test_attention_rope_of_the_gradients_under_a_mask():
    B, S, H, G, D = 1, 300, 4, 2, 64
    qkv, do = _packed(B, S, H, G, D, seed=1)
    table = K.rope_table(S, D, 10000.0, "cuda")
    q, k, v = _parts(qkv, H, G, D)
    spans = K.attention_spans(_documents(B, S, 60)[0])
    out, lse, plain = _run(qkv, do, B, S, H, G, D, spans=spans)
    d = torch.empty_like(qkv)
    K.attention_bwd(q, k, v, out, do, lse, *_parts(d, H, G, D), B, S, H, G, D, spans=spans, rope=table)
    K.rope_(plain, table, S, H + G, D, backward=True)
    # rotated before or after a rounding of at most U of the larger of a pair
    assert ((d.double() - plain.double()).abs() <= 4 * U * plain.double().abs().amax(1, keepdim=True)).all()


def test_attention_leaves_its_neighbours_alone():
    B, S, H, G, D = 2, 333, 4, 2, 128
    qkv, do = _packed(B, S, H, G, D, seed=2)
    spans = K.attention_spans(_documents(B, S, 100, True)[0])
    q, k, v = _parts(qkv, H, G, D)
    wide_o = torch.full((B * S + 5, H * D + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    wide_d = torch.full((B * S + 5, (H + 2 * G) * D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = wide_o[: B * S, : H * D], torch.empty(B, H, S, dtype=torch.float32, device="cuda")
    need = K.attention_bwd_scratch_bytes(B, S, H, G)
    scratch = torch.full((need + 64,), 7, dtype=torch.uint8, device="cuda")
    d = _parts(wide_d[: B * S, : (H + 2 * G) * D], H, G, D)
    K.attention_fwd(q, k, v, B, S, H, G, D, out, lse, spans=spans, softcap=30.0)
    K.attention_bwd(q, k, v, out, do, lse, *d, B, S, H, G, D, spans=spans, softcap=30.0, scratch=scratch[:need])
    K.check_status(out.device)
    assert (wide_o[B * S :] == 7).all() and (wide_o[:, H * D :] == 7).all() and (wide_d[B * S :] == 7).all()
    assert (wide_d[:, (H + 2 * G) * D :] == 7).all() and (scratch[need:] == 7).all()
    _check(qkv, do, B, S, H, G, D, spans.rows, (out, lse, wide_d[: B * S, : (H + 2 * G) * D]), softcap=30.0)


# ------------------------------------------------------------------ rotation


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("T,n,extra,dim,axes", [(1, 1, 0, 16, 1), (3, 6, 2, 64, 3), (257, 5, 1, 80, 2), (1000, 40, 8, 128, 3), (77, 1, 3, 256, 4),
                                                (5000, 3, 0, 32, 1)])
def test_rope_axes(T, n, extra, dim, axes, half, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + dim)
    positions = torch.randint(-(2**31), 2**31, (axes, T), device="cuda", generator=g).to(torch.int32)
    positions[0] = torch.arange(T, device="cuda")
    inv, axis = K.rope_axes_freqs([dim // 2 // axes] * (axes - 1) + [dim // 2 - dim // 2 // axes * (axes - 1)], 10000.0, "cuda")
    axis[-1], axis[0] = -1, axes  # outside: left as they are
    buf = torch.randn(T, (n + extra) * dim, device="cuda", generator=g).to(dtype)
    x = buf.double()[:, : n * dim].reshape(T, n, dim)
    ok = (axis >= 0) & (axis < axes)
    ang = torch.where(ok, positions.double()[axis.long().clamp(0, axes - 1)].t() * inv, 0.0)[:, None]
    for backward in (False, True):
        got = buf.clone()
        assert K.rope_axes_(got, positions, inv, axis, n, dim, half=half, backward=backward) is got
        a, b = (x[..., : dim // 2], x[..., dim // 2 :]) if half else (x[..., 0::2], x[..., 1::2])
        s = -ang.sin() if backward else ang.sin()
        y = (a * ang.cos() - b * s, a * s + b * ang.cos())
        want = torch.cat(y, -1) if half else torch.stack(y, -1).reshape(x.shape)
        size = torch.hypot(a, b)
        size = torch.cat([size, size], -1) if half else torch.stack([size, size], -1).reshape(x.shape)
        # half a step of the result; sine and cosine to 2^-22, products and sum to 2^-23, the angle's product in 64 bits to 2^-53 of 2^31 rad
        bound = torch.finfo(dtype).eps / 2 * want.abs() + size * (2.0**-21 + 2.0**-20)
        assert ((got.double()[:, : n * dim].reshape(T, n, dim) - want).abs() <= bound).all()
        assert torch.equal(got[:, n * dim :], buf[:, n * dim :])
        left = ~ok
        pair = torch.cat([left, left]) if half else left.repeat_interleave(2)
        assert torch.equal(got[:, : n * dim].reshape(T, n, dim)[..., pair], buf[:, : n * dim].reshape(T, n, dim)[..., pair])


def test_rope_axes_of_strided_rows():
    big = torch.full((50, 400), 7.0, dtype=torch.bfloat16, device="cuda")
    buf = big[:40, 8 : 8 + 3 * 64]
    buf.copy_(torch.randn(40, 192, device="cuda"))
    want = buf.clone()
    positions = torch.arange(40, dtype=torch.int32, device="cuda").view(1, -1)
    inv, axis = K.rope_axes_freqs([32], 10000.0, "cuda")
    K.rope_axes_(buf, positions, inv, axis, 3, 64)
    K.rope_(want, K.rope_table(40, 64, 10000.0, "cuda"), 40, 3, 64)
    assert ((buf.double() - want.double()).abs() <= 2 * U * want.double().abs() + 2.0**-18).all()
    assert (big[40:] == 7).all() and (big[:, :8] == 7).all() and (big[:, 200:] == 7).all()


# ------------------------------------------------------------------ layer norm


def _norm_inputs(T, D, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, m=0.0, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std + m).to(dtype)  # noqa: E731
    return r(T, D, m=0.5, std=2.0), r(D, m=1.0, std=0.2), r(D), r(T, D), r(T, D)


NORM_SHAPES = [(1, 8), (3, 64), (200, 256), (149, 264), (37, 512), (300, 520), (1000, 1024), (5, 2040), (600, 2048), (150, 4096), (130, 4104),
               (20, 8192), (160, 8200), (33, 16384)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", NORM_SHAPES)
@pytest.mark.parametrize("use_res,use_b", [(False, True), (True, False), (True, True)])
def test_layernorm_fwd(T, D, dtype, use_res, use_b):
    x, w, b, res, _ = _norm_inputs(T, D, dtype, T + D)
    y, mean, rstd, h = K.layernorm_fwd(x, w, b if use_b else None, 1e-5, res=res if use_res else None)
    want_h = (x.double() + res.double()) if use_res else x.double()
    u = torch.finfo(dtype).eps / 2
    # the sum of two is rounded once in fp32 and once to the type
    assert ((h.double() - want_h).abs() <= (u + 2.0**-24) * want_h.abs()).all()
    hd = h.double()
    m = hd.mean(1)
    var = (hd - m[:, None]).square().mean(1)
    r = 1 / torch.sqrt(var + 1e-5)
    # fp32 sums over groups of threads: at most 16 + log2(512) + 16 roundings one after another
    e = 45 * 2.0**-24
    size = hd.abs().mean(1)
    assert ((mean.double() - m).abs() <= e * size).all()
    # the mean's error enters the variance squared and, by rounding each centred value, twice its relative error
    assert ((rstd.double() - r).abs() <= r * (e + 4 * 2.0**-24 + (e * size) ** 2 * r * r)).all()
    want = (hd - m[:, None]) * r[:, None] * w.double() + (b.double() if use_b else 0)
    slack = (r[:, None] * (hd - m[:, None]).abs() * (e + 8 * 2.0**-24) + r[:, None] * e * size[:, None]) * w.double().abs()
    assert ((y.double() - want).abs() <= u * want.abs() + slack + 2.0**-23 * (b.double().abs() if use_b else 0)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", NORM_SHAPES)
@pytest.mark.parametrize("use_res,use_b,accumulate", [(False, True, False), (True, False, True), (True, True, True)])
def test_layernorm_bwd(T, D, dtype, use_res, use_b, accumulate):
    x, w, b, res, dy = _norm_inputs(T, D, dtype, T + D)
    _, mean, rstd, _ = K.layernorm_fwd(x, w, b)
    dw0, db0 = b.clone(), w.clone()
    dx, dw, db = K.layernorm_bwd(dy, x, w, mean, rstd, dres=res if use_res else None, dw=dw0.clone(), db=db0.clone() if use_b else None, bias=use_b,
                                 accumulate=accumulate)
    u, e = torch.finfo(dtype).eps / 2, 45 * 2.0**-24
    xd, wd, dyd, r = x.double(), w.double(), dy.double(), rstd.double()[:, None]
    xh = (xd - mean.double()[:, None]) * r
    g = dyd * wd
    want = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) + (res.double() if use_res else 0)
    slack = e * r * (g.abs() + g.abs().mean(1, keepdim=True) + 2 * xh.abs() * (g * xh).abs().mean(1, keepdim=True)) + (
        2.0**-23 * res.double().abs() if use_res else 0)
    assert ((dx.double() - want).abs() <= u * want.abs() + slack).all()
    assert (db is None) == (not use_b)
    # a column's fp32 sums: over a group's rows, the groups, the blocks
    chain = (T / (K._sm_count(0) * 1.0) + 16 + 5 + 8 + 4) * 2.0**-24
    for got, terms, before in ((dw, dyd * xh, dw0), (db, dyd, db0)):
        if got is not None:
            before = before.double() if accumulate else 0 * before.double()
            s = terms.sum(0) + before
            assert ((got.double() - s).abs() <= u * s.abs() + (chain + 2 * e) * terms.abs().sum(0) + 2.0**-23 * before.abs()).all()


def test_layernorm_gradient_is_that_of_differences():
    """fp32, along random directions: (L(x + h d) - L(x - h d)) / 2h of the forward kernel's outputs, summed in 64 bits."""
    T, D, h = 9, 512, 1e-2
    x, w, b, _, dy = _norm_inputs(T, D, torch.float32, 4)
    L = lambda x, w, b: (K.layernorm_fwd(x, w, b)[0].double() * dy.double()).sum()  # noqa: E731
    _, mean, rstd, _ = K.layernorm_fwd(x, w, b)
    dx, dw, db = K.layernorm_bwd(dy, x, w, mean, rstd)
    for i, grad in enumerate((dx, dw, db)):
        at = [x, w, b]
        d = torch.randn_like(at[i])
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        diff = (L(*up) - L(*down)) / (2 * h)
        want = (grad.double() * d.double()).sum()
        # fp32 outputs are off by 2^-23 of about 2 each, and their sum over T D terms like its root; the third derivative adds h^2 of the rest
        slack = (T * D) ** 0.5 * 2.0**-21 * 8 / (2 * h) + 2 * h * h * (grad.abs().double() * d.abs().double()).sum()
        assert abs(diff - want) <= slack


def test_layernorm_in_place_and_between_neighbours():
    x, w, b, res, dy = _norm_inputs(70, 1032, torch.bfloat16, 8)
    y, mean, rstd, h = K.layernorm_fwd(x, w, b, res=res)
    x2, r2 = x.clone(), res.clone()
    K.layernorm_fwd(x2, w, b, res=r2, out=x2, h_out=r2)
    assert torch.equal(x2, y) and torch.equal(r2, h)
    dx, dw, db = K.layernorm_bwd(dy, h, w, mean, rstd, dres=res)
    for i in range(3):
        a = [dy.clone(), h.clone(), res.clone()]
        K.layernorm_bwd(a[0], a[1], w, mean, rstd, dres=a[2], dx=a[i])
        assert torch.equal(a[i], dx)


# ------------------------------------------------------------------ together


def _block(x, wn, bn, wqkv, ids, positions, inv, axis, d_att, B, S, H, G, D, cap):
    """Norm, QKV product, rotation, masked attention and back to the norm's input."""
    spans = K.attention_spans(ids)
    n, mean, rstd, _ = K.layernorm_fwd(x, wn, bn)
    qkv = K.linear_fwd(n, wqkv)
    before = qkv.clone()
    K.rope_axes_(qkv, positions if positions is not None else spans.positions.view(1, -1), inv, axis, H + G, D)
    out, lse, d = _run_no_check(qkv, d_att, B, S, H, G, D, spans=spans, softcap=cap)
    d_rot = d.clone()
    K.rope_axes_(d, positions if positions is not None else spans.positions.view(1, -1), inv, axis, H + G, D, backward=True)
    dn = K.linear_dgrad(d, wqkv)
    dx, dwn, dbn = K.layernorm_bwd(dn, x, wn, mean, rstd)
    return {"n": n, "before": before, "qkv": qkv, "out": out, "lse": lse, "d_rot": d_rot, "d": d, "dn": dn, "dx": dx, "dwn": dwn, "dbn": dbn}


def _run_no_check(qkv, do, B, S, H, G, D, **how):
    out, lse, d = torch.empty_like(do), torch.empty(B, H, S, dtype=torch.float32, device="cuda"), torch.empty_like(qkv)
    K.attention_fwd(*_parts(qkv, H, G, D), B, S, H, G, D, out, lse, **how)
    K.attention_bwd(*_parts(qkv, H, G, D), out, do, lse, *_parts(d, H, G, D), B, S, H, G, D, **how)
    return out, lse, d


def _block_inputs(B, S, H, G, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    W = H * D
    r = lambda *s, std=1.0, m=0.0: (torch.randn(*s, device="cuda", generator=g) * std + m).to(torch.bfloat16)  # noqa: E731
    inv, axis = K.rope_axes_freqs([D // 2], 10000.0, "cuda")
    ids, _ = _documents(B, S, 90, pad=True, seed=seed)
    return r(B * S, W), r(W, std=0.1, m=1.0), r(W, std=0.1), r((H + 2 * G) * D, W, std=W**-0.5), ids, None, inv, axis, r(B * S, W)


def test_a_block_of_them_together():
    """The gradient at the block's input against autograd of the same block in 64 bits: each of ten roundings one after another (norm, product,
    rotation, P, output; dS, gradients, rotation back, product, norm) is off by u / sqrt(3) of its value on average and they are independent; the
    backward chain carries those of the forward pass too, so 2 x 10 of them."""
    B, S, H, G, D, cap = 2, 500, 4, 2, 64, 30.0
    a = _block_inputs(B, S, H, G, D, 11)
    got = _block(*a, B, S, H, G, D, cap)
    x, wn, bn, wqkv = (t.double().requires_grad_(True) for t in a[:4])
    ids, inv, axis, d_att = a[4], a[6], a[7], a[8].double()
    spans = K.attention_spans(ids)
    qkv = torch.nn.functional.layer_norm(x, (H * D,), wn, bn, 1e-5) @ wqkv.t()
    rot = qkv[:, : (H + G) * D].reshape(B * S, H + G, D // 2, 2)
    ang = spans.positions.view(-1, 1).double() * inv
    turned = torch.view_as_real(torch.view_as_complex(rot) * torch.polar(torch.ones_like(ang), ang)[:, None]).reshape(B, S, H + G, D)
    v = qkv[:, (H + G) * D :].reshape(B, S, G, D)
    o, _ = K.ref_attention_masked(turned[:, :, :H], turned[:, :, H:], v, spans.rows, softcap=cap)
    live = (ids >= 0).view(-1, 1)
    (o.reshape(B * S, -1) * d_att).sum().backward()
    for name, want in (("dx", x.grad), ("dwn", wn.grad), ("dbn", bn.grad)):
        rel = (got[name].double() - want).norm() / want.norm()
        assert rel < 20**0.5 * U / 3**0.5 * 2, (name, rel)
    assert not got["out"][~live.squeeze(1)].any()


def test_captured_and_replayed_on_two_streams():
    """Two graphs captured on one stream and replayed at once on two others, and eager calls on a side stream: what each gives is its own."""
    B, S, H, G, D, cap = 1, 700, 4, 2, 128, 0.0
    a = [_block_inputs(B, S, H, G, D, s) for s in (1, 2)]
    want = [_block(*x, B, S, H, G, D, cap) for x in a]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _block(*a[0], B, S, H, G, D, cap)
    side.synchronize()
    graphs, outs = [], []
    for x in a:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(_block(*x, B, S, H, G, D, cap))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in a]
    for _ in range(5):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        with torch.cuda.stream(side):
            eager = _block(*a[0], B, S, H, G, D, cap)
    torch.cuda.synchronize()
    K.check_status(a[0][0].device)
    for got, ref in list(zip(outs, want)) + [(eager, want[0])]:
        for k in ("n", "qkv", "out", "lse"):
            assert torch.equal(got[k], ref[k]), k
        # dQ is summed by atomics: fp32 sums in another order move a rounding by a step now and then
        assert ((got["dx"].double() - ref["dx"].double()).norm() / ref["dx"].double().norm()) < U


def test_a_misaligned_tensor_is_refused():
    T, D = 4, 64
    at = lambda n, dtype: torch.zeros(n + 1, dtype=dtype, device="cuda")[1:]  # noqa: E731
    x, odd, w = torch.zeros(T, D, device="cuda"), at(T * D, torch.float32).view(T, D), torch.ones(D, device="cuda")
    _, mean, rstd, _ = K.layernorm_fwd(x, w)
    for args in ((odd, w), (x, at(D, torch.float32))):
        with pytest.raises(K.N.KernelError):
            K.layernorm_fwd(*args)
    with pytest.raises(K.N.KernelError):
        K.layernorm_bwd(odd, x, w, mean, rstd)
    q, spans = at(T * D, torch.bfloat16).view(T, D), K.attention_spans(torch.zeros(1, T, dtype=torch.int32, device="cuda"))
    with pytest.raises(K.N.KernelError):
        K.attention_fwd(q, q, q, 1, T, 1, 1, D, torch.empty_like(q), spans=spans)


def test_threads_with_streams_of_their_own():
    B, S, H, G, D = 2, 300, 4, 2, 64
    ids, _ = _documents(B, S, 40)
    qkv, do = _packed(B, S, H, G, D, 3)
    spans = K.attention_spans(ids)
    want = _run_no_check(qkv, do, B, S, H, G, D, spans=spans)
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [_run_no_check(qkv, do, B, S, H, G, D, spans=K.attention_spans(ids)) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return got

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for many in pool.map(work, range(4)):
            for got in many:
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
                # dQ is summed by atomics, as above
                assert (got[2].double() - want[2].double()).norm() / want[2].double().norm() < U


def test_attention_without_a_log_sum_exp():
    B, S, H, G, D = 2, 200, 4, 1, 128
    ids, _ = _documents(B, S, 50, pad=True)
    spans = K.attention_spans(ids)
    qkv, do = _packed(B, S, H, G, D, 4)
    q, k, v = _parts(qkv, H, G, D)
    out, want = torch.empty_like(do), torch.empty_like(do)
    K.attention_fwd(q, k, v, B, S, H, G, D, out, spans=spans)
    K.attention_fwd(q, k, v, B, S, H, G, D, want, torch.empty(B, H, S, device="cuda"), spans=spans)
    assert torch.equal(out, want)


def test_attention_offsets_beyond_32_bits():
    """3.4 G elements of Q, K and V, 2.3 G of dQ: the last document against the same one by itself, where every tile and block begins alike."""
    S, H, G, D, last = 560000 // 128 * 128, 32, 8, 128, 640
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 60 GB")
    ids = (torch.arange(S, device="cuda") // 1000).to(torch.int32)
    ids[S - last :] = 1 << 20
    qkv = torch.zeros(S, (H + 2 * G) * D, dtype=torch.bfloat16, device="cuda")
    do = torch.zeros(S, H * D, dtype=torch.bfloat16, device="cuda")
    small, do_small = _packed(1, last, H, G, D, 1)
    qkv[S - last :], do[S - last :] = small, do_small
    out, lse, d = _run_no_check(qkv, do, 1, S, H, G, D, spans=K.attention_spans(ids.view(1, S)))
    o1, l1, d1 = _run_no_check(small, do_small, 1, last, H, G, D, spans=K.attention_spans(ids[S - last :].view(1, last)))
    K.check_status(qkv.device)
    assert torch.equal(out[S - last :], o1) and torch.equal(lse[..., S - last :], l1)
    assert not out[: S - last].any() and not d[: S - last].any()
    kv = slice(H * D, None)
    # dK and dV of a group in one sum or in four (few blocks by themselves are shared out); dQ by atomics: a rounding more of each
    torch.testing.assert_close(d[S - last :, kv].double(), d1[:, kv].double(), rtol=2 * U, atol=2.0**-12)
    torch.testing.assert_close(d[S - last :, : H * D].double(), d1[:, : H * D].double(), rtol=2 * U, atol=2.0**-12)


def test_rows_beyond_32_bits():
    T, D = 530000, 4096
    x = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, D, device="cuda").to(torch.bfloat16)
    w, b = torch.randn(2, D, device="cuda").to(torch.bfloat16)
    y, mean, rstd, _ = K.layernorm_fwd(x, w, b)
    y1, mean1, rstd1, _ = K.layernorm_fwd(x[-300:], w, b)
    # two shapes of threads: an element goes through at most 32 + 8 additions in either, each off by 2^-24 of sums up to mean |x| < 1 (of squares: of
    # their own sum, halved in rstd); y is rounded once more, or one step apart
    torch.testing.assert_close(mean[-300:], mean1, rtol=0, atol=80 * 2.0**-24)
    torch.testing.assert_close(rstd[-300:], rstd1, rtol=80 * 2.0**-24, atol=0)
    torch.testing.assert_close(y[-300:], y1, rtol=2 * U, atol=2 * U * 1e-2)
    assert torch.equal(y[: T - 300], b.expand(T - 300, D))
    dx, _, db = K.layernorm_bwd(x, x, w, mean, rstd, dx=y)
    dx1, _, db1 = K.layernorm_bwd(x[-300:], x[-300:], w, mean[-300:], rstd[-300:])
    assert torch.equal(dx[-300:], dx1) and not dx[: T - 300].any()
    # each column's 300 values, of any order
    torch.testing.assert_close(db, db1, rtol=2 * U, atol=300 * 2.0**-24 * float(x[-300:].float().abs().sum(0).max()))
    inv, axis = K.rope_axes_freqs([32, 32], 1e4, "cuda")
    at = torch.randint(0, 1 << 20, (2, T), dtype=torch.int32, device="cuda")
    want = K.rope_axes_(x[-300:].clone(), at[:, -300:].contiguous(), inv, axis, 32, 128)
    K.rope_axes_(x, at, inv, axis, 32, 128)
    assert torch.equal(x[-300:], want) and not x[: T - 300].any()
