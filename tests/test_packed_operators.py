"""Attention under masks and changed scores, rotary positions with several axes and layer norm: the plain forms against their
definitions, gradients against differences, and what the entry points refuse."""
import math

import pytest
import torch

from torchft_b200.ops import kernels as K


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _ids(*runs):
    return torch.tensor([[i for i, n in runs for _ in range(n)]], dtype=torch.int32)


# ------------------------------------------------------------------ spans


def _brute_seen(ids, flags, causal, window):
    """[query, key] by the definition, pair by pair, for one row."""
    S = ids.numel()
    doc, start = [], []
    for i in range(S):
        new = i == 0 or ids[i] != ids[i - 1]
        doc.append(doc[-1] + 1 if i and new else 0 if i == 0 else doc[-1])
        start.append(i if new else start[-1])
    opening = [flags is not None and bool(all(flags[j] for j in range(start[i], i + 1))) for i in range(S)]
    seen = torch.zeros(S, S, dtype=torch.bool)
    for i in range(S):
        for j in range(S):
            ok = doc[i] == doc[j] and ids[i] >= 0
            if causal:
                ok = ok and (j <= i or opening[j])
                if window:
                    ok = ok and j > i - window
            seen[i, j] = ok
    return seen


@pytest.mark.parametrize("causal,prefix,window", [(True, False, 0), (True, True, 0), (True, False, 1), (True, True, 4), (True, False, 6), (False, False, 0)])
@pytest.mark.parametrize("seed", range(6))
def test_spans_are_the_definition_s(causal, prefix, window, seed):
    g = torch.Generator().manual_seed(seed)
    S = 40
    ids = (torch.rand(1, S, generator=g) < 0.15).cumsum(1).to(torch.int32)
    ids[0, 12:15] = -1
    ids[0, 36:] = -3
    flags = (torch.rand(1, S, generator=g) < 0.8) if prefix else None
    spans = K.attention_spans(ids, prefix=flags, causal=causal, window=window)
    rows = spans.rows[0].long()
    at = torch.arange(S)
    seen = _brute_seen(ids[0], flags[0] if prefix else None, causal, window)
    assert torch.equal((at >= rows[:, :1]) & (at < rows[:, 1:2]), seen)
    assert torch.equal(((at >= rows[:, 2:3]) & (at < rows[:, 3:4])).t(), seen)
    live = ids[0] >= 0
    for c in range(4):  # what the kernels' ranges of tiles rest on
        assert (rows[live, c].diff() >= 0).all()
    assert spans.padded.tolist() == [[1]] and spans.tiles.shape == (1, 1, 8)
    assert spans.positions[0, 0] == 0 and (spans.positions[0][1:] - spans.positions[0][:-1] <= 1).all()


def test_spans_of_nothing():
    for shape in ((0, 5), (3, 0)):
        spans = K.attention_spans(torch.zeros(shape, dtype=torch.int32))
        assert spans.rows.shape == (*shape, 4)
    out = torch.empty(0, 128, dtype=torch.bfloat16)
    kv = torch.empty(0, 64, dtype=torch.bfloat16)
    K.attention_fwd(out, kv, kv, 3, 0, 2, 1, 64, out, spans=spans)
    K.attention_bwd(out, kv, kv, out, out, torch.empty(3, 2, 0), out, kv, kv, 3, 0, 2, 1, 64, spans=spans)


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("cap,bias", [(0.0, False), (4.0, False), (0.0, True), (2.5, True)])
def test_attention_by_pairs_and_by_differences(cap, bias):
    g = torch.Generator().manual_seed(3)
    B, S, H, G, D = 1, 14, 4, 2, 6
    q, k, v, do = (torch.randn(B, S, n, D, generator=g, dtype=torch.float64) for n in (H, G, G, H))
    ids = _ids((4, 5), (7, 6), (-1, 3))
    spans = K.attention_spans(ids)
    slopes = torch.tensor([0.5, 0.25, 0.125, 1.0]) if bias else None
    seen = _brute_seen(ids[0], None, True, 0)
    o, lse = K.ref_attention_masked(q, k, v, spans.rows, True, cap, slopes)
    for i in range(S):
        for h in range(H):
            keys = seen[i].nonzero().flatten().tolist()
            s = [float(q[0, i, h] @ k[0, j, h // 2]) / math.sqrt(D) for j in keys]
            s = [cap * math.tanh(x / cap) if cap else x for x in s]
            s = [x - (float(slopes[h]) * abs(i - j) if bias else 0.0) for x, j in zip(s, keys)]
            z = sum(map(math.exp, s))
            want = sum(math.exp(x) / z * v[0, j, h // 2] for x, j in zip(s, keys)) if keys else torch.zeros(D, dtype=torch.float64)
            torch.testing.assert_close(o[0, i, h], want, rtol=1e-12, atol=1e-12)
            assert lse[0, h, i] == (pytest.approx(math.log(z)) if keys else -math.inf)
    args = [t.clone().requires_grad_(True) for t in (q, k, v)]
    f = lambda *a: (K.ref_attention_masked(*a, spans.rows, True, cap, slopes)[0] * do).sum()  # noqa: E731
    grads = torch.autograd.grad(f(*args), args)
    for i, grad in enumerate(grads):
        step = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        up, down = [[t.detach() + (sign * 1e-5 * step if j == i else 0) for j, t in enumerate(args)] for sign in (1, -1)]
        # a central difference: an error of 1e-10 of the third derivative and of 1e-16 / 1e-5
        torch.testing.assert_close((f(*up) - f(*down)) / 2e-5, (grad * step).sum(), rtol=1e-7, atol=1e-7)


def test_attention_entries_run_the_plain_form_on_the_cpu():
    g = torch.Generator().manual_seed(1)
    B, S, H, G, D = 2, 9, 4, 2, 64
    qkv = torch.randn(B * S, (H + 2 * G) * D, generator=g).to(torch.bfloat16)
    do = torch.randn(B * S, H * D, generator=g).to(torch.bfloat16)
    cut = lambda t: (t[:, : H * D], t[:, H * D : (H + G) * D], t[:, (H + G) * D :])  # noqa: E731
    spans = K.attention_spans(torch.cat([_ids((0, 4), (1, 5)), _ids((0, 7), (-1, 2))]))
    out, lse, d = torch.empty_like(do), torch.empty(B, H, S), torch.empty_like(qkv)
    how = {"spans": spans, "softcap": 10.0, "slopes": torch.full((H,), 0.1)}
    K.attention_fwd(*cut(qkv), B, S, H, G, D, out, lse, **how)
    K.attention_bwd(*cut(qkv), out, do, lse, *cut(d), B, S, H, G, D, **how)
    q, k, v = (t.double().reshape(B, S, -1, D).requires_grad_(True) for t in cut(qkv))
    o, l = K.ref_attention_masked(q, k, v, spans.rows, True, 10.0, how["slopes"])
    o.backward(do.double().reshape(B, S, H, D))
    u = 2.0**-8 + 2.0**-12  # one rounding to bf16, and fp32 sums
    assert ((out.double() - o.reshape(B * S, -1)).abs() <= u * o.reshape(B * S, -1).abs() + 1e-5).all()
    torch.testing.assert_close(lse.double(), l, rtol=1e-5, atol=1e-5)
    for got, want in zip(cut(d), (q.grad, k.grad, v.grad)):
        assert ((got.double() - want.reshape(B * S, -1)).abs() <= u * want.reshape(B * S, -1).abs() + 1e-5).all()
    assert not out[-2:].any() and not d[-2:].any()


# ------------------------------------------------------------------ rotation and norm


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_axes_of_one_axis_is_rope(dtype):
    T, n, D = 12, 3, 16
    buf = torch.randn(T, 5 * D).to(dtype)
    inv, axis = K.rope_axes_freqs([D // 2], 1000.0, "cpu")
    got, want = buf.clone(), buf.clone()
    K.rope_axes_(got, torch.arange(T, dtype=torch.int32).view(1, -1), inv, axis, n, D)
    K.rope_(want, K.rope_table(T, D, 1000.0, "cpu"), T, n, D)
    torch.testing.assert_close(got, want, rtol=2.0**-7 if dtype == torch.bfloat16 else 1e-6, atol=1e-6)
    K.rope_axes_(got, torch.arange(T, dtype=torch.int32).view(1, -1), inv, axis, n, D, backward=True)
    # there and back: two roundings of each, of at most half a step of the pair's length
    torch.testing.assert_close(got, buf, rtol=0, atol=4 * torch.finfo(dtype).eps / 2 * float(buf.abs().max()) * 2)


def test_rope_axes_freqs():
    inv, axis = K.rope_axes_freqs([2, 3, 3], 100.0, "cpu")
    assert axis.tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
    torch.testing.assert_close(inv, 100.0 ** -(torch.arange(8, dtype=torch.float64) / 8))
    inv, axis = K.rope_axes_freqs([2, 4], 100.0, "cpu", restart=True)
    torch.testing.assert_close(inv, torch.cat([100.0 ** -(torch.arange(n, dtype=torch.float64) / n) for n in (2, 4)]))
    for bad in ([], [0, 0], [2, -1]):
        with pytest.raises(ValueError):
            K.rope_axes_freqs(bad, 100.0, "cpu")


@pytest.mark.parametrize("bias", [True, False])
def test_layernorm_on_the_cpu(bias):
    T, D = 7, 24
    x, res, dy = (torch.randn(T, D) for _ in range(3))
    w, b = torch.randn(D), torch.randn(D) if bias else None
    y, mean, rstd, h = K.layernorm_fwd(x, w, b, 1e-5, res=res)
    xd, wd = h.double().requires_grad_(True), w.double().requires_grad_(True)
    bd = b.double().requires_grad_(True) if bias else None
    want = torch.nn.functional.layer_norm(xd, (D,), wd, bd, 1e-5)
    want.backward(dy.double())
    torch.testing.assert_close(y.double(), want.detach(), rtol=1e-5, atol=1e-5)
    dx, dw, db = K.layernorm_bwd(dy, h, w, mean, rstd, dres=res, bias=bias)
    torch.testing.assert_close(dx.double(), xd.grad + res.double(), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(dw.double(), wd.grad, rtol=1e-5, atol=1e-5)
    assert (db is None) != bias
    dw2, db2 = dw.clone(), db.clone() if bias else None
    K.layernorm_bwd(dy, h, w, mean, rstd, dw=dw2, db=db2, bias=bias, accumulate=True)
    torch.testing.assert_close(dw2, 2 * dw)


def test_layernorm_of_no_rows():
    x, w = torch.empty(0, 16), torch.ones(16)
    y, mean, rstd, h = K.layernorm_fwd(x, w)
    assert y.shape == (0, 16) and mean.shape == (0,)
    dx, dw, db = K.layernorm_bwd(x, x, w, mean, rstd)
    assert not dw.any() and not db.any()
    kept, _, _ = K.layernorm_bwd(x, x, w, mean, rstd, dw=w.clone(), db=w.clone(), accumulate=True)[1], None, None
    assert torch.equal(kept, w)


# ------------------------------------------------------------------ refusals


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_of_spans(device):
    ids = torch.zeros(2, 5, dtype=torch.int32, device=device)
    for bad in (ids.long(), ids[0], ids.t()):
        with pytest.raises(ValueError):
            K.attention_spans(bad)
    with pytest.raises(ValueError):
        K.attention_spans(ids, prefix=torch.zeros(2, 4, dtype=torch.bool, device=device))
    with pytest.raises(ValueError):
        K.attention_spans(ids, prefix=ids)
    for window in (-1, 2**31):
        with pytest.raises(ValueError):
            K.attention_spans(ids, window=window)
    with pytest.raises(ValueError):
        K.attention_spans(ids, causal=False, window=3)
    with pytest.raises(ValueError):
        K.attention_spans(ids, causal=False, prefix=ids.bool())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_of_masked_attention(device):
    B, S, H, G, D = 2, 8, 4, 2, 64
    q, kv = torch.zeros(B * S, H * D, dtype=torch.bfloat16, device=device), torch.zeros(B * S, G * D, dtype=torch.bfloat16, device=device)
    lse = torch.zeros(B, H, S, device=device)
    spans = K.attention_spans(torch.zeros(B, S, dtype=torch.int32, device=device))

    def both(q=q, k=kv, lse=lse, heads=(H, G, D), spans=spans, dk=kv, **how):
        with pytest.raises(ValueError):
            K.attention_fwd(q, k, kv, B, S, *heads, torch.zeros_like(q), lse, spans=spans, **how)
        with pytest.raises(ValueError):
            K.attention_bwd(q, k, kv, q, q, lse, q, dk, kv, B, S, *heads, spans=spans, **how)

    both(q=q.float())
    both(q=q[:-1])
    both(k=q)
    both(lse=lse.double())
    both(lse=lse[:, :-1])
    both(heads=(H, 3, D))
    both(heads=(2 * H, 2 * G, 32))
    both(spans=K.attention_spans(torch.zeros(B, S + 1, dtype=torch.int32, device=device)))
    for cap in (-1.0, math.inf, math.nan, 1e-10, 1e31, 1e-50):
        both(softcap=cap)
    both(slopes=torch.zeros(H - 1, device=device))
    both(slopes=torch.zeros(H, device=device).double())
    with pytest.raises(ValueError):
        K.attention_bwd(q, kv, kv, q, q, lse, q, kv[:-1], kv, B, S, H, G, D, spans=spans)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_of_rope_axes(device):
    T, n, D = 4, 2, 16
    buf, pos = torch.zeros(T, 3 * D, device=device), torch.zeros(2, T, dtype=torch.int32, device=device)
    inv, axis = K.rope_axes_freqs([4, 4], 10.0, device)
    for args in ((buf.double(), pos, inv, axis, n, D), (buf.t(), pos, inv, axis, n, D), (buf, pos.long(), inv, axis, n, D),
                 (buf, pos[:, :-1], inv, axis, n, D), (buf, pos[0], inv, axis, n, D), (buf, pos, inv.float(), axis, n, D),
                 (buf, pos, inv[1:], axis, n, D), (buf, pos, inv, axis.long(), n, D), (buf, pos, inv, axis, 4, D), (buf, pos, inv, axis, 0, D),
                 (buf, pos, inv, axis, n, 15)):
        with pytest.raises(ValueError):
            K.rope_axes_(*args)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_of_layernorm(device):
    x, w, s = torch.zeros(4, 16, device=device), torch.zeros(16, device=device), torch.zeros(4, device=device)
    for args in ((x.double(), w), (x[:, :12], w[:12]), (x[0], w), (x, w[1:]), (x, w.bfloat16()), (x, w, w[1:]), (x.t(), w)):
        with pytest.raises(ValueError):
            K.layernorm_fwd(*args)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, w, res=x[1:])
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, w, res=x, out=x, h_out=x)
    for args in ((x[1:], x, w, s, s), (x, x, w, s[1:], s), (x, x, w, s, s.double()), (x.bfloat16(), x, w, s, s)):
        with pytest.raises(ValueError):
            K.layernorm_bwd(*args)
    with pytest.raises(ValueError):
        K.layernorm_bwd(x, x, w, s, s, accumulate=True)
    with pytest.raises(ValueError):
        K.layernorm_bwd(x, x, w, s, s, dw=w, accumulate=True)


@pytest.mark.parametrize("device", DEVICES)
def test_tensors_on_two_devices_are_refused(device):
    x, w = torch.zeros(4, 16, device=device), torch.zeros(16, device=device)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, w.to("meta"))
    with pytest.raises(ValueError):
        K.attention_spans(torch.zeros(2, 5, dtype=torch.int32, device=device), prefix=torch.zeros(2, 5, dtype=torch.bool, device="meta"))


def test_c_entries_refuse_before_they_launch():
    """The C side looks at sizes and alignment itself, without a GPU."""
    lib = K.N.lib()
    a, odd = 1 << 12, (1 << 12) + 8
    assert K._fn("layernorm_fwd")(a, None, None, a, None, a, a, a, 4, 12, 1e-5, 0, None) == -1
    assert K._fn("layernorm_fwd")(odd, None, None, a, None, a, a, a, 4, 16, 1e-5, 0, None) == -2
    assert K._fn("layernorm_fwd")(a, None, None, a, None, a, a, a, 4, 16392, 1e-5, 0, None) == -4
    assert K._fn("layernorm_bwd")(a, a, a, a, a, None, a, a, None, a, 4, 16392, 0, 0, None, None) == -4
    assert K._fn("layernorm_bwd")(a, odd, a, a, a, None, a, a, None, a, 4, 16, 0, 0, None, None) == -2
    assert K._fn("rope_axes")(odd, a, a, a, 4, 1, 2, 16, 32, 0, 0, 0, None) == -2
    assert K._fn("rope_axes")(a, a, a, a, 4, 1, 2, 20, 40, 0, 0, 0, None) == -2
    assert K._fn("rope_axes")(a, a, a, a, 4, 1, 2, 16, 36, 0, 0, 0, None) == -2
    assert K._fn("rope_axes")(a, a, a, a, 4, 1, 2, 24, 48, 0, 1, 0, None) == -2
    assert K._fn("rope_axes")(a, a, a, a, 4, 1, 1, 2048, 2048, 0, 0, 0, None) == -4
    assert K._fn("attention_spans")(a, None, odd, a, a, a, 1, 5, 1, 0, None) == -2
    assert K._fn("attention_spans")(a, a, a, a, a, a, 1, 5, 0, 0, None) == -1
    assert K._fn("attention_spans")(a, None, a, a, a, a, 1, (1 << 30) + 1, 1, 0, None) == -4
    fwd = lambda head_dim, q, rows, cap: K._fn("attention_masked_fwd")(  # noqa: E731
        q, a, a, a, None, rows, a, a, None, 1, 8, 2, 1, head_dim, 128, 64, 64, 128, 0.1, cap, 1, None, None)
    assert fwd(32, a, a, 0.0) == -1 and fwd(64, odd, a, 0.0) == -2
    bwd = lambda head_dim, q, rows, cap: K._fn("attention_masked_bwd")(  # noqa: E731
        q, a, a, a, a, a, a, a, a, a, rows, a, a, None, 1, 8, 2, 1, head_dim, 128, 64, 64, 128, 128, 128, 64, 64, 0.1, cap, 1, None, None, None)
    assert bwd(32, a, a, 0.0) == -1 and bwd(64, odd, a, 0.0) == -2
    assert bwd(64, a, None, 0.0) == -1 and bwd(64, a, odd, 0.0) == -2 and bwd(64, a, a, -1.0) == -1 and bwd(64, a, a, math.nan) == -1
    assert lib is K.N.lib()


def test_the_host_module_refuses_tensors_off_the_gpu():
    host = K.N.host()
    x, w, ids = torch.zeros(4, 16), torch.zeros(16), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="on a GPU"):
        host.layernorm_fwd(x, w, None, 1e-5, None, None, None, None, None)
    with pytest.raises(ValueError, match="on a GPU"):
        host.attention_spans(ids, None, True, 0)
    with pytest.raises(TypeError):
        host.attention_spans(ids, None, True)
    with pytest.raises(TypeError):
        host.attention_spans(None, None, True, 0)
    with pytest.raises(TypeError):
        host.attention_spans(ids, 3, True, 0)
