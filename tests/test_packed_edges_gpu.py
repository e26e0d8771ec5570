"""Packed-batch operators on the GPU at the edges of what their entries take."""
import math

import pytest
import torch

from torchft_b200.ops import kernels as K

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ layer norm


# Rows for two to three rounds through the ring of shared memory of every group: threads a row 32 (one and two vectors each), 64, 128, 256, 512 (two
# and four), and widths that fill no whole vector of threads.  The last group and the last round are partly empty.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", [(50011, 64), (40009, 264), (20011, 512), (20003, 520), (12007, 1024), (8192, 2048), (6007, 2040), (3001, 4096),
                                 (1501, 8192), (701, 16384)])
@pytest.mark.parametrize("use_res", [False, True])
def test_layernorm_bwd_of_many_rows_a_group(T, D, dtype, use_res):
    g = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s, m=0.0, std=1.0: (torch.randn(*s, device="cuda", generator=g) * std + m).to(dtype)  # noqa: E731
    x, dy, res, w, b = r(T, D, m=0.5, std=2.0), r(T, D), r(T, D), r(D, m=1.0, std=0.2), r(D)
    _, mean, rstd, _ = K.layernorm_fwd(x, w, b)
    dx, dw, db = K.layernorm_bwd(dy, x, w, mean, rstd, dres=res if use_res else None)
    K.check_status(x.device)
    again = K.layernorm_bwd(dy, x, w, mean, rstd, dres=res if use_res else None)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
    u, e = torch.finfo(dtype).eps / 2, 45 * 2.0**-24  # a row's sums over a group: at most 16 + log2(512) + 16 roundings one after another, and a few
    rs = rstd.double()[:, None]
    xh = (x.double() - mean.double()[:, None]) * rs
    dyd = dy.double()
    gw = dyd * w.double()
    want = rs * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True)) + (res.double() if use_res else 0)
    slack = e * rs * (gw.abs() + gw.abs().mean(1, keepdim=True) + 2 * xh.abs() * (gw * xh).abs().mean(1, keepdim=True)) + (
        2.0**-23 * res.double().abs() if use_res else 0)
    assert ((dx.double() - want).abs() <= u * want.abs() + slack).all()
    # a column's fp32 sums: a group's rows, at most 16 groups, the blocks five at a time and over 32 lanes
    chain = (T / K._sm_count(0) + 16 + 5 + 5 + 4) * 2.0**-24
    for got, terms in ((dw, dyd * xh), (db, dyd)):
        s = terms.sum(0)
        assert ((got.double() - s).abs() <= u * s.abs() + (chain + 2 * e) * terms.abs().sum(0)).all()


# ------------------------------------------------------------------ capped scores


def _spread(B, S, H, G, D, most, seed):
    """Queries whose scores go from a few units to `most`, small and large ones next to each other; keys and values of size one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n: torch.randn(B, S, n, D, device="cuda", generator=g)  # noqa: E731
    size = torch.exp(torch.rand(B, S, H, 1, device="cuda", generator=g) * math.log(most)) / 3
    return (r(H) * size).bfloat16(), r(G).bfloat16(), r(G).bfloat16(), r(H).bfloat16()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap,most", [(50.0, 100.0), (250.0, 500.0), (400.0, 50.0), (400.0, 800.0), (1000.0, 100.0), (1000.0, 2000.0), (1e6, 1000.0)])
def test_caps_of_every_size(cap, most, D):
    """A score is off by 2^-20 of itself (its product's fp32 sum 2^-22, the cap's form 2^-21) and 2^-21 of caps up to 260, whose large scores take the
    form of exponentials; a probability by that and, in the backward pass, by three roundings of the log-sum-exp."""
    B, S, H, G = 1, 300, 4, 2
    q, k, v, do = _spread(B, S, H, G, D, most, 1)
    flat = lambda t: t.reshape(B * S, -1)  # noqa: E731
    out, lse = torch.empty_like(flat(q)), torch.empty(B, H, S, device="cuda")
    grads = [torch.empty_like(flat(t)) for t in (q, k, v)]
    K.attention_fwd(flat(q), flat(k), flat(v), B, S, H, G, D, out, lse, softcap=cap)
    K.attention_bwd(flat(q), flat(k), flat(v), out, flat(do), lse, *grads, B, S, H, G, D, softcap=cap)
    K.check_status(q.device)

    u = 2.0**-8
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, do))
    k, v = k.repeat_interleave(H // G, 1), v.repeat_interleave(H // G, 1)
    scale = D**-0.5
    t = torch.tanh(q @ k.transpose(-1, -2) * scale / cap)
    s = (cap * t).masked_fill(~torch.ones(S, S, dtype=torch.bool, device="cuda").tril(), -math.inf)
    want_lse = torch.logsumexp(s, -1)
    # a product's fp32 sum is off by its terms' size, not its own
    sizes = (q.abs() @ k.abs().transpose(-1, -2)).clamp(max=1e30) * scale
    off = 2.0**-21 * (torch.minimum(sizes * (1 - t * t) + (cap * t).abs(), sizes)).amax(-1) + 2.0**-21 * min(cap, 260.0)
    assert ((lse.double() - want_lse).abs() <= off + 2.0**-20 * want_lse.abs() + 1e-6).all()
    p = torch.exp(s - want_lse[..., None])
    o = p @ v
    four = lambda t: t.reshape(B, S, -1, D).transpose(1, 2).double()  # noqa: E731
    e_p = 2 * off[..., None]
    e_o = u * (p @ v.abs() + o.abs()) * 1.05 + 2 * e_p * (p @ v.abs())
    assert ((four(out) - o).abs() <= e_o + 1e-6).all()
    delta, dp, f = (do * o).sum(-1, keepdim=True), do @ v.transpose(-1, -2), 1 - t * t
    e_pb = 2 * (off + 2.0**-21 * want_lse.abs())[..., None]
    ds = p * (dp - delta) * f * scale
    e_ds = u * ds.abs() + p * scale * (f * (do.abs() * e_o).sum(-1, keepdim=True) + (dp - delta).abs() * (e_pb * f + 2.0**-19))
    shared = lambda t: t.view(B, G, H // G, S, D).sum(2)  # noqa: E731
    back = lambda t: t.transpose(-1, -2)  # noqa: E731
    for what, got, want, bound in (("dq", grads[0], ds @ k, e_ds @ k.abs()), ("dk", grads[1], shared(back(ds) @ q), shared(back(e_ds) @ q.abs())),
                                   ("dv", grads[2], shared(back(p) @ do), shared(back(p * (u + e_pb)) @ do.abs()))):
        wrong = (four(got) - want).abs() / (1.05 * (bound + u * want.abs()) + 1e-6)
        assert (wrong <= 1).all(), (what, float(wrong.max()))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form,power", [((0.0475536, 0.0531143), 3), ((0.1327098, 0.1332105), 2)])
def test_caps_where_one_form_loses_a_coefficient_and_the_other_does_not(form, power, D):
    """Coefficient c_i of a form is c_i log2(e) cap (scale / cap)^(2 i + 1): at this cap the shorter form's is below the normal fp32 numbers."""
    scale = D**-0.5
    low, high = ((c * 1.442695 * scale ** (2 * power + 1) / torch.finfo(torch.float32).tiny) ** (1 / (2 * power)) for c in form)
    cap = (low * high) ** 0.5
    assert low < cap < high
    B, S, H, G = 1, 200, 2, 1
    q, k, v, _ = _spread(B, S, H, G, D, 10.0, 7)
    q = (q.double() * (cap / 60)).bfloat16()  # the largest scores about a third of the cap
    flat = lambda t: t.reshape(B * S, -1)  # noqa: E731
    out, lse = torch.empty_like(flat(q)), torch.empty(B, H, S, device="cuda")
    K.attention_fwd(flat(q), flat(k), flat(v), B, S, H, G, D, out, lse, softcap=cap)
    K.check_status(q.device)
    q, k = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(H // G, 1)
    s = (cap * torch.tanh(q @ k.transpose(-1, -2) * scale / cap)).masked_fill(~torch.ones(S, S, dtype=torch.bool, device="cuda").tril(), -math.inf)
    assert 0.1 * cap < s.max() < 0.4 * cap  # the short form's
    sizes = (q.abs() @ k.abs().transpose(-1, -2)).amax(-1) * scale
    want = torch.logsumexp(s, -1)
    assert ((lse.double() - want).abs() <= 2.0**-21 * sizes + 2.0**-20 * want.abs()).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [0.05, 1.0])
@pytest.mark.parametrize("cap", [1e12, 1e20, 1e30])
def test_caps_and_scores_beyond_sense(cap, size, D):
    """Scores below and about the cap, whose squares are no fp32 numbers any more."""
    B, S, H, G = 1, 200, 2, 1
    q, k, v, _ = _spread(B, S, H, G, D, 10.0, 2)
    q = q * size
    q, k = (q.double() * cap**0.5).bfloat16(), (k.double() * cap**0.5).bfloat16()
    flat = lambda t: t.reshape(B * S, -1)  # noqa: E731
    out, lse = torch.empty_like(flat(q)), torch.empty(B, H, S, device="cuda")
    K.attention_fwd(flat(q), flat(k), flat(v), B, S, H, G, D, out, lse, softcap=cap)
    K.check_status(q.device)
    q, k = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(H // G, 1)
    s = (cap * torch.tanh(q @ k.transpose(-1, -2) * D**-0.5 / cap)).masked_fill(~torch.ones(S, S, dtype=torch.bool, device="cuda").tril(), -math.inf)
    sizes = (q.abs() @ k.abs().transpose(-1, -2)).amax(-1) * D**-0.5
    assert out.isfinite().all()
    # the largest score, to 2^-21 of its terms and 2^-20 of itself
    want = torch.logsumexp(s, -1)
    assert ((lse.double() - want).abs() <= 2.0**-21 * sizes + 2.0**-20 * want.abs()).all()


# ------------------------------------------------------------------ rotation


@pytest.mark.parametrize("half", [False, True])
def test_rotation_by_angles_of_more_than_24_bits(half):
    """Of the pair (1, 0) the cosine and the sine are left, each within two steps of itself: one of the functions, half a one of what is added for the
    angle's further bits, half a one to spare; the product of position and frequency is off by 2^-53 of itself, thrice."""
    T, dim, n = 20000, 128, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    inv, axis = K.rope_axes_freqs([dim // 2], 10000.0, "cuda")
    pos = torch.randint(0, 1 << 14, (1, T), dtype=torch.int32, device="cuda", generator=g)
    buf = torch.zeros(T, n, dim, device="cuda")
    x, y = (buf[..., : dim // 2], buf[..., dim // 2 :]) if half else (buf[..., 0::2], buf[..., 1::2])
    x.fill_(1.0)
    K.rope_axes_(buf.view(T, n * dim), pos, inv, axis, n, dim, half=half)
    angle = (pos.double().t() * inv)[:, None]
    for got, want in ((x, angle.cos()), (y, angle.sin())):
        assert ((got.double() - want).abs() <= 2 * 2.0**-23 * want.abs() + 3 * 2.0**-53 * 2**14).all()
