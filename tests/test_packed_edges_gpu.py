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
