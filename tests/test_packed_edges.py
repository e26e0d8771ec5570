"""Packed-batch operators at the edges of what their entries take, without a GPU."""
import concurrent.futures
import math
import re
import subprocess

import pytest
import torch

from torchft_b200 import _build
from torchft_b200.ops import kernels as K


def test_the_masked_attention_kernels_keep_nothing_in_local_memory(tmp_path):
    """Their warpgroups share out registers, and no value of one share lies where another looks for it: the compiler's own report."""

    def report(name):
        src = _build.CSRC / "kernels" / f"{name}.cu"
        cmd = [_build._nvcc(), *_build.NVCC_FLAGS, f"-I{_build.CSRC / 'kernels'}", "-Xptxas", "-v", "-c", str(src), "-o", str(tmp_path / f"{name}.o")]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        assert proc.returncode == 0, proc.stderr
        return re.findall(r"Compiling entry function '(\S+)'.*?(\d+) bytes stack frame, (\d+) bytes spill stores, (\d+) bytes spill loads",
                          proc.stdout + proc.stderr, re.S)

    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        fwd, bwd = pool.map(report, ("attention_masked_fwd_tcgen05", "attention_bwd_tcgen05"))
    assert len(fwd) == 4
    masked = fwd + [r for r in bwd if "ELb1E" in r[0]]
    assert len(masked) == 8
    assert all(r[1:] == ("0", "0", "0") for r in masked), masked


# ------------------------------------------------------------------ padding


def _packed(B, S, H, G, D, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B * S, (H + 2 * G) * D, generator=g).to(torch.bfloat16)
    return qkv, torch.randn(B * S, H * D, generator=g).to(torch.bfloat16)


def _parts(t, H, G, D):
    return t[:, : H * D], t[:, H * D : (H + G) * D], t[:, (H + G) * D :]


def _both(qkv, do, B, S, H, G, D, **how):
    out, lse, d = torch.full_like(do, 7.0), torch.full((B, H, S), 7.0), torch.full_like(qkv, 7.0)
    K.attention_fwd(*_parts(qkv, H, G, D), B, S, H, G, D, out, lse, **how)
    K.attention_bwd(*_parts(qkv, H, G, D), out, do, lse, *_parts(d, H, G, D), B, S, H, G, D, **how)
    return out, lse, d


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("cap,slopes", [(0.0, None), (20.0, None), (0.0, 0.25)])
def test_padding_may_hold_anything(bad, cap, slopes):
    B, S, H, G, D = 2, 64, 4, 2, 64
    qkv, do = _packed(B, S, H, G, D, 5)
    ids = (torch.arange(S).expand(B, S) // 13).to(torch.int32).contiguous()
    ids[:, 40:] = -1
    ids[1, 7:9] = -2
    how = {"spans": K.attention_spans(ids), "softcap": cap, "slopes": None if slopes is None else torch.full((H,), slopes)}
    dead = (ids < 0).view(-1)
    clean = _both(qkv, do, B, S, H, G, D, **how)
    qkv[dead], do[dead] = bad, bad
    dirty = _both(qkv, do, B, S, H, G, D, **how)
    for x, y in zip(clean, dirty):
        assert torch.equal(x, y)
    assert not dirty[0][dead].any() and not dirty[2][dead].any()
    assert (dirty[1].transpose(1, 2)[ids < 0] == -math.inf).all()


# ------------------------------------------------------------------ results of a layer norm


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_layernorm_in_the_place_of_its_input_has_no_h(device):
    x, w, res = torch.randn(5, 16, device=device), torch.randn(16, device=device), torch.randn(5, 16, device=device)
    want, mean, rstd, h = K.layernorm_fwd(x, w)
    assert h is x or torch.equal(h, x)
    y = x.clone()
    out, _, _, h = K.layernorm_fwd(y, w, out=y)
    assert h is None and out.data_ptr() == y.data_ptr() and torch.equal(y, want)
    y = x.clone()
    assert K.layernorm_fwd(y, w, out=y.view(-1).view(5, 16))[3] is None  # the same memory as another tensor
    y = x.clone()
    out, _, _, h = K.layernorm_fwd(y, w, res=res, out=y)
    assert h is not None and torch.equal(h, x + res)


@pytest.mark.parametrize("device", DEVICES)
def test_results_of_a_layernorm_that_share_memory_are_refused(device):
    T, D = 6, 16
    buf = torch.randn(4 * T * D, device=device)
    x, shifted, res = buf[: T * D].view(T, D), buf[D : D + T * D].view(T, D), buf[2 * T * D : 3 * T * D].view(T, D)
    w, s = torch.randn(D, device=device), torch.randn(T, device=device)
    fwd = lambda **how: K.layernorm_fwd(x, w, **how)  # noqa: E731
    free = torch.empty_like(x)
    for how in ({"out": shifted}, {"res": res, "h_out": shifted}, {"res": res, "out": free, "h_out": free.view(-1).view(T, D)},
                {"mean": s, "rstd": s.view(1, -1).view(-1)}, {"mean": buf[:T]}, {"rstd": buf[3:3 + T]}):
        with pytest.raises(ValueError):
            fwd(**how)
    with pytest.raises(ValueError):
        K.layernorm_fwd(x, buf[:D], out=x)  # the weight lies in what is written
    _, mean, rstd, _ = fwd()
    dy = torch.randn_like(x)
    g = torch.empty(D, device=device)
    for how in ({"dx": shifted}, {"dw": w}, {"db": dy[0]}, {"dw": g, "db": g}, {"dw": g, "db": g.view(1, -1).view(-1)}, {"dx": free, "dw": free.view(-1)[:D]}):
        with pytest.raises(ValueError):
            K.layernorm_bwd(dy, x, w, mean, rstd, **how)


# ------------------------------------------------------------------ the same answer on both devices


@pytest.mark.parametrize("device", DEVICES)
def test_sizes_that_no_kernel_takes_are_refused_everywhere(device):
    pos = torch.zeros(1, 4, dtype=torch.int32, device=device)
    for dtype, dim, half in ((torch.bfloat16, 12, False), (torch.bfloat16, 8, True), (torch.bfloat16, 24, True), (torch.float32, 6, False),
                             (torch.float32, 4, True), (torch.float32, 12, True), (torch.float32, 1028, False), (torch.bfloat16, 0, False)):
        inv, axis = torch.ones(dim // 2, dtype=torch.float64, device=device), torch.zeros(dim // 2, dtype=torch.int32, device=device)
        with pytest.raises(ValueError, match="head_dim"):
            K.rope_axes_(torch.zeros(4, max(dim, 1), dtype=dtype, device=device), pos, inv, axis, 1, dim, half=half)
    inv, axis = K.rope_axes_freqs([8], 10.0, device)
    for dtype, width in ((torch.bfloat16, 20), (torch.float32, 18)):
        with pytest.raises(ValueError, match="apart"):
            K.rope_axes_(torch.zeros(4, width, dtype=dtype, device=device), pos, inv, axis, 1, 16)
    x, w = torch.zeros(2, 16392, device=device), torch.zeros(16392, device=device)
    with pytest.raises(ValueError, match="16384"):
        K.layernorm_fwd(x, w)
    with pytest.raises(ValueError, match="16384"):
        K.layernorm_bwd(x, x, w, x[:, 0].contiguous(), x[:, 0].contiguous())


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_share_memory_are_refused(device):
    B, S, H, D = 1, 4, 2, 64
    q = torch.zeros(S, H * D, dtype=torch.bfloat16, device=device)
    same = torch.zeros(1, H * D, dtype=torch.bfloat16, device=device).expand(S, H * D)
    lse = torch.zeros(B, H, S, device=device)
    for args in ((same, q, q, q), (q, same, q, q), (q, q, same, q), (q, q, q, same)):
        with pytest.raises(ValueError, match="apart"):
            K.attention_fwd(*args[:3], B, S, H, H, D, args[3], lse, softcap=10.0)
    for i in range(8):
        args = [q] * 8
        args[i] = same
        with pytest.raises(ValueError, match="apart"):
            K.attention_bwd(*args[:5], lse, *args[5:], B, S, H, H, D, softcap=10.0)


@pytest.mark.parametrize("device", DEVICES)
def test_one_row_has_no_stride(device):
    """What a single row's stride says means nothing: a column of another tensor, a width that is no multiple."""
    H, D = 2, 64
    g = torch.Generator().manual_seed(0)
    qkv = [torch.randn(H * D, 1, generator=g).to(device, torch.bfloat16) for _ in range(4)]
    flat = [t.view(1, -1) for t in qkv]
    odd = [t.t() for t in qkv]  # strides (1, 1)
    want, got = torch.empty_like(flat[0]), torch.empty(H * D, 1, dtype=torch.bfloat16, device=device).t()
    lse = torch.empty(1, H, 1, device=device)
    K.attention_fwd(*flat[:3], 1, 1, H, H, D, want, lse, softcap=10.0)
    K.attention_fwd(*odd[:3], 1, 1, H, H, D, got, lse, softcap=10.0)
    assert torch.equal(got, want)
    d, e = [torch.empty_like(t) for t in flat[:3]], [torch.empty(H * D, 1, dtype=torch.bfloat16, device=device).t() for _ in range(3)]
    K.attention_bwd(*flat[:3], want, flat[3], lse, *d, 1, 1, H, H, D, softcap=10.0)
    K.attention_bwd(*odd[:3], got, odd[3], lse, *e, 1, 1, H, H, D, softcap=10.0)
    assert all(torch.equal(x, y) for x, y in zip(d, e))
    inv, axis = K.rope_axes_freqs([8], 10.0, device)
    pos = torch.tensor([[5]], dtype=torch.int32, device=device)
    buf = torch.randn(1, 2 * 16 + 3, generator=g).to(device)
    even = buf[:, :32].contiguous()
    K.rope_axes_(buf, pos, inv, axis, 2, 16)
    assert torch.equal(buf[:, :32], K.rope_axes_(even, pos, inv, axis, 2, 16))


def test_the_reference_page_explains_every_argument_of_a_mask():
    page = (_build.REPO_DIR / "docs" / "api.md").read_text()
    for name in ("attention_fwd", "attention_bwd", "attention_spans"):
        text = page.split(f"### `{name}(", 1)[1].split("\n", 1)[1].split("\n### ", 1)[0]
        for arg in ("documents", "prefix", "causal", "window") if name == "attention_spans" else ("spans", "softcap", "slopes"):
            assert f"``{arg}``" in text, (name, arg)


@pytest.mark.parametrize("device", DEVICES)
def test_a_table_of_other_positions_is_refused(device):
    B, S, H, D = 1, 6, 2, 64
    q, lse = torch.zeros(B * S, H * D, dtype=torch.bfloat16, device=device), torch.zeros(B, H, S, device=device)
    call = lambda rope: K.attention_bwd(q, q, q, q, q, lse, *(torch.empty_like(q) for _ in range(3)), B, S, H, H, D, softcap=9.0, rope=rope)  # noqa: E731
    table = K.rope_table(S, D, 1e4, device)
    call(table)
    for bad in (table[:-1], table[:, :-1], table.double(), table.transpose(0, 1), table[0]):
        with pytest.raises(ValueError, match="rope"):
            call(bad)
