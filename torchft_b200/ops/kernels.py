"""Python entry points of the sm_100a kernels, with plain-PyTorch references.

Every public function dispatches on the device of its arguments:

* CUDA tensors run the hand-written kernel from ``libftb200_kernels.so`` on the
  current stream (never an eager fallback);
* CPU tensors run the ``ref_*`` function of the same name, an fp32 PyTorch
  restatement of the kernel's math.  The ``ref_*`` functions are also the oracles of
  the GPU numerics tests.
"""

from __future__ import annotations

import ctypes
import functools
import math
import os
from typing import Optional, Sequence, Tuple

import torch
import torch.nn.functional as F

from . import _native as N
from ._native import c_float, c_int, c_ll, c_void_p, ptr, stream_ptr

# --------------------------------------------------------------------------- status word

_status_words: dict = {}


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 word that kernels with bounded waits write a code into."""
    key = (device.type, device.index)
    w = _status_words.get(key)
    if w is None:
        w = torch.zeros(1, dtype=torch.int32, device=device)
        _status_words[key] = w
    return w


_status_ptrs: dict = {}


def _status_ptr(device: torch.device) -> int:
    at = _status_ptrs.get(device.index)
    if at is None:
        at = _status_ptrs[device.index] = status_word(device).data_ptr()
    return at


# The C functions get their argument types once and take plain numbers from then on: a ctypes object per argument and call
# is a tenth of the host's time for a launch (the prompt pass of two layers of width 256: 257 to 299 -> 250 us).
_ARGS = {
    "embedding_fwd": "pppiiip", "embedding_bwd": "pppiiip", "rmsnorm_fwd": "ppppppiifp", "rmsnorm_bwd": "ppppppppiiip",
    "rope": "ppliiilip", "swiglu_fwd": "pplip", "swiglu_bwd": "ppplip", "gemm_bf16_swiglu": "ppppiiillllpip",
    "gemm_bf16_dswiglu": "pppiiilllpp", "gemm_bf16_loss": "ppiiillppppp",
    "cross_entropy": "pppiilfip", "adamw": "ppppiplfffffipp", "sumsq": "pilpp", "clip_coef": "pfppp",
    "attention_fwd": "pppppiiiiillllfipp", "attention_fwd2": "pppppiiiiillllfiipp",
    "attention_bwd": "ppppppppppiiiiillllllllfippp", "gemm_bf16": "pppiiiiilllipip",
    "attention_spans": "ppppppiiiip", "attention_masked_fwd": "pppppppppiiiiillllffipp",
    "attention_masked_bwd": "ppppppppppppppiiiiillllllllffippp", "rope_axes": "ppppliiiliiip",
    "layernorm_fwd": "pppppppplifip", "layernorm_bwd": "ppppppppppliiipp",
}
_ARGS["gemm_bf16_2cta"] = _ARGS["gemm_bf16"]
_KIND = {"p": c_void_p, "i": c_int, "l": c_ll, "f": c_float}


def _fn(name: str):
    fn = getattr(N.lib(), "ftb200_" + name)
    if fn.argtypes is None:
        fn.argtypes = [_KIND[k] for k in _ARGS[name]]
    return fn


def _at(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def check_status(device: torch.device) -> None:
    """Synchronising read of the status word; raises if any kernel reported a failure."""
    w = status_word(device)
    code = int(w.item())
    if code != 0:
        w.zero_()
        raise N.KernelError(f"device-side status: {N.STATUS.get(code, code)}")


# --------------------------------------------------------------------------- GEMM


def _check_2d_bf16(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or t.dtype != torch.bfloat16 or t.stride(1) != 1:
        raise ValueError(f"{name} must be a 2-D bf16 tensor with unit inner stride")


# Which GEMM kernel `gemm` launches: "2cta" (pairs of CTAs, tcgen05.mma.cta_group::2) or
# "1cta".  Overridable per call and through the FTB200_GEMM environment variable.
GEMM_IMPL = os.environ.get("FTB200_GEMM", "2cta")


def gemm(
    a: torch.Tensor,
    b: torch.Tensor,
    a_mn_major: bool = False,
    b_mn_major: bool = False,
    out: Optional[torch.Tensor] = None,
    accumulate: bool = False,
    out_dtype: torch.dtype = torch.bfloat16,
    max_ctas: int = 0,
    impl: Optional[str] = None,
) -> torch.Tensor:
    """``out (+)= A @ B^T`` with logical ``A [M,K]`` and ``B [N,K]``.

    ``a_mn_major`` says ``a`` is stored as the row-major ``[K, M]`` matrix (and likewise
    for ``b``), which is how the dgrad and wgrad GEMMs of a linear layer read their
    operands without transposed copies.
    """
    _check_2d_bf16(a, "a")
    _check_2d_bf16(b, "b")
    if a_mn_major:
        K, M = a.shape
    else:
        M, K = a.shape
    if b_mn_major:
        Kb, Nn = b.shape
    else:
        Nn, Kb = b.shape
    if K != Kb:
        raise ValueError(f"reduction dims differ: {K} vs {Kb}")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs an output tensor")
        out = torch.empty(M, Nn, dtype=out_dtype, device=a.device)
    if out.shape != (M, Nn) or out.stride(1) != 1 or out.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("bad output tensor")
    if not a.is_cuda:
        af = a.float().t() if a_mn_major else a.float()
        bf = b.float() if b_mn_major else b.float().t()
        r = af @ bf
        if accumulate:
            r = r + out.float()
        out.copy_(r.to(out.dtype))
        return out
    flags = (1 if out.dtype == torch.float32 else 0) | (2 if accumulate else 0)
    rc = _fn("gemm_bf16_2cta" if (impl or GEMM_IMPL) == "2cta" else "gemm_bf16")(
        a.data_ptr(), b.data_ptr(), out.data_ptr(), M, Nn, K, int(a_mn_major), int(b_mn_major), a.stride(0), b.stride(0),
        out.stride(0), flags, _status_ptr(a.device), max_ctas, _stream(),
    )
    N.check(rc, "gemm_bf16")
    return out


class ScatterField:
    """Destination of a weight-gradient GEMM whose epilogue performs the reduce-scatter's
    transfer: a ``[rows, cols]`` field at element offset ``unit_off`` of a flat gradient unit
    sharded over ``world`` ranks; ``peers`` are the ranks' staging areas (``[world, shard]``)."""

    def __init__(self, peers, world: int, src_rank: int, shard_elems: int, unit_off: int, shape) -> None:
        self.peers, self.world, self.src_rank = peers, world, src_rank
        self.shard_elems, self.unit_off, self.shape = shard_elems, unit_off, tuple(shape)


def gemm_scatter(a: torch.Tensor, b: torch.Tensor, a_mn_major: bool, b_mn_major: bool, dst: ScatterField) -> None:
    """``A @ B^T`` written straight into the owners' staging areas (see :class:`ScatterField`)."""
    _check_2d_bf16(a, "a")
    _check_2d_bf16(b, "b")
    K_, M = a.shape if a_mn_major else a.shape[::-1]
    Kb, Nn = b.shape if b_mn_major else b.shape[::-1]
    if K_ != Kb or (M, Nn) != dst.shape:
        raise ValueError(f"shape mismatch: {(M, Nn)} vs field {dst.shape}")
    rc = N.lib().ftb200_gemm_bf16_scatter(
        ptr(a), ptr(b), c_int(M), c_int(Nn), c_int(K_), c_int(int(a_mn_major)), c_int(int(b_mn_major)), c_ll(a.stride(0)),
        c_ll(b.stride(0)), dst.peers, c_int(dst.world), c_int(dst.src_rank), c_ll(dst.shard_elems), c_ll(dst.unit_off),
        ptr(status_word(a.device)), c_int(0), stream_ptr())
    N.check(rc, "gemm_bf16_scatter")


def scatter_to_stage(src: torch.Tensor, dst: ScatterField) -> None:
    """Copy a small bf16 field (e.g. a norm-weight gradient) to its owners' staging areas."""
    N.check(N.lib().ftb200_scatter_to_stage(ptr(src), c_ll(src.numel()), c_ll(dst.unit_off), c_ll(dst.shard_elems), dst.peers,
                                            c_int(dst.world), c_int(dst.src_rank), stream_ptr()), "scatter_to_stage")


class GatherField:
    """A weight that is still spread over its shard group: ``local`` is its ``[N, K]`` place in this rank's gathered
    copy of a flat parameter unit (``unit_off`` elements from the unit's start), ``peers`` the ranks' shard buffers
    of that unit (``shard_elems`` elements each).  The first forward GEMM that consumes the field gathers it while
    it multiplies (:func:`gemm_gather`) and clears ``pending``; from then on ``local`` is the gathered weight."""

    def __init__(self, local: torch.Tensor, peers, world: int, shard_elems: int, unit_off: int, sync: torch.Tensor) -> None:
        self.local, self.peers, self.world = local, peers, world
        self.shard_elems, self.unit_off, self.sync = shard_elems, unit_off, sync
        self.pending = True

    @staticmethod
    def supported(shape, shard_elems: int) -> bool:
        return len(shape) == 2 and shape[0] % 128 == 0 and shape[1] % 64 == 0 and shard_elems >= 8192 and shard_elems % 8 == 0


def gemm_gather(x: torch.Tensor, w: GatherField, out: torch.Tensor, aux: Optional[torch.Tensor] = None) -> None:
    """``out = x @ W^T`` with the all-gather of ``W`` fused into the GEMM: extra warps of the kernel pull ``W``'s
    rows out of the shard owners' memory over NVLink in tile order while the tensor cores already work on the
    rows that have arrived.  ``aux`` as in :func:`linear_swiglu_fwd`."""
    _check_2d_bf16(x, "x")
    Nn, Kd = w.local.shape
    T = x.shape[0]
    if x.shape[1] != Kd or tuple(out.shape) != (T, Nn) or w.sync.numel() < 1 + Nn // 128:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w {(Nn, Kd)}, out {tuple(out.shape)}")
    rc = N.lib().ftb200_gemm_bf16_gather(
        ptr(x), ptr(w.local), ptr(out), c_int(T), c_int(Nn), c_int(Kd), c_ll(x.stride(0)), c_ll(out.stride(0)), w.peers,
        c_int(w.world), c_ll(w.shard_elems), c_ll(w.unit_off), ptr(w.sync), ptr(aux) if aux is not None else None,
        c_ll(aux.stride(0) if aux is not None else 0), ptr(status_word(x.device)), c_int(0), stream_ptr())
    N.check(rc, "gemm_bf16_gather")
    w.pending = False


def linear_fwd(x: torch.Tensor, w, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y = x @ w^T`` (x ``[T,K]``, w ``[N,K]`` or a :class:`GatherField`)."""
    if isinstance(w, GatherField):
        if w.pending:
            if out is None:
                out = torch.empty(x.shape[0], w.local.shape[0], dtype=x.dtype, device=x.device)
            gemm_gather(x, w, out)
            return out
        w = w.local
    return gemm(x, w, False, False, out=out)


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None,
                 accumulate: bool = False) -> torch.Tensor:
    """``dx = dy @ w`` (dy ``[T,N]``, w ``[N,K]``)."""
    return gemm(dy, w, False, True, out=out, accumulate=accumulate)


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, out: Optional[torch.Tensor] = None,
                 accumulate: bool = False, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dw = dy^T @ x`` (dy ``[T,N]``, x ``[T,K]``) -> ``[N,K]``.  ``out`` may be a
    :class:`ScatterField`: the result then goes straight to the shard owners."""
    if isinstance(out, ScatterField):
        if accumulate:
            raise ValueError("a scattered weight gradient cannot accumulate")
        gemm_scatter(dy, x, True, True, out)
        return out  # type: ignore[return-value]
    return gemm(dy, x, True, True, out=out, accumulate=accumulate, out_dtype=out_dtype)


# --------------------------------------------------------------------------- embedding


def embedding_fwd(tokens: torch.Tensor, table: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    T = tokens.numel()
    V, D = table.shape
    if out is None:
        out = torch.empty(T, D, dtype=table.dtype, device=table.device)
    if not table.is_cuda:
        out.copy_(table[tokens.reshape(-1)])
        return out
    N.check(_fn("embedding_fwd")(_at(tokens), _at(table), _at(out), T, D, V, _stream()),
            "embedding_fwd")
    return out


def embedding_bwd(tokens: torch.Tensor, dout: torch.Tensor, dtable: torch.Tensor) -> torch.Tensor:
    """``dtable[tokens[t]] += dout[t]`` (``dtable`` must be zeroed by the caller)."""
    T = tokens.numel()
    V, D = dtable.shape
    if not dtable.is_cuda:
        dtable.copy_(dtable.float().index_add_(0, tokens.reshape(-1), dout.float()).to(dtable.dtype))
        return dtable
    N.check(_fn("embedding_bwd")(_at(tokens), _at(dout), _at(dtable), T, D, V, _stream()),
            "embedding_bwd")
    return dtable


# --------------------------------------------------------------------------- RMSNorm


def ref_rmsnorm_fwd(x, w, eps, res=None):
    h = x.float()
    if res is not None:
        h = (h + res.float()).to(x.dtype).float()
    rstd = torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    return (h * rstd * w.float()).to(x.dtype), rstd.squeeze(-1), h.to(x.dtype)


def rmsnorm_fwd(
    x: torch.Tensor,
    w: torch.Tensor,
    eps: float = 1e-5,
    res: Optional[torch.Tensor] = None,
    h_out: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    rstd: Optional[torch.Tensor] = None,
    want_out: bool = True,
) -> Tuple[Optional[torch.Tensor], torch.Tensor, torch.Tensor]:
    """Returns ``(normed, rstd, h)`` where ``h = x + res`` (or ``x``)."""
    T, D = x.shape
    if rstd is None:
        rstd = torch.empty(T, dtype=torch.float32, device=x.device)
    if res is not None and h_out is None:
        h_out = torch.empty_like(x)
    if want_out and out is None:
        out = torch.empty_like(x)
    if not x.is_cuda:
        o, r, h = ref_rmsnorm_fwd(x, w, eps, res)
        rstd.copy_(r)
        if res is not None:
            h_out.copy_(h)
        if want_out:
            out.copy_(o)
        return (out if want_out else None), rstd, (h_out if res is not None else x)
    N.check(
        _fn("rmsnorm_fwd")(_at(x), _at(res), _at(h_out), _at(w), _at(out if want_out else None), _at(rstd), T, D, eps, _stream()),
        "rmsnorm_fwd",
    )
    return (out if want_out else None), rstd, (h_out if res is not None else x)


def ref_rmsnorm_bwd(dy, x, w, rstd, dres=None):
    dyf, xf, wf = dy.float(), x.float(), w.float()
    r = rstd.float().unsqueeze(-1)
    D = x.shape[-1]
    dot = (dyf * wf * xf).sum(-1, keepdim=True)
    dx = r * wf * dyf - xf * dot * r.pow(3) / D
    if dres is not None:
        dx = dx + dres.float()
    dw = (dyf * xf * r).sum(0)
    return dx.to(x.dtype), dw


_rms_scratch: dict = {}


@functools.lru_cache(maxsize=256)
def rmsnorm_bwd_scratch_floats(dim: int) -> int:
    """Size of the ``scratch`` that :func:`rmsnorm_bwd` takes."""
    lib = N.lib()
    lib.ftb200_rmsnorm_bwd_scratch_floats.restype = c_ll
    return int(lib.ftb200_rmsnorm_bwd_scratch_floats(dim))


def rmsnorm_bwd(
    dy: torch.Tensor,
    x: torch.Tensor,
    w: torch.Tensor,
    rstd: torch.Tensor,
    dres: Optional[torch.Tensor] = None,
    dx: Optional[torch.Tensor] = None,
    dw: Optional[torch.Tensor] = None,
    accumulate_dw: bool = False,
    scratch: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(dx, dw)`` of :func:`rmsnorm_fwd`.  The partial sums of ``dw`` lie in ``scratch`` (fp32 on the device,
    :func:`rmsnorm_bwd_scratch_floats` of them or more) between the two kernels, by default in a buffer of the current stream's
    that is reused across calls."""
    T, D = x.shape
    if dx is None:
        dx = torch.empty_like(x)
    if dw is None:
        dw = torch.zeros(D, dtype=w.dtype, device=x.device)
    if not x.is_cuda:
        rdx, rdw = ref_rmsnorm_bwd(dy, x, w, rstd, dres)
        dx.copy_(rdx)
        dw.copy_(((dw.float() if accumulate_dw else 0) + rdw).to(dw.dtype))
        return dx, dw
    if scratch is None:
        key = (x.device.index, _stream(), D)
        scratch = _rms_scratch.get(key)
        if scratch is None:
            scratch = _rms_scratch[key] = torch.empty(rmsnorm_bwd_scratch_floats(D), dtype=torch.float32, device=x.device)
    elif (scratch.device != x.device or scratch.dtype != torch.float32 or not scratch.is_contiguous()
          or scratch.numel() < rmsnorm_bwd_scratch_floats(D) or scratch.data_ptr() % 16):
        raise ValueError(f"scratch must be {rmsnorm_bwd_scratch_floats(D)} contiguous fp32 on {x.device}")
    N.check(
        _fn("rmsnorm_bwd")(_at(dy), _at(x), _at(w), _at(rstd), _at(dres), _at(dx), _at(dw), _at(scratch), T, D,
                           int(accumulate_dw), _stream()),
        "rmsnorm_bwd",
        launches=2,
    )
    return dx, dw


# --------------------------------------------------------------------------- layer norm


def _check_like(names: str, dtype: torch.dtype, shape, device: int, *tensors: Optional[torch.Tensor]) -> None:
    """Each of ``tensors`` that is not None is contiguous, of the type and shape, and on the device (-1: the CPU)."""
    for i, t in enumerate(tensors):
        if t is not None and (t.dtype != dtype or t.shape != shape or t.get_device() != device or t.is_meta or not t.is_contiguous()):
            where = "the CPU" if device < 0 else f"cuda:{device}"
            raise ValueError(f"{names.split()[i]} must be contiguous {dtype} of shape {tuple(shape)} on {where}, got {t.dtype} of {tuple(t.shape)} "
                             f"on {t.device}")


def _check_norm(x: torch.Tensor) -> None:
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float32) or x.shape[1] % 8 or not 0 < x.shape[1] <= 16384:
        raise ValueError("x must be [rows, width] in bf16 or fp32 with a width that is a multiple of 8 up to 16384")


def _result_apart(name: str, r: Optional[torch.Tensor], place: dict, others: dict) -> None:
    """A result (contiguous, like the others) is no part of what is read at other times than it is written, and of no other result.  ``place``: what
    it may be written over, as a whole."""
    if r is None or r.numel() == 0:
        return
    for as_a_whole, tensors in ((True, place), (False, others)):
        for what, t in tensors.items():
            if t is None or t.numel() == 0 or t.data_ptr() >= r.data_ptr() + r.nbytes or r.data_ptr() >= t.data_ptr() + t.nbytes:
                continue
            if not as_a_whole:
                raise ValueError(f"{name} and {what} share memory")
            if t.data_ptr() != r.data_ptr():
                raise ValueError(f"{name} may be {what} as a whole, but no part of its memory")


def ref_layernorm_fwd(x, w, b=None, eps=1e-5, res=None):
    h = x.float()
    if res is not None:
        h = (h + res.float()).to(x.dtype).float()
    mean = h.mean(-1)
    c = h - mean.unsqueeze(-1)
    rstd = torch.rsqrt(c.pow(2).mean(-1) + eps)
    y = c * rstd.unsqueeze(-1) * w.float()
    return (y if b is None else y + b.float()).to(x.dtype), mean, rstd, h.to(x.dtype)


def layernorm_fwd(
    x: torch.Tensor,
    w: torch.Tensor,
    b: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    res: Optional[torch.Tensor] = None,
    h_out: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    mean: Optional[torch.Tensor] = None,
    rstd: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Returns ``(normed, mean, rstd, h)`` where ``h = x + res`` (or ``x``), rounded to the type of ``x``, and ``normed = (h - mean) *
    rstd * w (+ b)``.  Rows of up to 16384 elements, all tensors in bf16 or all in fp32 (``mean`` and ``rstd`` in fp32).  ``out`` and
    ``h_out`` may be ``x`` or ``res`` as a whole; results share no other memory.  Without ``res`` and with ``out`` in the place of ``x``
    there is no ``h`` any more, and None stands for it."""
    if x.is_cuda:
        results = N.host().layernorm_fwd(x, w, b, eps, res, h_out, out, mean, rstd)
        N.launch_count += x.shape[0] > 0
        return results
    _check_norm(x)
    T, D = x.shape
    if mean is None:
        mean = torch.empty(T, dtype=torch.float32, device=x.device)
    if rstd is None:
        rstd = torch.empty(T, dtype=torch.float32, device=x.device)
    if res is not None and h_out is None:
        h_out = torch.empty_like(x)
    if out is None:
        out = torch.empty_like(x)
    dtype, at = x.dtype, x.get_device()
    _check_like("x res h_out out", dtype, x.shape, at, x, res, h_out, out)
    _check_like("w b", dtype, (D,), at, w, b)
    _check_like("mean rstd", torch.float32, (T,), at, mean, rstd)
    inputs, rows = {"x": x, "res": res}, {"w": w, "b": b, "mean": mean, "rstd": rstd}
    _result_apart("out", out, inputs, {**rows, "h_out": h_out if res is not None else None})
    _result_apart("h_out", h_out if res is not None else None, inputs, rows)
    _result_apart("mean", mean, {}, {**inputs, "w": w, "b": b, "rstd": rstd})
    _result_apart("rstd", rstd, {}, {**inputs, "w": w, "b": b})
    gone = res is None and out.data_ptr() == x.data_ptr() and x.numel() > 0
    o, m, r, h = ref_layernorm_fwd(x, w, b, eps, res)
    out.copy_(o)
    mean.copy_(m)
    rstd.copy_(r)
    if res is not None:
        h_out.copy_(h)
    return out, mean, rstd, h_out if res is not None else None if gone else x


def ref_layernorm_bwd(dy, x, w, mean, rstd, dres=None):
    xh = (x.float() - mean.unsqueeze(-1)) * rstd.unsqueeze(-1)
    dyf = dy.float()
    g = dyf * w.float()
    dx = rstd.unsqueeze(-1) * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    if dres is not None:
        dx = dx + dres.float()
    return dx.to(x.dtype), (dyf * xh).sum(0), dyf.sum(0)


@functools.lru_cache(maxsize=256)
def layernorm_bwd_scratch_floats(dim: int) -> int:
    """Size of the ``scratch`` that :func:`layernorm_bwd` takes."""
    lib = N.lib()
    lib.ftb200_layernorm_bwd_scratch_floats.restype = c_ll
    return int(lib.ftb200_layernorm_bwd_scratch_floats(dim))


def layernorm_bwd(
    dy: torch.Tensor,
    x: torch.Tensor,
    w: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    dres: Optional[torch.Tensor] = None,
    dx: Optional[torch.Tensor] = None,
    dw: Optional[torch.Tensor] = None,
    db: Optional[torch.Tensor] = None,
    bias: bool = True,
    accumulate: bool = False,
    scratch: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``(dx, dw, db)`` of :func:`layernorm_fwd`, whose ``h`` is ``x`` here; ``db`` is None without ``bias``.  ``dres`` is added to ``dx``,
    which may be ``dy``, ``x`` or ``dres`` as a whole (results share no other memory); with ``accumulate`` the sums are added to what ``dw``
    and ``db`` hold.  The partial sums lie in ``scratch`` (fp32 on the device, :func:`layernorm_bwd_scratch_floats` of them or more) between
    the two kernels, by default in memory of this call's own."""
    if x.is_cuda:
        results = N.host().layernorm_bwd(dy, x, w, mean, rstd, dres, dx, dw, db, bias, accumulate, scratch, _status_ptr(x.device))
        N.launch_count += 2 * (x.shape[0] > 0)
        return results
    _check_norm(x)
    T, D = x.shape
    if accumulate and (dw is None or (bias and db is None)):
        raise ValueError("accumulate needs dw and db")
    if dx is None:
        dx = torch.empty_like(x)
    if dw is None:
        dw = torch.empty_like(w)
    if not bias:
        db = None
    elif db is None:
        db = torch.empty_like(w)
    dtype, at = x.dtype, x.get_device()
    _check_like("x dy dres dx", dtype, x.shape, at, x, dy, dres, dx)
    _check_like("w dw db", dtype, (D,), at, w, dw, db)
    _check_like("mean rstd", torch.float32, (T,), at, mean, rstd)
    _result_apart("dx", dx, {"dy": dy, "x": x, "dres": dres}, {"w": w, "mean": mean, "rstd": rstd, "dw": dw, "db": db})
    for name, t in (("dw", dw), ("db", db)):
        _result_apart(name, t, {}, {"dy": dy, "x": x, "dres": dres, "w": w, "mean": mean, "rstd": rstd})
    _result_apart("dw", dw, {}, {"db": db})
    if T == 0:
        if not accumulate:
            dw.zero_()
            if db is not None:
                db.zero_()
        return dx, dw, db
    rdx, rdw, rdb = ref_layernorm_bwd(dy, x, w, mean, rstd, dres)
    dx.copy_(rdx)
    dw.copy_(((dw.float() if accumulate else 0) + rdw).to(dw.dtype))
    if db is not None:
        db.copy_(((db.float() if accumulate else 0) + rdb).to(db.dtype))
    return dx, dw, db


# --------------------------------------------------------------------------- RoPE


def rope_table(seq_len: int, head_dim: int, theta: float, device) -> torch.Tensor:
    """``[S, head_dim/2, 2]`` fp32 table of (cos, sin) for interleaved-pair rotation."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    ang = torch.outer(torch.arange(seq_len, dtype=torch.float64), inv)
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float().to(device).contiguous()


def ref_rope(buf, table, S, n_heads, head_dim, backward=False):
    T = buf.shape[0]
    rot = buf[:, : n_heads * head_dim].float().reshape(T, n_heads, head_dim // 2, 2)
    pos = torch.arange(T, device=buf.device) % S
    cs = table[pos].unsqueeze(1)  # T,1,Dh/2,2
    c, s = cs[..., 0], cs[..., 1]
    if backward:
        s = -s
    x0, x1 = rot[..., 0], rot[..., 1]
    o = torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], dim=-1).reshape(T, n_heads * head_dim)
    res = buf.clone()
    res[:, : n_heads * head_dim] = o.to(buf.dtype)
    return res


def rope_(buf: torch.Tensor, table: torch.Tensor, seq_len: int, n_heads: int, head_dim: int,
          backward: bool = False) -> torch.Tensor:
    """Rotate the first ``n_heads`` heads of every row of ``buf`` ``[T, >= n_heads*head_dim]`` in place."""
    T = buf.shape[0]
    if not buf.is_cuda:
        buf.copy_(ref_rope(buf, table, seq_len, n_heads, head_dim, backward))
        return buf
    N.check(
        _fn("rope")(_at(buf), _at(table), T, seq_len, n_heads, head_dim, buf.stride(0), int(backward), _stream()),
        "rope",
    )
    return buf


def rope_axes_freqs(sections: Sequence[int], theta: float, device, restart: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(inv_freq, axis)`` of :func:`rope_axes_` for a head whose first ``sections[0]`` pairs turn with the positions of axis 0, the next
    ``sections[1]`` with those of axis 1, and so on (time, height, width).  The frequencies fall from 1 to ``1 / theta`` over all pairs,
    or with ``restart`` over each section's own."""
    if not sections or any(n < 0 for n in sections) or sum(sections) == 0:
        raise ValueError("sections must be numbers of pairs, one per axis")
    total = sum(sections)
    inv, axis = [], []
    for a, n in enumerate(sections):
        at = torch.arange(n, dtype=torch.float64) / max(n, 1) if restart else (len(axis) + torch.arange(n, dtype=torch.float64)) / total
        inv.append(theta ** -at)
        axis += [a] * n
    return torch.cat(inv).to(device), torch.tensor(axis, dtype=torch.int32, device=device)


def ref_rope_axes(buf, positions, inv_freq, axis, n_heads, head_dim, half=False, backward=False):
    T, axes = buf.shape[0], positions.shape[0]
    turned = (axis >= 0) & (axis < axes)
    pos = positions.double()[axis.long().clamp(0, axes - 1)].t()  # [T, pairs]
    ang = torch.where(turned, pos * inv_freq, 0.0)
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    if backward:
        s = -s
    rot = buf[:, : n_heads * head_dim].float().reshape(T, n_heads, head_dim)
    x, y = (rot[..., : head_dim // 2], rot[..., head_dim // 2 :]) if half else (rot[..., 0::2], rot[..., 1::2])
    a, b = x * c - y * s, x * s + y * c
    o = torch.cat([a, b], -1) if half else torch.stack([a, b], -1)
    res = buf.clone()
    res[:, : n_heads * head_dim] = o.reshape(T, n_heads * head_dim).to(buf.dtype)
    return res


def rope_axes_(buf: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, axis: torch.Tensor, n_heads: int, head_dim: int,
               half: bool = False, backward: bool = False) -> torch.Tensor:
    """Rotate the first ``n_heads`` heads of every row of ``buf`` ``[T, >= n_heads*head_dim]`` (bf16 or fp32) in place by positions that
    the rows bring along: pair ``j`` of a head turns by ``positions[axis[j], t] * inv_freq[j]`` (``positions`` int32 ``[axes, T]``,
    ``inv_freq`` fp64 and ``axis`` int32, both ``[head_dim/2]``, see :func:`rope_axes_freqs`); an ``axis`` outside ``[0, axes)`` leaves the
    pair as it is.  Pairs are neighbours, as in :func:`rope_`, or with ``half`` elements ``j`` and ``j + head_dim/2``.  ``backward``
    turns back.  Heads and rows start on 16 bytes: ``head_dim`` is a multiple of 8 in bf16 and of 4 in fp32, with ``half`` of twice that, up
    to 1024, and so are the rows' strides of 8 and 4."""
    if buf.is_cuda:
        N.launch_count += N.host().rope_axes(buf, positions, inv_freq, axis, n_heads, head_dim, half, backward)
        return buf
    if buf.dim() != 2 or buf.dtype not in (torch.bfloat16, torch.float32) or (buf.shape[1] > 1 and buf.stride(1) != 1):
        raise ValueError("buf must be a 2-D bf16 or fp32 tensor with unit inner stride")
    T = buf.shape[0]
    vector = 4 if buf.dtype == torch.float32 else 8
    if not 0 < head_dim <= 1024 or head_dim % (2 * vector if half else vector):
        raise ValueError(f"head_dim must be a multiple of {2 * vector if half else vector} up to 1024 in {buf.dtype}{', half-split' if half else ''}")
    ld = buf.stride(0) if T > 1 else n_heads * head_dim  # of one row there is none
    if not 1 <= n_heads <= 1 << 20 or buf.shape[1] < n_heads * head_dim or ld < n_heads * head_dim:
        raise ValueError(f"buf of shape {tuple(buf.shape)} does not hold {n_heads} heads of {head_dim}")
    if ld % vector:
        raise ValueError(f"the rows of buf must start a multiple of {vector} elements apart")
    if positions.dim() != 2 or positions.shape[0] < 1:
        raise ValueError("positions must be contiguous int32 [axes, rows]")
    at = buf.get_device()
    _check_like("positions", torch.int32, (positions.shape[0], T), at, positions)
    _check_like("inv_freq", torch.float64, (head_dim // 2,), at, inv_freq)
    _check_like("axis", torch.int32, (head_dim // 2,), at, axis)
    if T > 0:
        buf.copy_(ref_rope_axes(buf, positions, inv_freq, axis, n_heads, head_dim, half, backward))
    return buf


# --------------------------------------------------------------------------- SwiGLU


def ref_swiglu_fwd(gu):
    """``gu`` rows are interleaved (gate, up) pairs."""
    g, u = gu[:, 0::2].float(), gu[:, 1::2].float()
    return (F.silu(g) * u).to(gu.dtype)


def swiglu_fwd(gu: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[:, j] = silu(gu[:, 2j]) * gu[:, 2j+1]`` (interleaved gate/up columns)."""
    T, F2 = gu.shape
    Fd = F2 // 2
    if out is None:
        out = torch.empty(T, Fd, dtype=gu.dtype, device=gu.device)
    if not gu.is_cuda:
        out.copy_(ref_swiglu_fwd(gu))
        return out
    N.check(_fn("swiglu_fwd")(_at(gu), _at(out), T, Fd, _stream()), "swiglu_fwd")
    return out


def ref_swiglu_bwd(ds, gu):
    g, u, d = gu[:, 0::2].float(), gu[:, 1::2].float(), ds.float()
    sg = torch.sigmoid(g)
    silu = g * sg
    out = torch.empty(gu.shape, dtype=torch.float32, device=gu.device)
    out[:, 0::2] = d * u * (sg + silu * (1 - sg))
    out[:, 1::2] = d * silu
    return out.to(gu.dtype)


def linear_dswiglu_(dy: torch.Tensor, w: torch.Tensor, gu: torch.Tensor, ds: torch.Tensor) -> None:
    """Backward of the down projection ``silu(gate) * up @ w^T`` into ``gu``, which holds the interleaved (gate, up) pairs and
    receives their gradients (:func:`linear_dgrad` into ``ds`` and :func:`swiglu_bwd` in place).  On the GPU it is one kernel
    from a width of 2048 on, and ``ds`` stays as it is: the gradient of the activation goes from the accumulator into the pairs
    without a rounding.  A product of fewer than 32 slabs does not hide the pairs' way in and out: 3000 rows, 2816 from 1024
    columns 31.7 -> 32.8 us; 4096 rows, 8192 from 2048 188 -> 154; 8192 rows, 14336 from 4096 758 -> 660."""
    T, F2 = gu.shape
    if (not dy.is_cuda or dy.shape[1] < 2048 or GEMM_IMPL != "2cta" or F2 % 16 or gu.stride(0) % 8 or gu.data_ptr() % 16 or gu.stride(0) < F2 or T < 1):
        if not gu.is_contiguous():
            raise ValueError("gu must be contiguous")
        linear_dgrad(dy, w, out=ds)
        swiglu_bwd(ds, gu, dgu=gu)
        return
    for t, name in ((dy, "dy"), (w, "w"), (gu, "gu")):
        _check_2d_bf16(t, name)
    if dy.shape[0] != T or tuple(w.shape) != (dy.shape[1], F2 // 2):
        raise ValueError(f"shape mismatch: dy {tuple(dy.shape)}, w {tuple(w.shape)}, gu {tuple(gu.shape)}")
    N.check(_fn("gemm_bf16_dswiglu")(dy.data_ptr(), w.data_ptr(), gu.data_ptr(), T, F2 // 2, dy.shape[1], dy.stride(0), w.stride(0),
                                     gu.stride(0), _status_ptr(dy.device), _stream()), "gemm_bf16_dswiglu")


def swiglu_bwd(ds: torch.Tensor, gu: torch.Tensor, dgu: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dgu`` may alias ``gu`` (in place)."""
    T, F2 = gu.shape
    if dgu is None:
        dgu = torch.empty_like(gu)
    if not gu.is_cuda:
        dgu.copy_(ref_swiglu_bwd(ds, gu))
        return dgu
    N.check(_fn("swiglu_bwd")(_at(ds), _at(gu), _at(dgu), T, F2 // 2, _stream()), "swiglu_bwd")
    return dgu


def linear_swiglu_fwd(x: torch.Tensor, w_gu: torch.Tensor, gu_out: torch.Tensor, s_out: torch.Tensor) -> None:
    """``gu_out = x @ w_gu^T`` and, from the same accumulator, ``s_out = silu(gate) * up``
    where ``w_gu``'s rows (``gu_out``'s columns) interleave gate and up."""
    if isinstance(w_gu, GatherField):
        if w_gu.pending:
            gemm_gather(x, w_gu, gu_out, aux=s_out)
            return
        w_gu = w_gu.local
    T, Kd = x.shape
    N2 = w_gu.shape[0]
    if not x.is_cuda or N2 % 32 or GEMM_IMPL != "2cta":
        gemm(x, w_gu, False, False, out=gu_out)
        swiglu_fwd(gu_out, out=s_out)
        return
    rc = _fn("gemm_bf16_swiglu")(
        _at(x), _at(w_gu), _at(gu_out), _at(s_out), T, N2, Kd, x.stride(0), w_gu.stride(0),
        gu_out.stride(0), s_out.stride(0), _status_ptr(x.device), 0, _stream())
    N.check(rc, "gemm_bf16_swiglu")


# --------------------------------------------------------------------------- cross-entropy


def ref_cross_entropy(logits, target, grad_scale):
    lf = logits.float()
    loss = F.cross_entropy(lf, target, reduction="none")
    p = torch.softmax(lf, dim=-1)
    p[torch.arange(lf.shape[0]), target] -= 1.0
    return loss, (p * grad_scale).to(logits.dtype)


def cross_entropy_(logits: torch.Tensor, target: torch.Tensor, grad_scale: float,
                   loss: Optional[torch.Tensor] = None, grad: bool = True) -> torch.Tensor:
    """Per-row loss; ``logits`` is overwritten by ``(softmax - onehot) * grad_scale`` (left as it is without ``grad``)."""
    T, V = logits.shape
    if loss is None:
        loss = torch.empty(T, dtype=torch.float32, device=logits.device)
    if not logits.is_cuda:
        l, g = ref_cross_entropy(logits, target, grad_scale)
        loss.copy_(l)
        if grad:
            logits.copy_(g)
        return loss
    N.check(
        _fn("cross_entropy")(_at(logits), _at(target), _at(loss), T, V, logits.stride(0), grad_scale, int(grad), _stream()),
        "cross_entropy",
    )
    return loss


def linear_loss_scratch_floats(rows: int, vocab: int) -> int:
    """Size of the ``scratch`` that :func:`linear_cross_entropy_` takes."""
    lib = N.lib()
    lib.ftb200_gemm_bf16_loss_scratch_floats.restype = c_ll
    return int(lib.ftb200_gemm_bf16_loss_scratch_floats(rows, vocab))


def linear_cross_entropy_(x: torch.Tensor, w, target: torch.Tensor, grad_scale: float, logits: torch.Tensor, loss: torch.Tensor,
                          grad: bool = True, scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`cross_entropy_` of the logits ``x @ w^T``.  With ``grad`` they end as their gradient in ``logits``; without it
    ``logits`` is a workspace that may or may not hold them afterwards: on the GPU the product's epilogue notes the rows' maxima,
    sums and target values (in fp32 ``scratch``, :func:`linear_loss_scratch_floats` of it or more) and they are not stored.  Not
    for fewer than 2^20 of them, where the second kernel costs more than it spares: 64 x 1024 8.7 -> 9.6 us, 750 x 8192 28 -> 24."""
    weight = w if not isinstance(w, GatherField) else None if w.pending else w.local
    T, Kd = x.shape
    V = logits.shape[1]
    if grad or weight is None or not x.is_cuda or GEMM_IMPL != "2cta" or V % 8 or T * V < 1 << 20:
        linear_fwd(x, w, out=logits)
        return cross_entropy_(logits, target, grad_scale, loss=loss, grad=grad)
    for t, name in ((x, "x"), (weight, "w"), (logits, "logits")):
        _check_2d_bf16(t, name)
    if tuple(weight.shape) != (V, Kd) or logits.shape[0] != T or target.numel() != T or loss.numel() != T:
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w {tuple(weight.shape)}, logits {tuple(logits.shape)}")
    if target.dtype != torch.int64 or not target.is_contiguous() or loss.dtype != torch.float32 or not loss.is_contiguous():
        raise ValueError("target must be contiguous int64, loss contiguous fp32")
    need = linear_loss_scratch_floats(T, V)
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.float32, device=x.device)
    elif scratch.device != x.device or scratch.dtype != torch.float32 or scratch.numel() < need or not scratch.is_contiguous():
        raise ValueError(f"scratch must be {need} contiguous fp32 on {x.device}")
    N.check(_fn("gemm_bf16_loss")(x.data_ptr(), weight.data_ptr(), T, V, Kd, x.stride(0), weight.stride(0), target.data_ptr(),
                                  loss.data_ptr(), scratch.data_ptr(), _status_ptr(x.device), _stream()), "gemm_bf16_loss",
            launches=2)
    return loss


# --------------------------------------------------------------------------- AdamW / grad norm


def ref_adamw(master, m, v, grad, lr, beta1, beta2, eps, wd, step, grad_scale=1.0):
    g = grad.float() * grad_scale
    m.mul_(beta1).add_(g, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2s = math.sqrt(1 - beta2 ** step)
    denom = v.sqrt() / bc2s + eps
    master.mul_(1 - lr * wd).addcdiv_(m, denom, value=-lr / bc1)


def adamw_(master: torch.Tensor, m: torch.Tensor, v: torch.Tensor, grad: torch.Tensor,
           param_lp: Optional[torch.Tensor], lr: float, beta1: float, beta2: float, eps: float, wd: float,
           step: int, grad_scale: Optional[torch.Tensor] = None) -> None:
    """One fused AdamW step over flat buffers (fp32 state, bf16 or fp32 grads, bf16 write-back)."""
    n = master.numel()
    if not master.is_cuda:
        gs = float(grad_scale.item()) if grad_scale is not None else 1.0
        ref_adamw(master.view(-1), m.view(-1), v.view(-1), grad.reshape(-1), lr, beta1, beta2, eps, wd, step, gs)
        if param_lp is not None:
            param_lp.view(-1).copy_(master.view(-1).to(param_lp.dtype))
        return
    N.check(
        _fn("adamw")(_at(master), _at(m), _at(v), _at(grad), int(grad.dtype == torch.float32), _at(param_lp), n, lr, beta1,
                     beta2, eps, wd, step, _at(grad_scale), _stream()),
        "adamw",
    )


def sumsq_(x: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """``out += sum(x^2)`` (``out`` is a 1-element fp32 tensor)."""
    if not x.is_cuda:
        out.add_(x.float().pow(2).sum())
        return out
    N.check(_fn("sumsq")(_at(x), int(x.dtype == torch.float32), x.numel(), _at(out), _stream()),
            "sumsq")
    return out


def clip_coef_(sumsq: torch.Tensor, max_norm: float, coef: torch.Tensor, norm_out: Optional[torch.Tensor] = None) -> None:
    if not sumsq.is_cuda:
        nrm = sumsq.sqrt()
        if norm_out is not None:
            norm_out.copy_(nrm)
        coef.copy_(torch.clamp(max_norm / (nrm + 1e-6), max=1.0) if max_norm > 0 else torch.ones_like(nrm))
        return
    N.check(_fn("clip_coef")(_at(sumsq), max_norm, _at(coef), _at(norm_out), _stream()), "clip_coef")


# --------------------------------------------------------------------------- attention


def ref_attention(q, k, v, causal=True):
    """q ``[B,S,Hq,Dh]``, k/v ``[B,S,Hkv,Dh]`` -> ``[B,S,Hq,Dh]`` (fp32 math)."""
    B, S, Hq, Dh = q.shape
    Hkv = k.shape[2]
    rep = Hq // Hkv
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    s = qf @ kf.transpose(-1, -2) / math.sqrt(Dh)
    if causal:
        mask = torch.ones(S, S, dtype=torch.bool, device=q.device).tril()
        s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return (p @ vf).permute(0, 2, 1, 3).to(q.dtype)


def ref_attention_lse(q, k, v, causal=True):
    """Row-wise ``logsumexp(scale * q k^T)`` ``[B,Hq,S]`` (fp32) of the same problem."""
    B, S, Hq, Dh = q.shape
    rep = Hq // k.shape[2]
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    s = qf @ kf.transpose(-1, -2) / math.sqrt(Dh)
    if causal:
        mask = torch.ones(S, S, dtype=torch.bool, device=q.device).tril()
        s = s.masked_fill(~mask, float("-inf"))
    return torch.logsumexp(s, dim=-1)


class AttentionSpans:
    """Which keys each query sees in rows of packed documents (:func:`attention_spans`): ``rows`` int32 ``[batch, seq, 4]`` holds the range
    ``[lo, hi)`` of the keys that a token sees and the range ``[from, to)`` of the queries that see it, both empty for padding;
    ``positions`` int32 ``[batch, seq]`` counts from 0 in every document (``positions.view(1, -1)`` goes into :func:`rope_axes_`).
    ``tiles`` and ``padded`` are what the kernels need of 128 and of 1024 tokens."""

    def __init__(self, batch: int, seq: int, device, buf: Optional[torch.Tensor] = None) -> None:
        self.batch, self.seq, self.n_tiles = batch, seq, (seq + 127) // 128
        a = 4 * batch * seq
        b = a + 8 * batch * self.n_tiles
        c = b + batch * seq
        self._at = (0, a, b, c, c + batch * ((seq + 1023) // 1024))
        self._buf = torch.zeros(self._at[4], dtype=torch.int32, device=device) if buf is None else buf  # zeros: nobody sees anything

    @property
    def device(self) -> torch.device:
        return self._buf.device

    def _part(self, i: int, *shape: int) -> torch.Tensor:
        return self._buf[self._at[i] : self._at[i + 1]].view(*shape)

    @property
    def rows(self) -> torch.Tensor:
        return self._part(0, self.batch, self.seq, 4)

    @property
    def tiles(self) -> torch.Tensor:
        return self._part(1, self.batch, self.n_tiles, 8)

    @property
    def positions(self) -> torch.Tensor:
        return self._part(2, self.batch, self.seq)

    @property
    def padded(self) -> torch.Tensor:
        return self._part(3, self.batch, (self.seq + 1023) // 1024)


_NONE = 2**31 - 1


def ref_attention_spans(documents, prefix=None, causal=True, window=0):
    """``(rows, positions, tiles, padded)`` of :func:`attention_spans`."""
    B, S = documents.shape
    at = torch.arange(S, device=documents.device).expand(B, S)
    first = torch.ones(B, S, dtype=torch.bool, device=documents.device)
    first[:, 1:] = documents[:, 1:] != documents[:, :-1]
    last = torch.ones_like(first)
    last[:, :-1] = first[:, 1:]
    start = torch.where(first, at, 0).cummax(1).values
    end = torch.where(last, at + 1, S).flip(1).cummin(1).values.flip(1)
    lo, hi, since, to = start, end, start, end
    if causal:
        plain = torch.where(prefix == 0, at, S) if prefix is not None else at
        pre = torch.minimum(plain.flip(1).cummin(1).values.flip(1).gather(1, start), end)  # where a document's prefix ends
        hi = torch.maximum(at + 1, pre)
        since = torch.where(at < pre, start, at)
        if window > 0:
            lo = torch.maximum(start, at - (window - 1))
            to = torch.minimum(end, at + window)
    rows = torch.stack([lo, hi, since, to], -1)
    live = (documents >= 0).unsqueeze(-1)
    rows = torch.where(live, rows, 0)
    n = (S + 127) // 128
    fill = torch.zeros(B, n * 128 - S, 4, dtype=rows.dtype, device=rows.device)
    r = torch.cat([rows, fill], 1).view(B, n, 128, 4)
    dead, beyond = r[..., 1] <= r[..., 0], torch.arange(n * 128, device=rows.device).view(n, 128) >= S
    least = torch.where(dead, _NONE, r[..., 0]).amin(-1), torch.where(dead, _NONE, r[..., 2]).amin(-1)
    most = r[..., 1].amax(-1), r[..., 3].amax(-1)
    hole = (dead & ~beyond).any(-1)
    odd = dead.any(-1)
    every = (torch.where(hole, _NONE, torch.where(dead, 0, r[..., 0]).amax(-1)), torch.where(hole, 0, torch.where(dead, _NONE, r[..., 1]).amin(-1)),
             torch.where(odd, _NONE, r[..., 2].amax(-1)), torch.where(odd, 0, torch.where(dead, _NONE, r[..., 3]).amin(-1)))
    tiles = torch.stack([least[0], most[0], every[0], every[1], least[1], most[1], every[2], every[3]], -1)
    return rows.to(torch.int32), (at - start).to(torch.int32), tiles.to(torch.int32), torch.stack(
        [(documents[:, i : i + 1024] < 0).any(1) for i in range(0, S, 1024)], 1).to(torch.int32)


def attention_spans(documents: torch.Tensor, prefix: Optional[torch.Tensor] = None, causal: bool = True, window: int = 0) -> AttentionSpans:
    """The mask of rows that hold documents one after another, for :func:`attention_fwd` and :func:`attention_bwd` (one for all layers and
    both passes of a batch).  ``documents`` int32 ``[batch, seq]``: a run of equal ids is a document, whose tokens see each other only;
    an id below zero is padding, which sees nothing (its output rows are zero) and is seen by nobody, whatever stands in it.  With
    ``causal`` a token sees itself and those before it, at most the last ``window`` of them (itself among them) where that is not 0, and
    the tokens that ``prefix`` (bool or uint8 ``[batch, seq]``) flags at the start of a document are seen by all of it, by each other in
    both directions too."""
    if documents.is_cuda:
        buf = N.host().attention_spans(documents, prefix, causal, window)
        N.launch_count += documents.numel() > 0
        return AttentionSpans(*documents.shape, None, buf)
    if documents.dim() != 2 or documents.dtype != torch.int32 or not documents.is_contiguous():
        raise ValueError("documents must be contiguous int32 [batch, seq]")
    if prefix is not None:
        if prefix.dtype not in (torch.bool, torch.uint8):
            raise ValueError("prefix must be bool or uint8")
        _check_like("prefix", prefix.dtype, documents.shape, documents.get_device(), prefix)
    if not 0 <= window < 2**31:
        raise ValueError("window must be 0 or a number of keys")
    if not causal and (window or prefix is not None):
        raise ValueError("a window or a prefix goes with a causal mask")
    B, S = documents.shape
    spans = AttentionSpans(B, S, documents.device)
    if B > 0 and S > 0:
        for mine, t in zip((spans.rows, spans.positions, spans.tiles, spans.padded), ref_attention_spans(documents, prefix, causal, window)):
            mine.copy_(t)
    return spans


def ref_attention_masked(q, k, v, rows=None, causal=True, softcap=0.0, slopes=None):
    """``(out, lse)`` of attention under a mask, in the type of the arguments: 4-D q, k, v as :func:`ref_attention`, ``rows`` as in
    :class:`AttentionSpans`.  What stands in padding reaches neither the others nor, as a gradient, padding."""
    B, S, Hq, Dh = q.shape
    rep = Hq // k.shape[2]
    if rows is not None:
        live = (rows[..., 1] > rows[..., 0])[..., None, None]
        q, k, v = (torch.where(live, t, 0.0) for t in (q, k, v))
    q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(rep, 1), v.transpose(1, 2).repeat_interleave(rep, 1)
    s = q @ k.transpose(-1, -2) / math.sqrt(Dh)
    if softcap > 0:
        s = softcap * torch.tanh(s / softcap)
    at = torch.arange(S, device=q.device)
    if slopes is not None:
        s = s - slopes.to(s.dtype)[:, None, None] * (at[:, None] - at[None, :]).abs()
    if rows is not None:
        seen = ((at >= rows[..., 0:1]) & (at < rows[..., 1:2])).unsqueeze(1)
    else:
        seen = (at[:, None] >= at[None, :]) | (not causal)
    s = s.masked_fill(~seen, -math.inf)
    top = s.detach().amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    o = ((p @ v) / torch.where(total > 0, total, 1.0)).transpose(1, 2)
    if rows is not None:
        o = torch.where(live, o, 0.0)  # with it the gradient that comes back
    return o, (top + total.log()).squeeze(-1).detach()


def _check_masked(of_q, of_kv, spans: Optional[AttentionSpans], softcap: float, slopes: Optional[torch.Tensor], lse: Optional[torch.Tensor],
                  batch: int, seq_len: int, n_heads: int, n_kv_heads: int, head_dim: int) -> None:
    if head_dim not in (64, 128) or n_heads < 1 or n_kv_heads < 1 or n_heads % n_kv_heads:
        raise ValueError("masked attention takes head dims 64 and 128 and groups of equally many query heads")
    at = of_q[0].get_device()
    for tensors, heads in ((of_q, n_heads), (of_kv, n_kv_heads)):
        shape = (batch * seq_len, heads * head_dim)
        for t in tensors:
            if t.shape != shape or t.dtype != torch.bfloat16 or t.stride(1) != 1 or t.get_device() != at or (shape[0] > 1 and t.stride(0) < shape[1]):
                raise ValueError(f"a tensor of {heads} heads must be bf16 {shape} with unit inner stride, its rows apart, on {of_q[0].device}, got "
                                 f"{t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}")
    if softcap != 0.0 and not 1e-9 <= softcap <= 1e30:
        raise ValueError("softcap must be 0 or a cap from 1e-9 to 1e30")
    if spans is not None and (spans.batch, spans.seq) != (batch, seq_len):
        raise ValueError(f"spans are of {(spans.batch, spans.seq)}, not of {(batch, seq_len)}")
    if spans is not None and spans.device != of_q[0].device:
        raise ValueError(f"spans are on {spans.device}")
    if slopes is not None:
        _check_like("slopes", torch.float32, (n_heads,), at, slopes)
    if lse is not None:
        _check_like("lse", torch.float32, (batch, n_heads, seq_len), at, lse)


def attention_supported(seq_len: int, head_dim: int) -> bool:
    """Shapes the tcgen05 attention kernels take: head dim 128 with 128-row blocks, or head dim 64 with
    sequences that are a multiple of 256 (the forward kernel for it works on two 128-query tiles per CTA)."""
    return (head_dim == 128 and seq_len % 128 == 0) or (head_dim == 64 and seq_len % 256 == 0)


@functools.lru_cache(maxsize=None)
def _sm_count(device_index: int) -> int:
    return torch.cuda.get_device_properties(device_index).multi_processor_count


def _two_query_tiles(batch: int, seq_len: int, n_heads: int, sms: int) -> bool:
    """Whether a CTA of the forward kernel takes two tiles of 128 queries at head dim 128: where the sequence divides into
    them and they fill the chip (475 us against 589 us at 1 x 8192, 32/8 heads, 148 SMs).  Up to one wave of 128-query
    CTAs the length of one CTA's chain counts, and that is shorter with one tile: 28.5 us against 40.7 us at 1 x 2048,
    8/8 heads; at twice a wave 28.6 against 22.9."""
    return seq_len % 256 == 0 and batch * n_heads * (seq_len // 128) > sms


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: int, seq_len: int, n_heads: int,
                  n_kv_heads: int, head_dim: int, out: torch.Tensor, lse: Optional[torch.Tensor] = None,
                  causal: bool = True, any_length: bool = False, spans: Optional[AttentionSpans] = None, softcap: float = 0.0,
                  slopes: Optional[torch.Tensor] = None) -> None:
    """Causal GQA attention forward.  ``q`` ``[batch*seq, n_heads*head_dim]`` and ``k``/``v``
    ``[batch*seq, n_kv_heads*head_dim]`` are 2-D bf16 views (column slices of the packed QKV
    activation are fine), ``out`` ``[batch*seq, n_heads*head_dim]``, ``lse`` ``[batch, n_heads,
    seq]`` fp32 (saved for the backward pass).  Sequence lengths are those of :func:`attention_supported`; ``any_length``
    takes every other one as well (of head dims 64 and 128).

    ``spans`` (:func:`attention_spans`) say which keys a query sees, in place of ``causal``. ``softcap`` caps the scaled scores: ``softcap *
    tanh(s / softcap)`` (a cap from 1e-9 to 1e30); ``slopes`` (fp32 ``[n_heads]``, not differentiated) lower them by ``slope * |query -
    key|``. With any of the three the sequence may have any length; a row that sees nothing gets zeros and a ``lse`` of -infinity. Keys and
    values that a row does not see, of another document or behind it, have to be finite where they share a block of 128 with some that it
    sees; padding need not."""
    if spans is not None or softcap != 0.0 or slopes is not None:
        if q.is_cuda:
            if spans is not None and (spans.batch != batch or spans.seq != seq_len):
                raise ValueError(f"spans are of {(spans.batch, spans.seq)}, not of {(batch, seq_len)}")
            N.launch_count += N.host().attention_masked_fwd(q, k, v, out, lse, None if spans is None else spans._buf, slopes, batch, seq_len,
                                                            n_heads, n_kv_heads, head_dim, softcap, causal, _status_ptr(q.device))
            return
        _check_masked((q, out), (k, v), spans, softcap, slopes, lse, batch, seq_len, n_heads, n_kv_heads, head_dim)
        if batch == 0 or seq_len == 0:
            return
        q4, k4, v4 = (t.reshape(batch, seq_len, -1, head_dim).float() for t in (q, k, v))
        o4, l4 = ref_attention_masked(q4, k4, v4, spans.rows if spans is not None else None, causal, softcap, slopes)
        out.copy_(o4.reshape(batch * seq_len, -1))
        if lse is not None:
            lse.copy_(l4)
        return
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (out, "out")):
        _check_2d_bf16(t, name)
    if not q.is_cuda:
        B, S = batch, seq_len
        q4, k4, v4 = (t.reshape(B, S, -1, head_dim) for t in (q, k, v))
        out.copy_(ref_attention(q4, k4, v4, causal).reshape(B * S, -1))
        if lse is not None:
            lse.copy_(ref_attention_lse(q4, k4, v4, causal))
        return
    scale = 1.0 / math.sqrt(head_dim)
    impl = os.environ.get("FTB200_ATTN_FWD", "auto")
    if seq_len % 256 and (head_dim != 128 or seq_len % 128 or impl == "pair"):
        if not any_length:
            N.check(-1, "attention_fwd")
        impl = "pair"  # the other kernel takes whole tiles only
    if impl == "auto":
        impl = "pair" if _two_query_tiles(batch, seq_len, n_heads, _sm_count(q.device.index)) else "single"
    if impl == "pair" or head_dim != 128:
        # two query tiles per CTA, one softmax thread per row (head dim 64 or 128, seq % 256 == 0).  At head dim 64 the
        # products are half as long and the exponential unit is the scarcer: a quarter of the exponentials goes to the
        # FMA pipe (8 x 2048, 32/8 heads: 303 us against 321); at head dim 128 none (475 us against 486).
        poly = int(os.environ.get("FTB200_ATTN_POLY") or ("2" if head_dim == 64 else "0"))
        N.check(
            _fn("attention_fwd2")(_at(q), _at(k), _at(v), _at(out), _at(lse), batch, seq_len, n_heads, n_kv_heads, head_dim,
                                  q.stride(0), k.stride(0), v.stride(0), out.stride(0), scale, int(causal), poly,
                                  _status_ptr(q.device), _stream()),
            "attention_fwd2",
        )
        return
    N.check(
        _fn("attention_fwd")(_at(q), _at(k), _at(v), _at(out), _at(lse), batch, seq_len, n_heads, n_kv_heads, head_dim,
                             q.stride(0), k.stride(0), v.stride(0), out.stride(0), scale, int(causal), _status_ptr(q.device),
                             _stream()),
        "attention_fwd",
    )


def ref_attention_bwd(q, k, v, d_o, causal=True):
    """(dq, dk, dv) of :func:`ref_attention` by autograd in fp32; 4-D inputs as there."""
    q, k, v = (t.detach().float().requires_grad_(True) for t in (q, k, v))
    o = ref_attention(q, k, v, causal)
    return torch.autograd.grad(o, (q, k, v), d_o.float())


_attn_scratch: dict = {}


def attention_bwd_scratch_bytes(batch: int, seq_len: int, n_heads: int, n_kv_heads: int) -> int:
    """Size of the ``scratch`` that :func:`attention_bwd` takes."""
    lib = N.lib()
    lib.ftb200_attention_bwd_scratch_bytes.restype = ctypes.c_longlong
    return int(lib.ftb200_attention_bwd_scratch_bytes(batch, seq_len, n_heads, n_kv_heads))


def attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, d_o: torch.Tensor,
                  lse: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, batch: int, seq_len: int,
                  n_heads: int, n_kv_heads: int, head_dim: int, causal: bool = True,
                  scratch: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None, any_length: bool = False,
                  spans: Optional[AttentionSpans] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None) -> None:
    """Backward of :func:`attention_fwd`: writes ``dq``, ``dk``, ``dv`` (2-D bf16 views like
    ``q``, ``k``, ``v``; column slices of a packed dQKV buffer are fine).  The fp32 dQ
    accumulator lives in ``scratch`` (bytes on the device, :func:`attention_bwd_scratch_bytes` of
    them or more), by default a per-device buffer that is reused across calls on the same stream.
    With ``rope``, the table (:func:`rope_table`) that ``q`` and ``k`` were rotated by, ``dq`` and ``dk``
    are the gradients of the values before the rotation.  Sequences are a multiple of 128 or, with
    ``any_length``, of any length.

    ``spans``, ``softcap`` and ``slopes`` as in the forward pass; with any of them sequences have any length, the default
    ``scratch`` is this call's own, and rows that see nothing, or are seen by nobody, get zeros.  Probabilities are made again from the
    fp32 ``lse`` and are off by about 2^-22 of the score's size, so that from scores of 10^5 on the gradients lose their meaning."""
    if spans is not None or softcap != 0.0 or slopes is not None:
        if q.is_cuda:
            if spans is not None and (spans.batch != batch or spans.seq != seq_len):
                raise ValueError(f"spans are of {(spans.batch, spans.seq)}, not of {(batch, seq_len)}")
            N.launch_count += N.host().attention_masked_bwd(
                q, k, v, o, d_o, lse, dq, dk, dv, scratch, rope, None if spans is None else spans._buf, slopes, batch, seq_len, n_heads, n_kv_heads,
                head_dim, softcap, causal, _status_ptr(q.device))
            return
        _check_masked((q, o, d_o, dq), (k, v, dk, dv), spans, softcap, slopes, lse, batch, seq_len, n_heads, n_kv_heads, head_dim)
        if rope is not None and (rope.dtype != torch.float32 or not rope.is_contiguous() or rope.get_device() != q.get_device() or rope.dim() != 3
                                 or rope.shape[0] < seq_len or rope.shape[1:] != (head_dim // 2, 2)):
            raise ValueError("rope must be the table of the sequence and head dim on the device of q")
        if batch == 0 or seq_len == 0:
            return
        q4, k4, v4 = (t.detach().reshape(batch, seq_len, -1, head_dim).float().requires_grad_(True) for t in (q, k, v))
        with torch.enable_grad():
            o4, _ = ref_attention_masked(q4, k4, v4, spans.rows if spans is not None else None, causal, softcap, slopes)
        for to, g in zip((dq, dk, dv), torch.autograd.grad(o4, (q4, k4, v4), d_o.reshape(batch, seq_len, -1, head_dim).float())):
            to.copy_(g.reshape(batch * seq_len, -1))
        if rope is not None:
            dq.copy_(ref_rope(dq, rope, seq_len, n_heads, head_dim, backward=True))
            dk.copy_(ref_rope(dk, rope, seq_len, n_kv_heads, head_dim, backward=True))
        return
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (o, "o"), (d_o, "d_o"), (dq, "dq"), (dk, "dk"), (dv, "dv")):
        _check_2d_bf16(t, name)
    if not q.is_cuda:
        B, S = batch, seq_len
        q4, k4, v4, do4 = (t.reshape(B, S, -1, head_dim) for t in (q, k, v, d_o))
        gq, gk, gv = ref_attention_bwd(q4, k4, v4, do4, causal)
        dq.copy_(gq.reshape(B * S, -1))
        dk.copy_(gk.reshape(B * S, -1))
        dv.copy_(gv.reshape(B * S, -1))
        if rope is not None:
            dq.copy_(ref_rope(dq, rope, S, n_heads, head_dim, backward=True))
            dk.copy_(ref_rope(dk, rope, S, n_kv_heads, head_dim, backward=True))
        return
    if seq_len % 128 and not any_length:
        N.check(-1, "attention_bwd")
    if rope is not None and (rope.dtype != torch.float32 or not rope.is_contiguous() or rope.device != q.device
                             or rope.shape[0] < seq_len or tuple(rope.shape[1:]) != (head_dim // 2, 2)):
        raise ValueError("rope must be the table of the sequence and head dim on the device of q")
    lib = N.lib()
    need = attention_bwd_scratch_bytes(batch, seq_len, n_heads, n_kv_heads)
    if scratch is None:
        key = (q.device.index, _stream())
        scratch = _attn_scratch.get(key)
        if scratch is None or scratch.numel() < need:
            scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
            _attn_scratch[key] = scratch
    elif scratch.device != q.device or scratch.dtype != torch.uint8 or scratch.numel() < need or not scratch.is_contiguous():
        raise ValueError(f"scratch must be {need} contiguous bytes on {q.device}")
    scale = 1.0 / math.sqrt(head_dim)
    N.check(
        _fn("attention_bwd")(_at(q), _at(k), _at(v), _at(o), _at(d_o), _at(lse), _at(dq), _at(dk), _at(dv), _at(scratch),
                             batch, seq_len, n_heads, n_kv_heads, head_dim, q.stride(0), k.stride(0), v.stride(0), o.stride(0),
                             d_o.stride(0), dq.stride(0), dk.stride(0), dv.stride(0), scale, int(causal), _at(rope),
                             _status_ptr(q.device), _stream()),
        "attention_bwd", launches=3,
    )
