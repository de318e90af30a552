"""Decode-path kernels with the entry points of the reference's ``app/kernels.py``.

Same names, argument order and tensor layouts as the reference, so an engine written
against it runs unchanged:

    int8_mm(x, w, s, res=None)                                   app/kernels.py:40-54
    rms(x, w, eps=1e-5)                                          app/kernels.py:70-74
    _rope_cache[grid](qkv, rope, pos, q, kc, vc, S, Hq, Hk, L, HD=, HALF=)    :78-107
    _attn[grid](q, kc, vc, pos, o, pm, pl, pa, S, Hq, Hk, L, scale,
                HD=, HDP=, G=, BLK=, NSPLIT=, num_warps=)                     :111-153
    _attn_combine[grid](pm, pl, pa, o, HD=, HDP=, NSPLIT=)                    :156-167
    _silu_mul[grid](x, y, F_, BLOCK=)                                         :171-180

Every call goes to a hand-written gfx950 HIP kernel through the C ABI of
``libecdecode.so``, on the current HIP stream, so it can be captured in a hipGraph.
The Triton tiling knobs (HALF, HDP, BLK, BLOCK, num_warps) are accepted for drop-in
compatibility and checked for consistency, but the HIP kernels choose their own tiling;
the grid must be the one the reference launches with.  Tensors must be fp16 (the
reference GPU default, app/engine.py:219-222) and live on a ROCm device.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from . import _ffi

__all__ = ["int8_mm", "rms", "_rope_cache", "_attn", "_attn_combine", "_silu_mul",
           "next_power_of_2", "cdiv", "stream_ptr"]


def next_power_of_2(n: int) -> int:
    """Host helper the reference engine takes from Triton (app/engine.py:192,194)."""
    n = int(n)
    return 1 if n <= 1 else 1 << (n - 1).bit_length()


def cdiv(a: int, b: int) -> int:
    return -(-int(a) // int(b))


def stream_ptr(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _dev(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError(f"{name}: the decode path runs only on a ROCm GPU tensor (got {t.device})")
    return t.device


def _f16(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.float16:
        raise TypeError(f"{name}: expected float16, got {t.dtype}")


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------- GEMV int8 (+ optional residual)
def int8_mm(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, res: torch.Tensor | None = None):
    """x [..., K] fp16, w [N, K] int8, s [N] fp16 -> [..., N] (+ res).

    M = prod(x.shape[:-1]) <= 16 uses the reference GEMV numerics (scale after the fp32
    dot product); M > 16 uses its dequantise-then-GEMM numerics (app/kernels.py:46-49)."""
    dev = _dev(x, "int8_mm")
    _f16(x, "int8_mm x")
    if w.dtype != torch.int8 or w.dim() != 2 or not w.is_contiguous():
        raise TypeError("int8_mm: w must be a contiguous [N, K] int8 tensor")
    if s.dtype != torch.float16 or s.numel() != w.shape[0] or not s.is_contiguous():
        raise TypeError("int8_mm: s must be a contiguous [N] float16 tensor")
    shp = x.shape
    K = shp[-1]
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"int8_mm: x has K={K}, w has K={w.shape[1]}")
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or x2.stride(0) < K:
        x2 = x2.contiguous()
    M = x2.shape[0]
    y = torch.empty(M, N, device=dev, dtype=torch.float16)
    r2 = None
    if res is not None:
        _f16(res, "int8_mm res")
        r2 = res.reshape(M, N)
        if r2.stride(-1) != 1 or r2.stride(0) < N:
            r2 = r2.contiguous()
    if M == 0:
        return y.reshape(*shp[:-1], N)
    _ffi.call("ecd_gemv_i8", x2.data_ptr(), x2.stride(0), w.data_ptr(), s.data_ptr(), _ptr(r2),
              r2.stride(0) if r2 is not None else 0, y.data_ptr(), N, M, N, K, int(M > 16),
              stream_ptr(dev))
    return y.reshape(*shp[:-1], N)


# ---------------------------------------------------------------- RMSNorm
def rms(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-5):
    """x [R, D] fp16, w [D] fp16 -> fp16(fp16(x * rsqrt(mean(x^2) + eps)) * w)."""
    dev = _dev(x, "rms")
    _f16(x, "rms x")
    _f16(w, "rms w")
    R, D = x.shape
    if w.numel() != D:
        raise ValueError("rms: weight size mismatch")
    if x.stride(-1) != 1:
        x = x.contiguous()
    y = torch.empty(R, D, device=dev, dtype=torch.float16)
    _ffi.call("ecd_rmsnorm", x.data_ptr(), x.stride(0), w.data_ptr(), y.data_ptr(), D, R, D,
              float(eps), stream_ptr(dev))
    return y


class _Launcher:
    """``kernel[grid](...)`` call syntax of the reference's Triton launchers."""

    def __init__(self, name, fn, grid_fn):
        self.__name__ = name
        self._fn = fn
        self._grid_fn = grid_fn

    def __getitem__(self, grid):
        grid = tuple(grid) if isinstance(grid, (tuple, list)) else (grid,)

        def launch(*args, **kwargs):
            want = self._grid_fn(*args, **kwargs)
            if tuple(grid) != tuple(want):
                raise ValueError(f"{self.__name__}: grid {grid} does not match the launch {want}")
            return self._fn(*args, **kwargs)

        return launch

    def __call__(self, *args, **kwargs):  # direct call without a grid
        return self._fn(*args, **kwargs)


# ---------------------------------------------------------------- RoPE + KV-cache write
def _rope_cache_impl(qkv, rope, pos, q, kc, vc, S, Hq, Hk, L, HD, HALF=None):
    dev = _dev(qkv, "_rope_cache")
    for t, n in ((qkv, "qkv"), (q, "q"), (kc, "kc"), (vc, "vc")):
        _f16(t, f"_rope_cache {n}")
        if not t.is_contiguous():
            raise ValueError(f"_rope_cache: {n} must be contiguous")
    if rope.dtype != torch.float32 or not rope.is_contiguous():
        raise TypeError("_rope_cache: rope table must be contiguous float32 [L, HD/2, 2]")
    if pos.dtype != torch.int64 or not pos.is_contiguous():
        raise TypeError("_rope_cache: pos must be contiguous int64")
    if HALF is not None and HALF < HD // 2:
        raise ValueError("_rope_cache: HALF must cover HD // 2")
    R = qkv.shape[0]
    if qkv.shape[1] != (Hq + 2 * Hk) * HD or q.numel() != R * Hq * HD or pos.numel() != R:
        raise ValueError("_rope_cache: shape mismatch")
    if kc.shape[-1] != HD or kc.shape[-2] != L or kc.shape[1] != Hk or kc.shape[0] * S < R:
        raise ValueError("_rope_cache: cache must be [B, Hk, L, HD] with B >= R / S")
    if rope.shape[0] < L or rope.shape[1] != HD // 2:
        raise ValueError("_rope_cache: rope table must have >= L rows of HD/2 pairs")
    _ffi.call("ecd_rope_kv_write", qkv.data_ptr(), rope.data_ptr(), pos.data_ptr(), q.data_ptr(),
              kc.data_ptr(), vc.data_ptr(), R, S, Hq, Hk, L, HD, stream_ptr(dev))


_rope_cache = _Launcher("_rope_cache", _rope_cache_impl,
                        lambda qkv, rope, pos, q, kc, vc, S, Hq, Hk, L, HD=None, HALF=None:
                        (qkv.shape[0], Hq + Hk))


# ---------------------------------------------------------------- decode attention
def _attn_impl(q, kc, vc, pos, o, pm, pl, pa, S, Hq, Hk, L, scale, HD, HDP=None, G=None,
               BLK=None, NSPLIT=16, num_warps=None):
    dev = _dev(q, "_attn")
    for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (o, "o")):
        _f16(t, f"_attn {n}")
        if not t.is_contiguous():
            raise ValueError(f"_attn: {n} must be contiguous")
    if pos.dtype != torch.int64 or not pos.is_contiguous():
        raise TypeError("_attn: pos must be contiguous int64")
    if G is not None and G != Hq // Hk:
        raise ValueError("_attn: G must equal Hq // Hk")
    R = q.shape[0]
    if q.numel() != R * Hq * HD or pos.numel() != R or o.numel() != R * Hq * HD:
        raise ValueError("_attn: shape mismatch")
    if kc.shape[-1] != HD or kc.shape[-2] != L or kc.shape[1] != Hk or kc.shape[0] * S < R:
        raise ValueError("_attn: cache must be [B, Hk, L, HD] with B >= R / S")
    if NSPLIT > 1:
        need = R * Hq * NSPLIT
        for t, n, k in ((pm, "pm", need), (pl, "pl", need), (pa, "pa", need * HD)):
            if t.dtype != torch.float32 or t.numel() < k or not t.is_contiguous():
                raise ValueError(f"_attn: {n} must be float32 with >= {k} elements")
        ptrs = (pm.data_ptr(), pl.data_ptr(), pa.data_ptr())
    else:
        ptrs = (None, None, None)
    _ffi.call("ecd_decode_attn", q.data_ptr(), kc.data_ptr(), vc.data_ptr(), pos.data_ptr(),
              o.data_ptr(), *ptrs, R, S, Hq, Hk, L, HD, int(NSPLIT), float(scale), stream_ptr(dev))


_attn = _Launcher("_attn", _attn_impl,
                  lambda q, kc, vc, pos, o, pm, pl, pa, S, Hq, Hk, L, scale, HD=None, HDP=None,
                  G=None, BLK=None, NSPLIT=16, num_warps=None: (q.shape[0], Hk, NSPLIT))


def _attn_combine_impl(pm, pl, pa, o, HD, HDP=None, NSPLIT=16):
    dev = _dev(o, "_attn_combine")
    _f16(o, "_attn_combine o")
    RH = o.numel() // HD
    for t, n, k in ((pm, "pm", RH * NSPLIT), (pl, "pl", RH * NSPLIT), (pa, "pa", RH * NSPLIT * HD)):
        if t.dtype != torch.float32 or t.numel() < k or not t.is_contiguous():
            raise ValueError(f"_attn_combine: {n} must be float32 with >= {k} elements")
    _ffi.call("ecd_attn_combine", pm.data_ptr(), pl.data_ptr(), pa.data_ptr(), o.data_ptr(), RH,
              HD, int(NSPLIT), stream_ptr(dev))


_attn_combine = _Launcher("_attn_combine", _attn_combine_impl,
                          lambda pm, pl, pa, o, HD=None, HDP=None, NSPLIT=16: (o.numel() // HD,))


def decode_attn_noalloc(q, kc, vc, pos, S, Hq, Hk, L, scale, nsplit=16, out=None):
    """_attn + _attn_combine in one call whose split partials live in the library's static
    device workspace (8 MiB per GPU): nothing is allocated when ``out`` is given, so it can run
    under hipGraph capture without a memory pool.  Raises MemoryError when R * Hq * nsplit
    partials do not fit.  Calls overlapping on one GPU share the workspace."""
    dev = _dev(q, "decode_attn_noalloc")
    for t, n in ((q, "q"), (kc, "kc"), (vc, "vc")):
        _f16(t, f"decode_attn_noalloc {n}")
        if not t.is_contiguous():
            raise ValueError(f"decode_attn_noalloc: {n} must be contiguous")
    if pos.dtype != torch.int64 or not pos.is_contiguous():
        raise TypeError("decode_attn_noalloc: pos must be contiguous int64")
    R = q.shape[0]
    HD = kc.shape[-1]
    if q.numel() != R * Hq * HD or pos.numel() != R or kc.shape[1] != Hk or kc.shape[-2] != L \
            or kc.shape[0] * S < R or vc.shape != kc.shape:
        raise ValueError("decode_attn_noalloc: shape mismatch")
    o = out if out is not None else torch.empty_like(q)
    if o.shape != q.shape or o.dtype != torch.float16 or not o.is_contiguous():
        raise ValueError("decode_attn_noalloc: out must be a contiguous fp16 tensor shaped like q")
    _ffi.call("ecd_decode_attn_noalloc", q.data_ptr(), kc.data_ptr(), vc.data_ptr(), pos.data_ptr(),
              o.data_ptr(), R, S, Hq, Hk, L, HD, int(nsplit), float(scale), stream_ptr(dev))
    return o


# ---------------------------------------------------------------- SiLU(a) * b
def _silu_mul_impl(x, y, F_, BLOCK=None):
    dev = _dev(x, "_silu_mul")
    _f16(x, "_silu_mul x")
    _f16(y, "_silu_mul y")
    if not (x.is_contiguous() and y.is_contiguous()):
        raise ValueError("_silu_mul: tensors must be contiguous")
    R = y.numel() // F_
    if x.numel() != 2 * R * F_:
        raise ValueError("_silu_mul: x must be [R, 2F] for y [R, F]")
    _ffi.call("ecd_silu_mul", x.data_ptr(), y.data_ptr(), R, F_, stream_ptr(dev))


_silu_mul = _Launcher("_silu_mul", _silu_mul_impl,
                      lambda x, y, F_, BLOCK=1024: (y.numel() // F_, cdiv(F_, BLOCK)))


# ---------------------------------------------------------------- fused sampler
def sample_topk(logits, N, cfg, temp, topk, out, seed=None, pos=None, salt=0, noise=None,
                rows=None, x=None, qkv=None, kc=None, vc=None, p=0, o=None, ev=None, xe=None):
    """CFG mix + temperature + top-k + softmax(log_softmax) + Exponential race in one kernel
    (the math of _sample/_guided, app/engine.py:291-305).

    logits [B, V] fp16 (B = 2N: cond rows then uncond rows; B = N: no CFG); out: int64 view
    with out[b] the token slot of row b (any row stride).  The Exponential(1) draws come from
    a counter-based Philox keyed by seed (int64 device scalar) at frame position pos (int64
    device scalar) and ``salt``, or from ``noise`` [N, V] float32 when given.

    With ``rows`` [>= V, D] fp16 and ``x`` [B, D] fp16, row b of x also receives rows[token of
    row b] (zeros where the race had no winner): the next decoder pass's input when rows[t]
    holds projection(embedding of token t) (app/engine.py:343).  With ``qkv`` [>= V,
    (Hq + 2 Hk) * HD] fp16 as well (the next pass's layer-0 q | k | v of each token at slot
    ``p``), k and v also go to slot p of the caches ``kc`` / ``vc`` [B, Hk, L, HD] and each
    row's decode attention over slots 0 .. p goes to ``o`` [B, Hq * HD] (HD = 128, or 384 with
    the arithmetic of the short-cache attention kernel).  With ``ev`` and ``xe`` ([>= B, D]
    each), rows of ev are copied to the same rows of xe as they are."""
    dev = _dev(logits, "sample_topk")
    _f16(logits, "sample_topk logits")
    B, V = logits.shape
    if logits.stride(-1) != 1:
        raise ValueError("sample_topk: logits rows must be contiguous")
    if out.dtype != torch.int64 or out.shape[0] != B:
        raise ValueError("sample_topk: out must be int64 with one slot per row")
    if noise is not None:
        if noise.dtype != torch.float32 or tuple(noise.shape) != (N, V) or not noise.is_contiguous():
            raise ValueError("sample_topk: noise must be contiguous float32 [N, V]")
    elif seed is None or pos is None:
        raise ValueError("sample_topk: seed and pos device scalars are required without noise")
    if (rows is None) != (x is None):
        raise ValueError("sample_topk: rows and x go together")
    if rows is None:
        _ffi.call("ecd_sample_topk", logits.data_ptr(), logits.stride(0), B, N, float(cfg),
                  float(temp), int(topk), V, _ptr(noise), _ptr(seed), _ptr(pos), int(salt),
                  out.data_ptr(), out.stride(0), stream_ptr(dev))
        return
    _f16(rows, "sample_topk rows")
    _f16(x, "sample_topk x")
    D = x.shape[1]
    if rows.dim() != 2 or rows.shape[0] < V or rows.shape[1] != D or rows.stride(1) != 1 or \
            x.dim() != 2 or x.shape[0] < B or x.stride(1) != 1:
        raise ValueError("sample_topk: rows must be [>= V, D] and x [>= B, D] with contiguous rows")
    Hq = Hk = L = HD = 0
    if qkv is not None:
        _f16(qkv, "sample_topk qkv")
        _f16(o, "sample_topk o")
        _f16(kc, "sample_topk kc")
        _f16(vc, "sample_topk vc")
        if kc.dim() != 4:
            raise ValueError("sample_topk: caches must be [>= B, Hk, L, HD]")
        Hk, L, HD = kc.shape[1], kc.shape[2], kc.shape[3]
        Hq = o.shape[1] // HD
        if HD not in (128, 384) or kc.shape[0] < B or vc.shape != kc.shape or \
                not kc.is_contiguous() or not vc.is_contiguous() or o.shape[0] < B or \
                o.stride(1) != 1 or qkv.dim() != 2 or qkv.shape[1] != (Hq + 2 * Hk) * HD or \
                qkv.stride(1) != 1:
            raise ValueError("sample_topk: qkv [>= V, (Hq + 2 Hk) HD], caches [>= B, Hk, L, HD], "
                             "o [>= B, Hq HD], HD 128 or 384")
    if (ev is None) != (xe is None):
        raise ValueError("sample_topk: ev and xe go together")
    if ev is not None:
        _f16(ev, "sample_topk ev")
        _f16(xe, "sample_topk xe")
        if ev.shape[0] < B or xe.shape[0] < B or ev.shape[1] != D or xe.shape[1] != D or \
                ev.stride(1) != 1 or xe.stride(1) != 1:
            raise ValueError("sample_topk: ev and xe must be [>= B, D] with contiguous rows")
    _ffi.call("ecd_sample_topk_next", logits.data_ptr(), logits.stride(0), B, N, float(cfg),
              float(temp), int(topk), V, _ptr(noise), _ptr(seed), _ptr(pos), int(salt),
              out.data_ptr(), out.stride(0), rows.data_ptr(), rows.stride(0), rows.shape[0],
              x.data_ptr(), x.stride(0), D, _ptr(qkv), 0 if qkv is None else qkv.stride(0),
              0 if qkv is None else qkv.shape[0], _ptr(kc), _ptr(vc), L, int(p), _ptr(o),
              0 if o is None else o.stride(0), Hq, Hk, HD, _ptr(ev),
              0 if ev is None else ev.stride(0),
              _ptr(xe), 0 if xe is None else xe.stride(0), stream_ptr(dev))


# ---------------------------------------------------------------- packed weights + fused GEMVs
def pack_i8(w: torch.Tensor, interleave: bool = False) -> torch.Tensor:
    """Lane-ordered 16 x 64 tile layout of an int8 [N, K] matrix (K % 64 == 0) for the fused
    GEMVs.  With ``interleave`` the two halves of w are row-interleaved (w1 | w3 -> pairs)."""
    dev = _dev(w, "pack_i8")
    if w.dtype != torch.int8 or w.dim() != 2 or not w.is_contiguous():
        raise TypeError("pack_i8: w must be a contiguous [N, K] int8 tensor")
    N, K = w.shape
    if K % 64 or (interleave and N % 2):
        raise ValueError("pack_i8: K must be a multiple of 64 (and N even to interleave)")
    out = torch.empty(-(-N // 16) * 16 * K, dtype=torch.int8, device=dev)
    _ffi.call("ecd_pack_i8", w.data_ptr(), N, K, int(interleave), out.data_ptr(), stream_ptr(dev))
    return out


def _check_x(x, K, name):
    _dev(x, name)
    _f16(x, name + " x")
    if x.dim() != 2 or x.shape[1] != K or x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        raise ValueError(f"{name}: x must be [M, {K}] fp16 with unit inner stride, 16-byte rows")


def _flags(M, stream):
    return int(M > 16) | (2 if stream else 0)


def gemv_packed(x, wp, s, N, K, res=None, out=None, stream=False):
    """y = int8_mm(x, w, s, res) on packed weights (same numerics).  ``stream``: the weights are
    read once per frame (nontemporal loads)."""
    _check_x(x, K, "gemv_packed")
    M = x.shape[0]
    y = out if out is not None else torch.empty(M, N, device=x.device, dtype=torch.float16)
    if res is not None:
        _f16(res, "gemv_packed res")
        if res.shape != (M, N) or res.stride(1) != 1:
            raise ValueError("gemv_packed: res must be [M, N] with unit inner stride")
    _ffi.call("ecd_gemv_i8p", x.data_ptr(), x.stride(0), wp.data_ptr(), s.data_ptr(), _ptr(res),
              res.stride(0) if res is not None else 0, y.data_ptr(), y.stride(0), M, N, K,
              _flags(M, stream), 0, 0, stream_ptr(x.device))
    return y


def gemv_packed_splitk(x, wp, s, N, K, ks, res=None, stream=False):
    """gemv_packed with K split over ``ks`` workgroups per tile (fp32 partial sums added in a
    fixed order by a second kernel): for few output tiles over a long K, where one workgroup
    per tile leaves most CUs idle.  Same numerics up to the fp32 summation order."""
    _check_x(x, K, "gemv_packed_splitk")
    M = x.shape[0]
    y = torch.empty(M, N, device=x.device, dtype=torch.float16)
    ws = torch.empty(ks * M * N, device=x.device, dtype=torch.float32)
    if res is not None:
        _f16(res, "gemv_packed_splitk res")
        if res.shape != (M, N) or res.stride(1) != 1:
            raise ValueError("gemv_packed_splitk: res must be [M, N] with unit inner stride")
    _ffi.call("ecd_gemv_i8p_splitk", x.data_ptr(), x.stride(0), wp.data_ptr(), s.data_ptr(),
              _ptr(res), res.stride(0) if res is not None else 0, y.data_ptr(), y.stride(0), M, N,
              K, int(ks), ws.data_ptr(), _flags(M, stream), stream_ptr(x.device))
    return y


def gemm_packed(x, wp, s, N, K, res=None):
    """int8_mm(x, w, s, res) for many rows (the dense numerics, y = fp16(x @ fp16(q * s)^T))
    on packed weights, tiled on MFMA; ``res`` is added in fp16."""
    _check_x(x, K, "gemm_packed")
    M = x.shape[0]
    y = torch.empty(M, N, device=x.device, dtype=torch.float16)
    if res is not None:
        _f16(res, "gemm_packed res")
        if res.shape != (M, N) or res.stride(1) != 1:
            raise ValueError("gemm_packed: res must be [M, N] with unit inner stride")
    _ffi.call("ecd_gemm_i8p", x.data_ptr(), x.stride(0), wp.data_ptr(), s.data_ptr(), _ptr(res),
              res.stride(0) if res is not None else 0, y.data_ptr(), y.stride(0), M, N, K,
              stream_ptr(x.device))
    return y


def gemm_rms_packed(x, wp, s, N, K, res, nw, eps=1e-5):
    """(h, rms(h, nw)) with h = gemm_packed(x, wp, s, N, K, res): a residual branch and the next layer's
    norm.  With few rows the product is split over K and one kernel adds the fp32 partial sums and the
    residual and forms the norm; the rounding points are the same.  The number of ways, and with it the
    grouping of the fp32 sums, depends on M: a row's low bits may differ between calls of few and of many rows."""
    M = x.shape[0]
    ks = _ffi.lib().ecd_gemm_i8p_splits(M, N, K) if N <= 4096 and res.is_contiguous() and \
        res.data_ptr() % 16 == 0 and nw.data_ptr() % 16 == 0 else 1
    if ks == 1:
        h = gemm_packed(x, wp, s, N, K, res)
        return h, rms(h, nw, eps)
    _check_x(x, K, "gemm_rms_packed")
    _f16(res, "gemm_rms_packed res")
    _f16(nw, "gemm_rms_packed nw")
    if res.shape != (M, N) or nw.numel() != N or not nw.is_contiguous():
        raise ValueError("gemm_rms_packed: res must be [M, N] and nw [N]")
    ws = torch.empty(ks * M * N, device=x.device, dtype=torch.float32)
    h = torch.empty(M, N, device=x.device, dtype=torch.float16)
    y = torch.empty_like(h)
    st = stream_ptr(x.device)
    _ffi.call("ecd_gemm_i8p_partial", x.data_ptr(), x.stride(0), wp.data_ptr(), s.data_ptr(), ws.data_ptr(), M, N,
              K, ks, st)
    _ffi.call("ecd_rms_sum", ws.data_ptr(), ks, res.data_ptr(), nw.data_ptr(), h.data_ptr(), y.data_ptr(), M, N,
              float(eps), st)
    return h, y


def gemm_silu_packed(x, wp, s, F, K):
    """_silu_mul(int8_mm(x, w1|w3, s)) for many rows on row-interleaved packed w1|w3
    (pack_i8(..., interleave=True)) -> [M, F]."""
    _check_x(x, K, "gemm_silu_packed")
    M = x.shape[0]
    mm = torch.empty(M, F, device=x.device, dtype=torch.float16)
    _ffi.call("ecd_gemm_i8p_silu", x.data_ptr(), x.stride(0), wp.data_ptr(), s.data_ptr(),
              mm.data_ptr(), mm.stride(0), M, F, K, stream_ptr(x.device))
    return mm


def gemm_rope_packed(x, wp, s, rope, pos, q, kc, vc, S, Hq, Hk, L, HD, K):
    """int8_mm(x, wq|wk|wv, s) followed by _rope_cache (app/kernels.py:78-107) in one launch:
    the q | k | v GEMM of many rows with RoPE and the cache write in its epilogue.  pos [M] int64
    (row m -> batch item m // S); writes q [M, Hq * HD] and the cache slots of kc / vc."""
    _check_x(x, K, "gemm_rope_packed")
    M = x.shape[0]
    for t, nm in ((q, "q"), (kc, "kc"), (vc, "vc")):
        _f16(t, f"gemm_rope_packed {nm}")
        if not t.is_contiguous():
            raise ValueError(f"gemm_rope_packed: {nm} must be contiguous")
    if q.shape != (M, Hq * HD):
        raise ValueError("gemm_rope_packed: q must be [M, Hq * HD]")
    if pos.dtype != torch.int64 or pos.numel() != M or not pos.is_contiguous():
        raise ValueError("gemm_rope_packed: pos must be a contiguous int64 vector of M rows")
    if rope.dtype != torch.float32 or not rope.is_contiguous() or rope.numel() < L * HD:
        raise ValueError("gemm_rope_packed: rope must be a contiguous fp32 [L, HD] table")
    if kc.shape[1:] != (Hk, L, HD) or vc.shape != kc.shape or kc.shape[0] * S < M:
        raise ValueError("gemm_rope_packed: kc / vc must be [B, Hk, L, HD] with B * S >= M")
    _ffi.call("ecd_gemm_i8p_rope", x.data_ptr(), x.stride(0), wp.data_ptr(), s.data_ptr(),
              rope.data_ptr(), pos.data_ptr(), q.data_ptr(), kc.data_ptr(), vc.data_ptr(), M, S,
              Hq, Hk, L, HD, K, stream_ptr(x.device))
    return q


def pack_f16(w: torch.Tensor, interleave: bool = False) -> torch.Tensor:
    """Lane-ordered 16 x 64 tile layout (2 KB tiles) of an fp16 [N, K] matrix (K % 64 == 0) for
    the fp16-weight GEMM; ``interleave`` row-interleaves the two halves (gate | up -> pairs)."""
    dev = _dev(w, "pack_f16")
    if w.dtype != torch.float16 or w.dim() != 2 or not w.is_contiguous():
        raise ValueError("pack_f16: w must be a contiguous fp16 [N, K] matrix")
    N, K = w.shape
    out = torch.empty(_ffi.lib().ecd_packed_bytes_f16(N, K) // 2, device=dev, dtype=torch.float16)
    _ffi.call("ecd_pack_f16", w.data_ptr(), N, K, int(interleave), out.data_ptr(), stream_ptr(dev))
    return out


def gemm_f16_packed(x, wp, N, K, bias=None, alpha=1.0, res=None, out=None):
    """F.linear(x, w, bias) on packed fp16 weights (fp32 accumulation and bias, one fp16 rounding),
    optionally scaled by ``alpha`` (rounded again) and plus ``res`` (fp16 add) -> [M, N]."""
    _check_x(x, K, "gemm_f16_packed")
    M = x.shape[0]
    y = out if out is not None else torch.empty(M, N, device=x.device, dtype=torch.float16)
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != N):
        raise ValueError("gemm_f16_packed: bias must be fp32 [N]")
    _ffi.call("ecd_gemm_f16p", x.data_ptr(), x.stride(0), wp.data_ptr(),
              bias.data_ptr() if bias is not None else None, float(alpha),
              res.data_ptr() if res is not None else None, res.stride(0) if res is not None else 0,
              y.data_ptr(), y.stride(0), M, N, K, stream_ptr(x.device))
    return y


def gemm_f16_silu_packed(x, wp, F, K, out=None):
    """silu(x @ gate^T) * (x @ up^T) on interleaved packed fp16 gate | up -> [M, F]."""
    _check_x(x, K, "gemm_f16_silu_packed")
    M = x.shape[0]
    mm = out if out is not None else torch.empty(M, F, device=x.device, dtype=torch.float16)
    if mm.shape != (M, F) or mm.dtype != torch.float16 or mm.stride(1) != 1:
        raise ValueError("gemm_f16_silu_packed: out must be fp16 [M, F] with unit inner stride")
    _ffi.call("ecd_gemm_f16p_silu", x.data_ptr(), x.stride(0), wp.data_ptr(), mm.data_ptr(),
              mm.stride(0), M, F, K, stream_ptr(x.device))
    return mm


def prefill_attn(q, kc, vc, pos, S, Hq, Hk, scale=None, out=None):
    """Causal prompt-pass attention on MFMA: q [B*S, Hq*HD] fp16, kc/vc [B, Hk, L, HD] holding
    the prompt's K/V, pos [B*S] int64 -> o [B*S, Hq*HD] (row r attends slots [0, pos[r]])."""
    R = q.shape[0]
    B, _, L, HD = kc.shape
    if q.dtype != torch.float16 or not q.is_contiguous() or q.shape[1] != Hq * HD or R != B * S:
        raise ValueError("prefill_attn: q must be contiguous fp16 [B*S, Hq*HD]")
    if not (kc.is_contiguous() and vc.is_contiguous()) or pos.dtype != torch.int64:
        raise ValueError("prefill_attn: contiguous caches and int64 positions required")
    o = out if out is not None else torch.empty_like(q)
    if o.shape != q.shape or o.dtype != torch.float16 or not o.is_contiguous():
        raise ValueError("prefill_attn: out must be a contiguous fp16 tensor shaped like q")
    pc = pos.contiguous()
    _ffi.call("ecd_prefill_attn", q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
              pc.data_ptr(), o.data_ptr(), B, S, Hq, Hk, L, HD,
              float(scale if scale is not None else 1.0 / math.sqrt(HD)), stream_ptr(q.device))
    return o


def rms_gemv_packed(x, nw, wp, s, N, K, eps=1e-5, stream=False, out=None):
    """int8_mm(rms(x, nw), w, s) in one kernel.  ``out``: optional [M, N] fp16 destination with
    unit inner stride (any row stride)."""
    _check_x(x, K, "rms_gemv_packed")
    M = x.shape[0]
    y = out if out is not None else torch.empty(M, N, device=x.device, dtype=torch.float16)
    if y.shape != (M, N) or y.dtype != torch.float16 or y.stride(1) != 1:
        raise ValueError("rms_gemv_packed: out must be fp16 [M, N] with unit inner stride")
    _ffi.call("ecd_rms_gemv_i8p", x.data_ptr(), x.stride(0), nw.data_ptr(), float(eps), wp.data_ptr(),
              s.data_ptr(), y.data_ptr(), y.stride(0), M, N, K, _flags(M, stream), stream_ptr(x.device))
    return y


def rms_qkv_rope(x, nw, wp, s, rope, pos, q, kc, vc, S, Hq, Hk, L, HD, eps=1e-5, stream=False):
    """rms -> fused q|k|v GEMV -> RoPE of q and k -> q out, k/v into the cache at pos (one kernel)."""
    K = x.shape[1]
    _check_x(x, K, "rms_qkv_rope")
    M = x.shape[0]
    if pos.dtype != torch.int64 or pos.numel() != M or not pos.is_contiguous():
        raise ValueError("rms_qkv_rope: pos must be contiguous int64 [M]")
    if kc.shape != (kc.shape[0], Hk, L, HD) or kc.shape[0] * S < M or vc.shape != kc.shape:
        raise ValueError("rms_qkv_rope: caches must be [B, Hk, L, HD] with B * S >= M")
    if rope.shape[0] < L or rope.shape[1] != HD // 2 or rope.dtype != torch.float32:
        raise ValueError("rms_qkv_rope: rope table must be float32 [>= L, HD/2, 2]")
    if q.numel() != M * Hq * HD or not (q.is_contiguous() and kc.is_contiguous() and vc.is_contiguous()):
        raise ValueError("rms_qkv_rope: q/kc/vc must be contiguous")
    _ffi.call("ecd_rms_qkv_rope", x.data_ptr(), x.stride(0), nw.data_ptr(), float(eps), wp.data_ptr(),
              s.data_ptr(), rope.data_ptr(), pos.data_ptr(), q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
              M, S, Hq, Hk, L, HD, K, _flags(M, stream), stream_ptr(x.device))


def rms_qkv_rope_rows(x, nw, wp, s, rope, pos, out, Hq, Hk, HD, eps=1e-5, dense=False):
    """rms -> fused q|k|v GEMV -> RoPE of q and k at pos[m] -> out[m] = q | k | v of row m
    ([M, (Hq + 2Hk) HD], row stride N, no cache write), one kernel for any M.  ``dense=False``
    keeps the numerics of a decode step of at most 16 rows (per-row scale after the int8 sum)
    whatever M is."""
    K = x.shape[1]
    _check_x(x, K, "rms_qkv_rope_rows")
    M = x.shape[0]
    N = (Hq + 2 * Hk) * HD
    if pos.dtype != torch.int64 or pos.numel() != M or not pos.is_contiguous():
        raise ValueError("rms_qkv_rope_rows: pos must be contiguous int64 [M]")
    if rope.dim() != 3 or rope.shape[1] != HD // 2 or rope.dtype != torch.float32:
        raise ValueError("rms_qkv_rope_rows: rope table must be float32 [L, HD/2, 2]")
    _f16(out, "rms_qkv_rope_rows out")
    if out.shape != (M, N) or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"rms_qkv_rope_rows: out must be contiguous [{M}, {N}]")
    L = rope.shape[0]
    _ffi.call("ecd_rms_qkv_rope", x.data_ptr(), x.stride(0), nw.data_ptr(), float(eps), wp.data_ptr(),
              s.data_ptr(), rope.data_ptr(), pos.data_ptr(), out.data_ptr(), None, None,
              M, 1, Hq, Hk, L, HD, K, int(bool(dense)) | 4, stream_ptr(x.device))
    return out


def rms_w13_silu(x, nw, wp, s_il, F, eps=1e-5, stream=False):
    """rms -> [w1 | w3] GEMV on row-interleaved packed weights -> fp16(silu(a)) * b, [M, F]."""
    K = x.shape[1]
    _check_x(x, K, "rms_w13_silu")
    M = x.shape[0]
    mm = torch.empty(M, F, device=x.device, dtype=torch.float16)
    _ffi.call("ecd_rms_w13_silu", x.data_ptr(), x.stride(0), nw.data_ptr(), float(eps), wp.data_ptr(),
              s_il.data_ptr(), mm.data_ptr(), M, F, K, _flags(M, stream), stream_ptr(x.device))
    return mm


def layer_tail_supported(M, D, F, Hq, Hk, HD, L=1, attention=False):
    """True when ``layer_tail`` runs these shapes on the current device (with ``attention``: the
    next layer's attention over an L-slot cache inside the same launch)."""
    return _ffi.lib().ecd_layer_tail_supported(int(M), int(D), int(F), int(Hq), int(Hk), int(HD),
                                               int(L), int(bool(attention))) == _ffi.ECD_OK


def layer_tail_ws_bytes(D, Hq, Hk, HD):
    """Bytes of the layer-tail workspace for these shapes on the current device."""
    return int(_ffi.lib().ecd_layer_tail_ws_bytes(int(D), int(Hq), int(Hk), int(HD)))


def layer_tail(o, xin, wo, so, n2, w13, s13, w2, s2, x1, mm, xout, sync, err, ws, nxt=None,
               o_next=None, eps=1e-5, stream=False, no_wait=False, kv_nt=False):
    """One launch for the tail of a decode layer (app/engine.py:206-210: O projection +
    residual, rms -> w1|w3 -> SiLU * mul, w2 + residual) and, with ``nxt``, the next layer's
    rms -> q|k|v -> RoPE -> q, cache slot (:189-192) and, with ``o_next`` [M, Hq * HD], that
    layer's decode attention (:194-204) into o_next.  Writes x1 [M, D], mm [M, F] and the layer
    output xout [M, D] (which must not alias xin, o, x1 or mm).  ``nxt``: dict with n1, wq
    (packed), sq, rope, pos, q, kc, vc, S, Hq, Hk, L, HD.  ``sync`` (int32 [>= 4096], zero before
    first use) and ``err`` (int32 [1]) persist between calls; ``ws``: float32 workspace of
    layer_tail_ws_bytes bytes, zero before first use and kept with its ``sync`` (partials are
    recognised by the sync region's gate count).  ``no_wait``: every wait gives up at once (tests
    of the error path: err becomes 1 and sync, ws and err must be zeroed before the next call).
    ``kv_nt``: the attention reads every cache slot with nontemporal loads (else only splits of
    more than 32 slots), for callers whose other data should stay in the Infinity Cache."""
    dev = _dev(o, "layer_tail")
    M, D = o.shape
    F = mm.shape[1]
    for t, n in ((o, "o"), (xin, "xin"), (x1, "x1"), (mm, "mm"), (xout, "xout")):
        _f16(t, f"layer_tail {n}")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"layer_tail: {n} must be contiguous and 16-byte aligned")
    if xin.shape != (M, D) or x1.shape != (M, D) or xout.shape != (M, D) or mm.shape[0] != M:
        raise ValueError("layer_tail: o, xin, x1, xout must be [M, D] and mm [M, F]")
    lo, hi = xout.data_ptr(), xout.data_ptr() + xout.numel() * 2
    for t in (o, xin, x1, mm):
        if t.data_ptr() < hi and lo < t.data_ptr() + t.numel() * 2:
            raise ValueError("layer_tail: xout must not alias o, xin, x1 or mm")
    if sync.dtype != torch.int32 or sync.numel() < 4096 or sync.data_ptr() % 256:
        raise ValueError("layer_tail: sync must be int32 [>= 4096], 256-byte aligned")
    if err.dtype != torch.int32 or err.numel() < 1:
        raise ValueError("layer_tail: err must be int32 [1]")
    if ws.dtype != torch.float32 or ws.data_ptr() % 16:
        raise ValueError("layer_tail: ws must be float32, 16-byte aligned")
    if nxt is None:
        nargs = [None] * 8
        S = Hq = Hk = L = HD = 1
    else:
        n = nxt
        pos, kc = n["pos"], n["kc"]
        S, Hq, Hk, L, HD = n["S"], n["Hq"], n["Hk"], n["L"], n["HD"]
        if pos.dtype != torch.int64 or pos.numel() != M or not pos.is_contiguous():
            raise ValueError("layer_tail: pos must be contiguous int64 [M]")
        if kc.shape != (kc.shape[0], Hk, L, HD) or kc.shape[0] * S < M or n["vc"].shape != kc.shape:
            raise ValueError("layer_tail: caches must be [B, Hk, L, HD] with B * S >= M")
        if n["q"].numel() != M * Hq * HD or not n["q"].is_contiguous():
            raise ValueError("layer_tail: q must be contiguous [M, Hq * HD]")
        if n["rope"].shape[0] < L or n["rope"].shape[1] != HD // 2:
            raise ValueError("layer_tail: rope table must be float32 [>= L, HD/2, 2]")
        nargs = [n["n1"].data_ptr(), n["wq"].data_ptr(), n["sq"].data_ptr(), n["rope"].data_ptr(),
                 pos.data_ptr(), n["q"].data_ptr(), kc.data_ptr(), n["vc"].data_ptr()]
    if ws.numel() * 4 < layer_tail_ws_bytes(D, Hq, Hk, HD):
        raise ValueError("layer_tail: ws is smaller than layer_tail_ws_bytes")
    if o_next is not None:
        if nxt is None:
            raise ValueError("layer_tail: o_next needs the next layer (nxt)")
        _f16(o_next, "layer_tail o_next")
        if o_next.numel() != M * Hq * HD or not o_next.is_contiguous() or o_next.data_ptr() % 16:
            raise ValueError("layer_tail: o_next must be contiguous [M, Hq * HD]")
    _ffi.call("ecd_layer_tail", o.data_ptr(), xin.data_ptr(), wo.data_ptr(), so.data_ptr(),
              n2.data_ptr(), w13.data_ptr(), s13.data_ptr(), w2.data_ptr(), s2.data_ptr(), *nargs,
              _ptr(o_next), x1.data_ptr(), mm.data_ptr(), xout.data_ptr(), sync.data_ptr(),
              err.data_ptr(),
              ws.data_ptr(), M, D, F, S, Hq, Hk, L, HD, float(eps),
              _flags(M, stream) | (4 if no_wait else 0) | (8 if kv_nt else 0), stream_ptr(dev))
    return xout


# order of a layer record of ecd_layer_stack (ecd_layer_rec)
STACK_FIELDS = ("wo", "so", "n2", "w13", "s13", "w2", "s2", "n1", "wq", "sq", "kc", "vc", "x1",
                "mm", "xout", "o_next", "y")


def layer_stack_supported(nl, M, D, F, Hq, Hk, HD, L, stream=False, kv_nt=False):
    """True when ``layer_stack`` runs nl layers of these shapes with these weight / cache-load
    modes."""
    return _ffi.lib().ecd_layer_stack_supported(
        int(nl), int(M), int(D), int(F), int(Hq), int(Hk), int(HD), int(L),
        (2 if stream else 0) | (8 if kv_nt else 0)) == _ffi.ECD_OK


def layer_stack_layers_per_launch(nl, M, D, F, Hq, Hk, HD, L, stream=False, kv_nt=False):
    """Layers per kernel launch of a ``layer_stack`` call (0 when not supported)."""
    r = _ffi.lib().ecd_layer_stack_layers_per_launch(
        int(nl), int(M), int(D), int(F), int(Hq), int(Hk), int(HD), int(L),
        (2 if stream else 0) | (8 if kv_nt else 0))
    return max(int(r), 0)


def layer_stack_plan(layers, M, D, F, Hq, Hk, HD, dev):
    """The device plan of a layer stack: ``layers`` is a list of dicts with the tensors of
    STACK_FIELDS (n1, wq, sq, kc, vc, o_next None only for the last layer; ``y``, a [M, N] view
    with 16-byte aligned rows, only in the last layer of a 1024-wide stack: it then ends in a
    codebook head with n1, wq, sq the head's norm, packed weights and scales, and no caches).
    The library checks the records (alignment, every layer but the last running the next layer's
    attention, all outputs disjoint) and copies them to the returned uint8 device tensor."""
    nl = len(layers)
    rec = np.zeros((nl, len(STACK_FIELDS)), np.uint64)
    for i, lay in enumerate(layers):
        for j, f in enumerate(STACK_FIELDS):
            t = lay.get(f)
            rec[i, j] = 0 if t is None else t.data_ptr()
    y = layers[-1].get("y")
    yld = 0 if y is None else y.stride(0)
    if y is not None and (y.stride(1) != 1 or yld % 8 or y.shape[0] != M):
        raise ValueError("layer_stack_plan: y must be [M, N], unit column stride, 16-byte rows")
    nb = int(_ffi.lib().ecd_layer_stack_plan_bytes(nl))
    plan = torch.empty(max(nb, 16), device=dev, dtype=torch.uint8)
    _ffi.call("ecd_layer_stack_plan", rec.ctypes.data, nl, M, D, F, Hq, Hk, HD, yld,
              plan.data_ptr(), stream_ptr(dev))
    return plan


def layer_stack(plan, nl, o, xin, xout, rope, pos, q, sync, err, ws, S, Hq, Hk, L, HD, F,
                eps=1e-5, stream=False, no_wait=False, kv_nt=False, y=None):
    """The nl layer tails of ``plan`` (layer_stack_plan) as one launch: layer 0 starts from o
    [M, Hq * HD] and xin [M, D]; each layer's attention output and result feed the next layer.
    Returns ``xout``, the last layer's output buffer of the plan, or ``y``, the logits of a plan
    that ends in a codebook head (the plan's y).  rope, pos, q, sync, err, ws, ``no_wait`` and
    ``kv_nt`` as for layer_tail (sync, err and ws shared with the stack's other layer-tail
    launches)."""
    dev = _dev(o, "layer_stack")
    M, D = xin.shape
    for t, n in ((o, "o"), (xin, "xin")):
        _f16(t, f"layer_stack {n}")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"layer_stack: {n} must be contiguous and 16-byte aligned")
    if o.numel() != M * Hq * HD:
        raise ValueError("layer_stack: o must be [M, Hq * HD]")
    if pos.dtype != torch.int64 or pos.numel() != M or not pos.is_contiguous():
        raise ValueError("layer_stack: pos must be contiguous int64 [M]")
    if q.numel() != M * Hq * HD or not q.is_contiguous():
        raise ValueError("layer_stack: q must be contiguous [M, Hq * HD]")
    if rope.shape[0] < L or rope.shape[1] != HD // 2:
        raise ValueError("layer_stack: rope table must be float32 [>= L, HD/2, 2]")
    if sync.dtype != torch.int32 or sync.numel() < 4096 or sync.data_ptr() % 256:
        raise ValueError("layer_stack: sync must be int32 [>= 4096], 256-byte aligned")
    if err.dtype != torch.int32 or err.numel() < 1:
        raise ValueError("layer_stack: err must be int32 [1]")
    if ws.dtype != torch.float32 or ws.data_ptr() % 16 or \
            ws.numel() * 4 < layer_tail_ws_bytes(D, Hq, Hk, HD):
        raise ValueError("layer_stack: ws must be float32, 16-byte aligned, layer_tail_ws_bytes")
    if plan.dtype != torch.uint8 or plan.numel() < int(_ffi.lib().ecd_layer_stack_plan_bytes(nl)):
        raise ValueError("layer_stack: plan must come from layer_stack_plan for nl layers")
    _ffi.call("ecd_layer_stack", plan.data_ptr(), nl, o.data_ptr(), xin.data_ptr(),
              rope.data_ptr(), pos.data_ptr(), q.data_ptr(), sync.data_ptr(), err.data_ptr(),
              ws.data_ptr(), M, D, F, S, Hq, Hk, L, HD, 0 if y is None else y.shape[1],
              0 if y is None else y.stride(0), float(eps),
              _flags(M, stream) | (4 if no_wait else 0) | (8 if kv_nt else 0), stream_ptr(dev))
    return xout if y is None else y


def layer_head(x, nxt, o_next, F, sync, err, ws, eps=1e-5, stream=False, no_wait=False,
               kv_nt=False):
    """A stack's first layer up to its attention as one launch (app/engine.py:189-204 for layer
    0): rms(x, n1) -> q|k|v -> RoPE -> q and the cache slot, and the decode attention into
    o_next [M, Hq * HD].  ``nxt`` as for layer_tail (that layer's n1, wq, ..., S = 1); F: the
    stack's FFN width; sync, err, ws: the stack's layer_tail buffers; ``no_wait`` and
    ``kv_nt`` as for layer_tail."""
    dev = _dev(x, "layer_head")
    M, D = x.shape
    _f16(x, "layer_head x")
    _f16(o_next, "layer_head o_next")
    n = nxt
    pos, kc = n["pos"], n["kc"]
    S, Hq, Hk, L, HD = n["S"], n["Hq"], n["Hk"], n["L"], n["HD"]
    if not x.is_contiguous() or x.data_ptr() % 16:
        raise ValueError("layer_head: x must be contiguous and 16-byte aligned")
    if pos.dtype != torch.int64 or pos.numel() != M or not pos.is_contiguous():
        raise ValueError("layer_head: pos must be contiguous int64 [M]")
    if kc.shape != (kc.shape[0], Hk, L, HD) or kc.shape[0] * S < M or n["vc"].shape != kc.shape:
        raise ValueError("layer_head: caches must be [B, Hk, L, HD] with B * S >= M")
    if n["q"].numel() != M * Hq * HD or not n["q"].is_contiguous():
        raise ValueError("layer_head: q must be contiguous [M, Hq * HD]")
    if n["rope"].shape[0] < L or n["rope"].shape[1] != HD // 2:
        raise ValueError("layer_head: rope table must be float32 [>= L, HD/2, 2]")
    if o_next.numel() != M * Hq * HD or not o_next.is_contiguous() or o_next.data_ptr() % 16:
        raise ValueError("layer_head: o_next must be contiguous [M, Hq * HD]")
    if sync.dtype != torch.int32 or sync.numel() < 4096 or sync.data_ptr() % 256:
        raise ValueError("layer_head: sync must be int32 [>= 4096], 256-byte aligned")
    if err.dtype != torch.int32 or err.numel() < 1:
        raise ValueError("layer_head: err must be int32 [1]")
    if ws.dtype != torch.float32 or ws.data_ptr() % 16 or \
            ws.numel() * 4 < layer_tail_ws_bytes(D, Hq, Hk, HD):
        raise ValueError("layer_head: ws must be float32, 16-byte aligned, layer_tail_ws_bytes")
    _ffi.call("ecd_layer_head", x.data_ptr(), n["n1"].data_ptr(), n["wq"].data_ptr(),
              n["sq"].data_ptr(), n["rope"].data_ptr(), pos.data_ptr(), n["q"].data_ptr(),
              kc.data_ptr(), n["vc"].data_ptr(), o_next.data_ptr(), sync.data_ptr(),
              err.data_ptr(), ws.data_ptr(), M, D, F, S, Hq, Hk, L, HD, float(eps),
              _flags(M, stream) | (4 if no_wait else 0) | (8 if kv_nt else 0), stream_ptr(dev))
    return o_next


def embed_gemv_packed(tok, table, tscale, cb, vocab, wp, s, N, even=None, stream=False, out=None,
                      dense=None):
    """int8_mm(Emb(tok[:, 0] + cb * vocab), w, s); with ``even`` [B, K] the input rows are the
    interleave (even[b], emb[b]) and the output has 2B rows.  ``table`` holds int8 rows scaled by
    ``tscale``, or dense fp16 rows when ``tscale`` is None.  ``out``: a contiguous [M, N] fp16
    destination; ``dense``: the numerics (None: int8_mm's rule, dense for more than 16 rows)."""
    dev = _dev(tok, "embed_gemv_packed")
    if tok.dtype != torch.int64:
        raise TypeError("embed_gemv_packed: tok must be int64")
    if (tscale is None) != (table.dtype == torch.float16) or table.dtype not in (torch.int8, torch.float16):
        raise TypeError("embed_gemv_packed: int8 table with scales, or fp16 table without")
    B = tok.shape[0]
    K = table.shape[1]
    M = 2 * B if even is not None else B
    if even is not None:
        _f16(even, "embed_gemv_packed even")
        if even.shape != (B, K) or not even.is_contiguous() or even.data_ptr() % 16:
            raise ValueError("embed_gemv_packed: even must be contiguous [B, K]")
    if out is not None:
        _f16(out, "embed_gemv_packed out")
        if out.shape != (M, N) or not out.is_contiguous():
            raise ValueError(f"embed_gemv_packed: out must be contiguous [{M}, {N}]")
    y = torch.empty(M, N, device=dev, dtype=torch.float16) if out is None else out
    fl = _flags(M, stream) if dense is None else (int(bool(dense)) | (2 if stream else 0))
    _ffi.call("ecd_embed_gemv_i8p", tok.data_ptr(), tok.stride(0), table.data_ptr(), _ptr(tscale),
              table.shape[0], int(cb), int(vocab), _ptr(even), wp.data_ptr(), s.data_ptr(),
              y.data_ptr(), N, M, N, K, fl, stream_ptr(dev))
    return y


# ---------------------------------------------------------------- pages of a KV cache
def _on(t, dev, call, name, dtype, shape):
    """t is a contiguous tensor of dtype and shape on dev."""
    if t.dtype is dtype and t.shape == shape and t.device == dev and t.is_contiguous():
        return
    if t.dtype is not dtype:
        raise TypeError(f"{call}: {name}: expected {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{call}: {name} is on {t.device}, the call's other tensors on {dev}")
    raise ValueError(f"{call}: {name}: expected a contiguous tensor of shape {tuple(shape)}, got {tuple(t.shape)}")


def _call_on(dev, name, *args):
    """_ffi.call with the tensors' device as the current one, on its current stream (asked for as its handle: a stream
    object costs as much as a launch)."""
    i = dev.index
    if i == torch._C._cuda_getDevice():  # (_ffi.call's steps, without passing the arguments on once more)
        rc = getattr(_ffi.lib(), name)(*args, torch._C._cuda_getCurrentRawStream(i))
        if rc:
            _ffi.check(rc, name)
    else:
        with torch.cuda.device(dev):
            _ffi.call(name, *args, torch._C._cuda_getCurrentRawStream(i))


INT_MOST = 0x7FFFFFFF  # (the library takes counts as 32-bit numbers: a larger one would wrap)


def _page_state(name, ref, table, length, err, page=1):
    dev = _dev(ref, name)
    if not 1 <= page <= INT_MOST:
        raise ValueError(f"{name}: {page} slots of a page")
    if table.dim() != 2:
        raise ValueError(f"{name}: table must be [B, MP]")
    B, MP = table.shape
    _on(ref, dev, name, "ref", torch.int32, (ref.numel(),))
    _on(table, dev, name, "table", torch.int32, (B, MP))
    _on(length, dev, name, "length", torch.int64, (B,))
    _on(err, dev, name, "err", torch.int32, (1,))
    return dev, ref.numel(), B, MP


def _page_pool(name, kv, ref):
    if kv.dim() != 6:
        raise ValueError(f"{name}: kv must be [layers, 2, NP, Hk, P, HD]")
    layers, _, NP, Hk, P, HD = kv.shape
    _on(kv, ref.device, name, "kv", torch.float16, (layers, 2, ref.numel(), Hk, P, HD))
    if HD % 8 or kv.data_ptr() % 16:
        raise ValueError(f"{name}: head_dim must be a multiple of 8 and kv 16-byte aligned")
    return layers * 2, Hk, P, HD


def page_free(ref, table, length, seqs, page, err):
    """The sequences ``seqs`` [n] int32 give their pages back: a page whose last owner goes is free.  ``ref`` [NP] int32
    owners of each page, ``table`` [B, MP] int32 page numbers (-1 behind a sequence's last), ``length`` [B] int64 slots
    held, ``page`` slots of a page; ``err`` [1] int32 collects what was refused (include/ecdecode.h lists its bits)."""
    dev, NP, B, MP = _page_state("page_free", ref, table, length, err, page)
    n = seqs.numel()
    _on(seqs, dev, "page_free", "seqs", torch.int32, (n,))
    if n:
        _call_on(dev, "ecd_page_free", ref.data_ptr(), NP, table.data_ptr(), MP, length.data_ptr(), B, int(page),
                 seqs.data_ptr(), n, err.data_ptr())


def page_fork(kv, ref, table, length, src, dst, err):
    """Sequence dst[i] (holding nothing) becomes a copy of src[i] (int32 [n], n <= 1024): whole pages shared, the slots
    of a last page that is not full copied into a page of its own in every layer of ``kv`` [layers, 2, NP, Hk, P, HD]."""
    dev, NP, B, MP = _page_state("page_fork", ref, table, length, err)
    planes, Hk, P, HD = _page_pool("page_fork", kv, ref)
    n = src.numel()
    _on(src, dev, "page_fork", "src", torch.int32, (n,))
    _on(dst, dev, "page_fork", "dst", torch.int32, (n,))
    if n:
        plan = torch.empty(4 * n, device=dev, dtype=torch.int32)
        _call_on(dev, "ecd_page_fork", kv.data_ptr(), ref.data_ptr(), NP, table.data_ptr(), MP, length.data_ptr(), B,
                 src.data_ptr(), dst.data_ptr(), n, plan.data_ptr(), err.data_ptr(), planes, Hk, P, HD)


def page_extend(ref, table, length, pos, page, err):
    """Every sequence b holds slot pos[b] (int64 [B], B <= 1024) afterwards; -1, or a slot it holds, leaves it alone."""
    dev, NP, B, MP = _page_state("page_extend", ref, table, length, err, page)
    _on(pos, dev, "page_extend", "pos", torch.int64, (B,))
    _call_on(dev, "ecd_page_extend", ref.data_ptr(), NP, table.data_ptr(), MP, length.data_ptr(), B, int(page),
             pos.data_ptr(), err.data_ptr())


def page_compact(kv, ref, table, length, kv2, ref2, table2, length2, err):
    """The pages in use, in ascending order, to the first pages of another pool kv2 [layers, 2, NP2, Hk, P, HD], with the
    state ref2 [NP2], table2 [B, MP], length2 [B] that goes with them.  The first pool and its state stay as they are."""
    dev, NP, B, MP = _page_state("page_compact", ref, table, length, err)
    planes, Hk, P, HD = _page_pool("page_compact", kv, ref)
    NP2 = ref2.numel()
    _on(ref2, dev, "page_compact", "ref2", torch.int32, (NP2,))
    _on(kv2, dev, "page_compact", "kv2", torch.float16, (kv.shape[0], 2, NP2, Hk, P, HD))
    _on(table2, dev, "page_compact", "table2", torch.int32, (B, MP))
    _on(length2, dev, "page_compact", "length2", torch.int64, (B,))
    for a, b in ((kv, kv2), (ref, ref2), (table, table2), (length, length2)):
        lo, hi = a.data_ptr(), a.data_ptr() + a.numel() * a.element_size()
        if b.data_ptr() < hi and lo < b.data_ptr() + b.numel() * b.element_size():
            raise ValueError("page_compact: the two pools and their states must not overlap")
    ws = torch.empty(1 + 2 * NP, device=dev, dtype=torch.int32)
    _call_on(dev, "ecd_page_compact", kv.data_ptr(), ref.data_ptr(), NP, table.data_ptr(), length.data_ptr(),
             kv2.data_ptr(), ref2.data_ptr(), NP2, table2.data_ptr(), length2.data_ptr(), B, MP, ws.data_ptr(),
             err.data_ptr(), planes, Hk, P, HD)


def _paged(name, kp, vp, table, dev):
    """(NP, Hk, P, HD, MP, table stride) of the pages and the table of a call."""
    if kp.dim() != 4 or table.dim() != 2:
        raise ValueError(f"{name}: kp / vp must be [NP, Hk, P, HD] and table [B, MP]")
    shape = kp.shape
    _on(kp, dev, name, "kp", torch.float16, shape)
    _on(vp, dev, name, "vp", torch.float16, shape)
    MP, (ld, one) = table.shape[1], table.stride()
    if table.dtype is not torch.int32 or table.device != dev or one != 1 or ld < MP:
        raise ValueError(f"{name}: table must be int32 [B, MP] with contiguous rows on {dev}")
    if kp.data_ptr() % 16 or vp.data_ptr() % 16:
        raise ValueError(f"{name}: kp and vp must be 16-byte aligned")
    return *shape, MP, ld


def _rows16(t, name):
    """(device, row stride) of a [M, N] fp16 GPU tensor with unit inner stride and 16-byte rows."""
    dev = t.device
    if t.dtype is torch.float16 and t.is_cuda and t.dim() == 2:
        ld, one = t.stride()
        if one == 1 and ld % 8 == 0 and t.data_ptr() % 16 == 0:
            return dev, ld
    _dev(t, name)
    _f16(t, name)
    raise ValueError(f"{name}: must be [M, N] with unit inner stride and 16-byte rows")


def paged_write(qkv, kp, vp, table, pos, S, Hq, Hk, rope=None, q=None):
    """K and V of the rows of ``qkv`` [M, (Hq + 2 Hk) HD] into pages: row m belongs to sequence m // S at slot pos[m]
    (int64 [M]); ``kp`` / ``vp`` [NP, Hk, P, HD], ``table`` [B, MP] int32 with B S >= M.  With ``rope`` [L, HD/2, 2]
    float32, q and k are rotated first (the numerics of _rope_cache) and q [M, Hq HD] is returned (``q``: its
    destination); without it nothing is.  A row whose slot has no page writes nothing into the cache; the others of a call
    name different slots."""
    dev, ld = _rows16(qkv, "paged_write qkv")
    NP, hk, P, HD, MP, ldt = _paged("paged_write", kp, vp, table, dev)
    M, W = qkv.shape
    if hk != Hk or W != (Hq + 2 * Hk) * HD or HD % 8 or not 1 <= S <= INT_MOST or table.shape[0] * S < M:
        raise ValueError("paged_write: qkv must be [M, (Hq + 2 Hk) HD], kp / vp [NP, Hk, P, HD], table [B, MP] with "
                         "B * S >= M")
    _on(pos, dev, "paged_write", "pos", torch.int64, (M,))
    L = 0
    if rope is not None:
        L = rope.shape[0]
        _on(rope, dev, "paged_write", "rope", torch.float32, (L, HD // 2, 2))
        q = torch.empty(M, Hq * HD, device=dev, dtype=torch.float16) if q is None else q
        _on(q, dev, "paged_write", "q", torch.float16, (M, Hq * HD))
    else:
        q = None
    if M:
        _call_on(dev, "ecd_paged_write", qkv.data_ptr(), ld, _ptr(rope), L, pos.data_ptr(), _ptr(q), kp.data_ptr(),
                 vp.data_ptr(), table.data_ptr(), ldt, MP, NP, M, int(S), Hq, Hk, P, HD)
    return q


class PagedAttnPlan:
    """How paged_attn cuts a batch into parts (paged_attn_plan)."""

    def __init__(self, items, rows, nown, parts, ctiles, waves, Hq, Hk, HD, dev):
        self.nitems, self.R, self.nown, self.parts = len(items), len(rows), nown, parts
        self.ctiles, self.waves = ctiles, waves
        self.Hq, self.Hk, self.HD = Hq, Hk, HD
        flat = torch.tensor([v for x in rows for v in x] + [v for x in items for v in x], dtype=torch.int32, device=dev)
        self.flat = flat
        self.rows_ptr, self.items_ptr = flat.data_ptr(), flat.data_ptr() + 8 * self.R
        heads = self.R * Hq
        self.ws = 0 if parts == 1 else 2 * (-(-heads * parts // 4) * 4) + heads * parts * HD
        self.dev = flat.device


# How a batch is cut, from times on an MI355X (24 query heads on 8 kv heads of 128; other heads follow the same rules, by their
# bytes and slots, not measured one by one; us):
# sharing pays where it saves this many bytes of the other rows' reads, else the parts cost more than they save; taken for the
# whole batch, since one group's parts already bring the join: then every prefix is shared, a short one too
# (shared / not: 8 rows of 4096 + 64 slots, 117 MB saved, 16.0 / 22.7; 2 x 4 of 1500 + 500, 37 MB, 14.5 / 14.0; 2 x 16 of
# 256 + 500, 31 MB, 18.0 / 15.1; 2 x 4 of 256 + 494, 6 MB, 10.3 / 10.4)
PLAN_SAVED = 48 << 20
# workgroups that the shared parts are cut for (2 x 16 rows of 4096: 128 28.1, 256 29.1, 384 32.2; 2 x 32 of 7000: 42.1 with
# 256, 46.0 with 384)
PLAN_SHARED_WG = 256
# a row's own slots: parts so that all rows together have this many workgroups and, as far as PLAN_OWN_MOST parts go, none has
# more than PLAN_OWN_SLOTS of the longest row that max_len allows (8 rows of 256 + 3000: 4 parts 22.4, 7 parts 23.1; 2 x 16 of
# 1000 + 4000: 2 parts 71, 4 parts 64)
PLAN_OWN_WG, PLAN_OWN_SLOTS, PLAN_OWN_MOST = 256, 1280, 16
# one workgroup (of eight waves; head_dim 256 of four) for a row and kv head, nothing to join: rows of few slots (8 rows of
# 160: 5.7, in parts 7.5; of 750: 11.7 and 10.4), or as many pairs as CUs (2 x 16 rows of 100 + 2000, ragged: 32.6 and 35.6)
PLAN_SOLO_BYTES, PLAN_SOLO_WG = 512 * 512, 256


def paged_attn_plan(groups, Hq, Hk, HD, max_len, device="cuda", share=None):
    """The plan of paged_attn for rows in ``groups``: a list of (rows, prefix), consecutive rows whose first ``prefix``
    slots are the same (0: nothing shared).  ``max_len``: the most slots that a row may come to hold (a prefix of more is
    not shared: no row attends all of it).  Made once for all layers and steps in which the groups stay the same (it
    copies to the device: not under graph capture), and kept until the work that uses it is done.  ``share``: whether
    prefixes are read once per group (None: where that saves more than joining the parts costs, for the whole batch)."""
    dev = torch.device(device)
    if dev.type != "cuda":
        raise RuntimeError("paged_attn_plan: the decode path runs only on a ROCm GPU")
    groups = [(int(n), int(p)) for n, p in groups]
    if not groups or max_len < 0 or any(n < 1 or p < 0 for n, p in groups):
        raise ValueError("paged_attn_plan: groups must be (rows >= 1, prefix >= 0) pairs and max_len >= 0")
    if Hk < 1 or Hq % Hk or Hq // Hk > 16 or HD not in (64, 128, 256):
        raise ValueError("paged_attn_plan: head_dim 64, 128 or 256 and at most 16 query heads per kv head")
    return _make_plan(groups, Hq, Hk, HD, int(max_len), dev, share)


def _make_plan(groups, Hq, Hk, HD, max_len, dev, share=None):
    G = Hq // Hk
    groups = [(n, p if p <= max_len else 0) for n, p in groups]
    R = sum(n for n, _ in groups)
    slot = 4 * HD  # bytes of a slot's key and value
    if share is None:
        share = sum((n - 1) * p for n, p in groups) * Hk * slot > PLAN_SAVED
    if not share and (R * Hk >= PLAN_SOLO_WG or max_len * slot <= PLAN_SOLO_BYTES):
        # one workgroup per row and kv head, which writes the output itself
        return PagedAttnPlan([], [(0, 0)] * R, 1, 1, 1, 8 if HD <= 128 else 4, Hq, Hk, HD, dev)
    shared = [share and n > 1 and p > 0 for n, p in groups]
    cols = max([n * G for (n, p), s in zip(groups, shared) if s], default=0)
    ct = 2 if cols > 16 and HD <= 128 else 1
    fit = 16 * ct // G  # rows of a shared part
    slots = sum(p * -(-n // fit) for (n, p), s in zip(groups, shared) if s) * Hk
    per = max(128, -(-slots // (PLAN_SHARED_WG * 128)) * 128)
    units, rows, r0, most = [], [], 0, 0
    for (n, p), s in zip(groups, shared):
        splits = -(-p // per) if s else 0
        chunks = -(-n // fit)
        for k in range(splits):
            units += [[(r0 + n * c // chunks, n * (c + 1) // chunks - n * c // chunks, k * per, min(p, (k + 1) * per), k, h)
                       for c in range(chunks)] for h in range(Hk)]
        rows += [(p if s else 0, splits)] * n
        most = max(most, splits)
        r0 += n
    # the parts that read the same slots get numbers that are equal modulo 8: one XCD, whose L2 then holds the slots
    items = []
    for u in range(0, len(units), 8):
        eight = units[u:u + 8]
        for c in range(max(len(x) for x in eight)):
            items += [x[c] for x in eight if c < len(x)]
    longest = max(max_len - (p if s else 0) for (n, p), s in zip(groups, shared))
    nown = max(1, min(PLAN_OWN_MOST, max(-(-PLAN_OWN_WG // (R * Hk)), -(-longest // PLAN_OWN_SLOTS)), -(-longest // 128)))
    return PagedAttnPlan(items, rows, nown, most + nown, ct, 4, Hq, Hk, HD, dev)


def paged_attn(q, kp, vp, table, pos, plan, S=1, scale=None, out=None):
    """Decode attention over pages: row r of ``q`` [>= R, Hq HD] (R: the plan's rows) attends slots [0, pos[r]] of
    sequence r // S through ``table`` [B, MP] int32, and the slots that a group shares are read once for the group.
    ``kp`` / ``vp`` [NP, Hk, P, HD], P a power of two from 16; ``pos`` int64 [>= R], -1: the row attends nothing and its
    output is 0; a position behind the table's last slot: all of them.  Rows of ``out`` behind the plan's are left as they
    are (whatever the memory holds where out is None).  The result of a row does not depend on what lies in slots that it
    does not attend."""
    dev, ldq = _rows16(q, "paged_attn q")
    NP, hk, P, hd, MP, ldt = _paged("paged_attn", kp, vp, table, dev)
    R, Hq, Hk, HD = plan.R, plan.Hq, plan.Hk, plan.HD
    rows, wide = q.shape
    if plan.dev != dev:
        raise ValueError(f"paged_attn: the plan is on {plan.dev}, the tensors on {dev}")
    if hk != Hk or hd != HD or wide != Hq * HD or rows < R or not 1 <= S <= INT_MOST or table.shape[0] * S < R:
        raise ValueError("paged_attn: q [>= R, Hq HD], kp / vp [NP, Hk, P, HD] and table [B, MP] (B * S >= R) must fit "
                         "the plan")
    if P < 16 or P & (P - 1):
        raise ValueError("paged_attn: the page size must be a power of two from 16")
    n = pos.numel()
    _on(pos, dev, "paged_attn", "pos", torch.int64, (n,))
    if n < R:
        raise ValueError("paged_attn: pos must hold a slot for each row")
    scale = HD ** -0.5 if scale is None else float(scale)
    if not scale > 0:
        raise ValueError("paged_attn: scale must be positive")
    if out is None:
        o = torch.empty(rows, wide, device=dev, dtype=torch.float16)
    else:
        o = out
        _on(o, dev, "paged_attn", "out", torch.float16, (rows, wide))
    ws = torch.empty(plan.ws, device=dev, dtype=torch.float32) if plan.ws else None  # (held until the launch)
    _call_on(dev, "ecd_paged_attn", q.data_ptr(), ldq, kp.data_ptr(), vp.data_ptr(), table.data_ptr(), ldt,
             pos.data_ptr(), o.data_ptr(), _ptr(ws), plan.items_ptr, plan.rows_ptr, plan.nitems, plan.nown, plan.parts,
             plan.ctiles, plan.waves, R, int(S), MP, NP, Hq, Hk, P, HD, scale)
    return o


# ---------------------------------------------------------------- int8 activations
def quant_a8(x, nw=None, eps=1e-5):
    """(codes, scale) of the rows of x [M, K] fp16, or of their RMS norm with weight ``nw`` [K] (kept in fp32, not
    rounded to fp16): scale[m] = max |y[m]| / 127 fp32, codes int8 [M, K] = rint(127 y / max |y|), ties to even.  A row
    of zeros has scale 0; one that holds an infinity or a NaN has scale NaN.  The codes' rows are zero padded to a
    multiple of 128 (their stride)."""
    dev, ld = _rows16(x, "quant_a8 x")
    M, K = x.shape
    if K % 64 or not 0 < K <= 1 << 17:
        raise ValueError("quant_a8: K must be a multiple of 64, at most 131072")
    if nw is not None:
        _on(nw, dev, "quant_a8", "nw", torch.float16, (K,))
        if nw.data_ptr() % 16:
            raise ValueError("quant_a8: nw must be 16-byte aligned")
    ldc = -(-K // 128) * 128
    c = torch.empty(M, ldc, device=dev, dtype=torch.int8)
    s = torch.empty(M, device=dev, dtype=torch.float32)
    if M:
        _call_on(dev, "ecd_quant_a8", x.data_ptr(), ld, _ptr(nw), float(eps), c.data_ptr(), ldc, s.data_ptr(), M, K)
    return (c if ldc == K else c[:, :K]), s


def _a8_args(name, c, sx, wp, s, N, K):
    dev = _dev(c, name)
    if c.dtype is not torch.int8 or c.dim() != 2 or c.shape[1] != K or c.stride(1) != 1 or c.stride(0) % 128 or \
            c.data_ptr() % 16:
        raise ValueError(f"{name}: codes must come from quant_a8 (int8 [M, {K}], rows padded to a multiple of 128)")
    M = c.shape[0]
    _on(sx, dev, name, "scale", torch.float32, (M,))
    _on(s, dev, name, "s", torch.float16, (N,))
    if wp.dtype is not torch.int8 or wp.device != dev or not wp.is_contiguous() or wp.numel() < -(-N // 16) * 16 * K:
        raise ValueError(f"{name}: wp must be pack_i8 of an [N, K] matrix on {dev}")
    return dev, M


def gemm_a8_packed(c, sx, wp, s, N, K, res=None, out=None):
    """y[m, n] = fp16(sx[m] s[n] sum_k c[m, k] q[n, k] (+ res[m, n])) -> [M, N]: int8 codes (quant_a8) times int8
    weights (pack_i8) with one scale per row and per output channel, the sum exact, one rounding at the end.  A row's
    result does not depend on the other rows of the call."""
    dev, M = _a8_args("gemm_a8_packed", c, sx, wp, s, N, K)
    y = torch.empty(M, N, device=dev, dtype=torch.float16) if out is None else out
    for t, nm in ((y, "out"), (res, "res")):
        if t is not None and (t.dtype != torch.float16 or t.device != dev or t.shape != (M, N) or t.stride(1) != 1
                              or t.stride(0) < N):
            raise ValueError(f"gemm_a8_packed: {nm} must be fp16 [M, N] with unit inner stride")
    if M:
        _call_on(dev, "ecd_gemm_a8", c.data_ptr(), c.stride(0), sx.data_ptr(), wp.data_ptr(), s.data_ptr(), _ptr(res),
                 0 if res is None else res.stride(0), y.data_ptr(), y.stride(0), M, N, K)
    return y


def gemm_a8_silu_packed(c, sx, wp, s, F, K, out=None):
    """silu(a) * b -> [M, F] for the products a, b of gemm_a8_packed on row-interleaved w1 | w3 (pack_i8(...,
    interleave=True), ``s`` interleaved likewise), in fp32 with one rounding at the end."""
    dev, M = _a8_args("gemm_a8_silu_packed", c, sx, wp, s, 2 * F, K)
    mm = torch.empty(M, F, device=dev, dtype=torch.float16) if out is None else out
    if mm.dtype != torch.float16 or mm.device != dev or mm.shape != (M, F) or mm.stride(1) != 1 or mm.stride(0) < F:
        raise ValueError("gemm_a8_silu_packed: out must be fp16 [M, F] with unit inner stride")
    if M:
        _call_on(dev, "ecd_gemm_a8_silu", c.data_ptr(), c.stride(0), sx.data_ptr(), wp.data_ptr(), s.data_ptr(),
                 mm.data_ptr(), mm.stride(0), M, F, K)
    return mm


# ---------------------------------------------------------------- 4-bit weights
class PackedQ4:
    """An [N, K] matrix of 4-bit weights laid out for mm_q4 and mm_q4_silu (pack_q4)."""

    def __init__(self, codes, scales, N, K, group, zeros, interleave):
        self.codes, self.scales = codes, scales
        self.N, self.K, self.group, self.zeros, self.interleave = N, K, group, zeros, interleave
        self.dev = codes.device
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()
        self.plans = {}  # rows -> plan(rows): it depends on sizes alone

    def plan(self, M):
        """(choice of the kernel, workspace bytes) of a product of M rows, and of one with a norm."""
        lib, N, K = _ffi.lib(), self.N, self.K
        n, f = lib.ecd_mm_q4_choice(M, N, K), lib.ecd_mm_q4_norm_choice(M, N, K, self.interleave)
        p = self.plans[M] = ((n, lib.ecd_mm_q4_ws_bytes(M, N, K, n, 0)), (f, lib.ecd_mm_q4_ws_bytes(M, N, K, f, 1)))
        return p

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel() * 2


def pack_q4(q4, s4, z4=None, interleave=False):
    """4-bit weights in groups (quant.q4_rows) -> PackedQ4: q4 uint8 [N, K / 2] (element 2 i in the low half of byte i), s4
    fp16 [N, groups], z4 uint8 [N, groups] or None (zero point 8), groups = K / 32, 64 or 128 rounded up.  With
    ``interleave`` the two halves of the rows are interleaved (w1 | w3 -> pairs, for mm_q4_silu)."""
    dev = _dev(q4, "pack_q4")
    if q4.dim() != 2 or s4.dim() != 2:
        raise ValueError("pack_q4: q4 must be [N, K / 2] and s4 [N, groups]")
    N, K = q4.shape[0], 2 * q4.shape[1]
    if K % 64 or not 0 < K <= INT_MOST or not 0 < N <= INT_MOST - 32 or (interleave and N % 2):
        raise ValueError("pack_q4: K must be a multiple of 64 (and N even to interleave)")
    ng = s4.shape[1]
    group = next((g for g in (128, 64, 32) if -(-K // g) == ng), 0)
    if not group:
        raise ValueError(f"pack_q4: {ng} groups of {K} weights are none of 32, 64 or 128")
    _on(q4, dev, "pack_q4", "q4", torch.uint8, (N, K // 2))
    _on(s4, dev, "pack_q4", "s4", torch.float16, (N, ng))
    if z4 is not None:
        _on(z4, dev, "pack_q4", "z4", torch.uint8, (N, ng))
    if q4.data_ptr() % 4:
        q4 = q4.clone()
    codes = torch.empty(_ffi.lib().ecd_packed_bytes_q4(N, K), device=dev, dtype=torch.uint8)
    scales = torch.empty(ng * (-(-N // 32) * 32) * (1 if z4 is None else 2), device=dev, dtype=torch.float16)
    _call_on(dev, "ecd_pack_q4", q4.data_ptr(), s4.data_ptr(), _ptr(z4), N, K, group, int(interleave), codes.data_ptr(),
             scales.data_ptr())
    return PackedQ4(codes, scales, N, K, group, z4 is not None, bool(interleave))


Q4_TILE_LD = 1 << 23  # the largest stride of x's rows that every tile takes


def _mm_q4(name, x, w, cols, res, nw, eps, out, silu):
    try:
        dev, ldx = _rows16(x, name)
    except ValueError:
        if x.dim() != 2 or x.shape[0] != 1 or x.shape[1] % 8:
            raise
        x = x.as_strided(x.shape, (x.shape[1], x.stride(1)))  # (one row: its stride says nothing)
        dev, ldx = _rows16(x, name)
    M, K = x.shape
    if K != w.K or dev != w.dev or w.interleave is not silu or M > INT_MOST:
        if w.interleave is not silu:
            raise ValueError(f"{name}: the weights were packed {'with' if w.interleave else 'without'} interleave")
        if dev != w.dev:
            raise ValueError(f"{name}: the weights are on {w.dev}, x on {dev}")
        raise ValueError(f"{name}: x must be [M, {w.K}]")
    if M <= 1:
        ldx = K
    np = rp = wp = None
    ldr = 0
    if nw is not None:
        _on(nw, dev, name, "nw", torch.float16, (K,))
        np = nw.data_ptr()
        if np % 16:
            raise ValueError(f"{name}: nw must be 16-byte aligned")
    if res is not None:
        ldr = _rows_of(res, M, cols, dev, name, "res")
        rp = res.data_ptr()
    if out is None:
        out, ldy = torch.empty(M, cols, device=dev, dtype=torch.float16), cols
    else:
        ldy = _rows_of(out, M, cols, dev, name, "out")
        if _meet(out, ldy, x, ldx):
            raise ValueError(f"{name}: out must not overlap x")
        if res is not None and _meet(out, ldy, res, ldr) and not (rp == out.data_ptr() and (ldy == ldr or M == 1)):
            raise ValueError(f"{name}: out must be apart from res or the same rows")
    if M:
        plan, nb = (w.plans.get(M) or w.plan(M))[0 if np is None else 1]
        if ldx > Q4_TILE_LD and M > 16 and np is None:  # (the few-row kernel's offsets reach 8 times as far as a tile's)
            plan, nb = 19 + 256, 0
        if nb:
            ws = torch.empty(nb, device=dev, dtype=torch.uint8)  # (held until the launch)
            wp = ws.data_ptr()
        _call_on(dev, "ecd_mm_q4", x.data_ptr(), ldx, np, eps, w.codes_ptr, w.scales_ptr, w.zeros, w.group, rp, ldr,
                 out.data_ptr(), ldy, M, w.N, K, silu, plan, wp)
    return out


def _ends(t):
    """First byte of a tensor with positive strides, and the one behind its last."""
    a = t.data_ptr()
    return a, a + (1 + sum((n - 1) * d for n, d in zip(t.shape, t.stride()))) * t.element_size() if t.numel() else a


def _meet(t, ldt, u, ldu):
    """Whether fp16 matrices of row strides ldt and ldu (at least their width) share memory, or might: columns of the same wide
    rows that do not meet share none."""
    (lo, hi), (a, b) = _ends(t), _ends(u)
    if lo >= b or a >= hi:
        return False
    at = (a - lo) // 2 % ldt  # where u's rows begin between t's
    return ldt != ldu or (a - lo) % 2 != 0 or at < t.shape[1] or at + u.shape[1] > ldt


def _rows_of(t, M, N, dev, call, name):
    """Row stride of an fp16 [M, N] tensor on dev with unit inner stride and rows that do not overlap."""
    if t.dtype is torch.float16 and t.device == dev and t.shape == (M, N):
        ld, one = t.stride()
        if (one == 1 or N == 1) and (ld >= N or M == 1):
            return max(ld, N)
    raise ValueError(f"{call}: {name} must be fp16 [{M}, {N}] on {dev} with unit inner stride")


def mm_q4(x, w, res=None, nw=None, eps=1e-5, out=None):
    """y = x @ w^T (+ res) -> [M, N] for 4-bit weights ``w`` (pack_q4) and x [M, K] fp16, or with ``nw`` [K] the RMS norm of
    x's rows: scales, sums, the norm's statistics and the residual in fp32, one rounding at the end (of products of more than 16
    rows those that go by matrix tiles, most of them, round the normed rows to fp16 before: 2.9e-4 of the result for 2.1e-4).
    Any number of rows.
    ``out`` may be ``res``, or apart from it, and not x (columns of the same rows that do not meet are apart)."""
    return _mm_q4("mm_q4", x, w, w.N, res, nw, eps, out, False)


def mm_q4_silu(x, w, nw=None, eps=1e-5, out=None):
    """silu(a) * b -> [M, N / 2] for the products a, b of mm_q4 on interleaved w1 | w3 (pack_q4(..., interleave=True)), in fp32
    with one rounding at the end (normed rows count in two fp16 parts)."""
    return _mm_q4("mm_q4_silu", x, w, w.N // 2, None, nw, eps, out, True)


# ---------------------------------------------------------------- logits before the sampler
def _per_row(t, N, dev, name):
    """(address, whether there is an element per row) of a penalty."""
    if t.dtype is torch.float32 and t.device == dev and t.dim() == 1 and t.is_contiguous():
        n = t.numel()
        if n == N:
            return t.data_ptr(), N != 1
        if n == 1:
            return t.data_ptr(), False
    raise ValueError(f"process_logits: {name} must be float32 [{N}] or [1] on {dev}")


def pack_mask(keep):
    """bool [A, V] (or [V]) of allowed tokens -> the int32 [A, ceil(V / 32)] masks of process_logits, bit v % 32 of word
    v // 32.  Set-up work: elementary torch operations."""
    if keep.dtype is not torch.bool or keep.dim() not in (1, 2):
        raise TypeError("pack_mask: keep must be bool [A, V] or [V]")
    keep = keep if keep.dim() == 2 else keep[None]
    A, V = keep.shape
    bits = torch.zeros(A, -(-V // 32) * 32, device=keep.device, dtype=torch.int64)
    bits[:, :V] = keep
    w = (bits.view(A, -1, 32) << torch.arange(32, device=keep.device)).sum(2)
    return torch.where(w < 1 << 31, w, w - (1 << 32)).to(torch.int32)


def process_logits(logits, hist=None, length=None, window=0, repetition=None, presence=None, frequency=None, bias=None,
                   allowed=None, state=None, cfg=None, out=None):
    """Logits [B, V] fp16 -> those that sample_topk draws from [N, V], in fp32 with one rounding to fp16:

    guidance (``cfg`` given: B = 2N, cond rows then uncond rows): l = uncond + (cond - uncond) cfg; else N = B;
    a token that occurs n > 0 times in the row's history: l / ``repetition`` if l > 0, else l * ``repetition``; then
    l - (``presence`` + ``frequency`` * n) (each float32 [N] or [1], read on the device);
    l + ``bias`` (float32 [V], or [N, V]);
    -inf for tokens that the row's mask does not allow, whatever their logits hold (a row that may draw nothing is all -inf).
    A finite result above fp16's range is 65504, its largest number (several such tokens are then equally likely); one below
    it is -inf.

    ``hist`` int64 [N, T] with any strides: the row's tokens, of which the first ``length`` (int64 [N] on the device; None: T)
    are there and the last ``window`` of those count (0: all); tokens outside [0, V) count for nothing.  ``allowed`` int32
    [A, ceil(V / 32)]: masks of allowed tokens, bit v % 32 of word v // 32; ``state`` int32 [N] gives each row its mask (-1:
    none; any other number outside [0, A): nothing is allowed), without it A is 1 or N.  ``out``: the destination; it may be
    the first N rows of ``logits``."""
    dev = logits.device
    if logits.dtype is not torch.float16 or not logits.is_cuda:
        _dev(logits, "process_logits")
        _f16(logits, "process_logits logits")
    if logits.dim() != 2:
        raise ValueError("process_logits: logits must be [B, V]")
    (B, V), (ld, one) = logits.shape, logits.stride()
    guided = cfg is not None
    N = B // 2 if guided else B
    if (one != 1 and V != 1) or (ld < V and B != 1) or not 1 <= V <= INT_MOST - 8192 or (guided and B % 2):
        raise ValueError("process_logits: logits must be [B, V] with contiguous rows (B even with cfg)")
    hp = lp = rp = pp = fp = bp = ap = sp = None
    hrow = htok = T = ldb = lda = A = flags = 0
    if hist is not None:
        if hist.dtype is not torch.int64 or hist.device != dev or hist.dim() != 2:
            raise ValueError(f"process_logits: hist must be int64 [{N}, T] on {dev}")
        (rows, T), (hrow, htok) = hist.shape, hist.stride()
        if rows != N or T > INT_MOST:
            raise ValueError(f"process_logits: hist must be int64 [{N}, T] on {dev}")
        if length is not None:
            _on(length, dev, "process_logits", "length", torch.int64, (N,))
            lp = length.data_ptr()
        if not 0 <= window <= INT_MOST:
            raise ValueError("process_logits: window must be 0 (all tokens) or a number of tokens")
        if repetition is not None:
            rp, flags = _per_row(repetition, N, dev, "repetition")
        if presence is not None:
            pp, f = _per_row(presence, N, dev, "presence")
            flags |= f << 1
        if frequency is not None:
            fp, f = _per_row(frequency, N, dev, "frequency")
            flags |= f << 2
        if T and (rp or pp or fp):
            hp = hist.data_ptr()
        else:  # nothing to count, or nothing that depends on it
            rp = pp = fp = None
    elif length is not None or window or repetition is not None or presence is not None or frequency is not None:
        raise ValueError("process_logits: penalties need a history (hist)")
    if bias is not None:
        shape, step = bias.shape, bias.stride()
        if len(shape) == 2:
            ldb = step[0] if N > 1 else V
        if bias.dtype is not torch.float32 or bias.device != dev or shape not in ((V,), (N, V)) or \
                (step[-1] != 1 and V != 1) or (len(shape) == 2 and ldb < V):
            raise ValueError(f"process_logits: bias must be float32 [{V}] or [{N}, {V}] on {dev} with contiguous rows")
        bp = bias.data_ptr()
    if allowed is not None:
        lda = -(-V // 32)
        A = allowed.shape[0] if allowed.dim() == 2 else 0
        if not 1 <= A <= INT_MOST or (state is None and A != 1 and A != N):
            raise ValueError(f"process_logits: allowed must be [A, {lda}] (A 1 or {N} without state)")
        _on(allowed, dev, "process_logits", "allowed", torch.int32, (A, lda))
        ap = allowed.data_ptr()
        if state is not None:
            _on(state, dev, "process_logits", "state", torch.int32, (N,))
            sp = state.data_ptr()
    elif state is not None:
        raise ValueError("process_logits: state needs masks (allowed)")
    if out is None:  # rows start aligned for the sampler
        ldo = -(-V // 64) * 64
        out = torch.empty_strided((N, V), (ldo, 1), device=dev, dtype=torch.float16)
    else:
        ldo = _rows_of(out, N, V, dev, "process_logits", "out")
        if _meet(out, ldo, logits, ld) and not (out.data_ptr() == logits.data_ptr() and (ldo == ld or N == 1)):
            raise ValueError("process_logits: out must be apart from logits or their first rows")
    if N:
        _call_on(dev, "ecd_process_logits", logits.data_ptr(), max(ld, V), guided, cfg if guided else 1.0, hp, hrow, htok, T, lp,
                 window, rp, pp, fp, flags, bp, ldb, ap, lda, A, sp, out.data_ptr(), ldo, N, V)
    return out
