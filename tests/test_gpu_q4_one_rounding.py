"""4-bit products by every kernel with one rounding: sums and scales in 32 bits, nothing rounded to fp16 on the way.

A result's error beside half a step of fp16 is that of fp32 sums (2^-23 for each addition at most, a truncating adder) and of the quotients of
scales (one for each K / 32 at most, 2^-22 + 2^-24 with its reciprocal and product), both of the sum of magnitudes.  A rounding's error is even
over a step d of the value, so d / sqrt(12) in the mean; over 2000 results and more the mean square is known to 2%, fp32 sums add 2% at most, and
an operand, a weight or a partial sum rounded to fp16 as well would add 60% and more."""
import numpy as np
import pytest

from helpers import randn16, rng
from test_gpu_q4 import H, _t, make, norm64, packed

pytestmark = pytest.mark.gpu


def bound(x, w):
    K = x.shape[1]
    return (2.0 ** -23 * (64 + K // 64 + 32) + K / 32 * 1.25 * 2.0 ** -22) * (np.abs(x) @ np.abs(w).T)


def silu_of(y, t):
    F = y.shape[1] // 2
    a, b, ta, tb = y[:, :F], y[:, F:], t[:, :F], t[:, F:]
    f = a / (1 + np.exp(-a))
    return f * b, (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb


def check(got, want, tol, what):
    err = np.abs(got.double().cpu().numpy() - want)
    bad = ~(err <= tol + H * (np.abs(want) + tol) + 2.0 ** -25)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}"
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(want), 2.0 ** -14))) - 10)
    assert want.size >= 2000 and (err ** 2).mean() <= 1.2 * (step ** 2).mean() / 12, what


@pytest.mark.parametrize("M,N,K", [(1, 4100, 1024), (8, 1000, 3072), (16, 400, 8192), (40, 300, 448), (64, 514, 3072), (187, 256, 8192),
                                   (600, 130, 1088)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_calls(dev, M, N, K, group, zeros):
    """The calls as they choose their kernels; a norm up to 16 rows and before a SiLU counts in two parts."""
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    q, s, z, w = make(M + N + K, N, K, group, zeros)
    x, res = randn16(M, M, K), randn16(M + 1, M, N)
    wp, wi, x64 = packed(dev, q, s, z), packed(dev, q, s, z, True), x.astype(np.float64)
    tol = bound(x64, w)
    check(mm_q4(_t(x, dev), wp), x64 @ w.T, tol, "product")
    check(mm_q4(_t(x, dev), wp, res=_t(res, dev)), x64 @ w.T + res, tol, "residual")
    check(mm_q4_silu(_t(x, dev), wi), *silu_of(x64 @ w.T, tol), "silu")
    nw = (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    xn = norm64(x, nw)
    # x' in two parts: 2^-22 of it and what of the second is subnormal, the norm's fp32 roundings 2^-22 (few rows: in units of up to
    # 2 sqrt(K / 256) of the row)
    tn = bound(xn, w) + 2.0 ** -21 * (np.abs(xn) @ np.abs(w).T) + 2.0 ** -25 * 2 * np.sqrt(K / 256 + 1) * np.abs(w).sum(1)
    if M <= 16:
        check(mm_q4(_t(x, dev), wp, nw=_t(nw, dev)), xn @ w.T, tn, "norm")
    check(mm_q4_silu(_t(x, dev), wi, nw=_t(nw, dev)), *silu_of(xn @ w.T, tn + bound(xn, w)), "norm and silu")


@pytest.mark.parametrize("plan", [1, 2 + 512, 3, 4 + 256, 5 + 512, 6, 17, 18, 19])
@pytest.mark.parametrize("M,N,K", [(40, 130, 320), (150, 258, 1088)])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False)])
@pytest.mark.parametrize("silu", [False, True])
def test_kernels(dev, plan, M, N, K, group, zeros, silu):
    import torch
    from estudiocanciones_amd import _ffi
    q, s, z, w = make(M + N + K, N, K, group, zeros)
    wp = packed(dev, q, s, z, silu)
    x = randn16(M, M, K)
    x64, cols, xt = x.astype(np.float64), N // 2 if silu else N, _t(x, dev)
    plan = (plan & 255) + 256 * (1 + (plan >> 8))
    ws = torch.full((_ffi.lib().ecd_mm_q4_ws_bytes(M, N, K, plan, 0) // 4 + 4,), float("nan"), device=dev)
    y = torch.full((M, cols), 7.0, device=dev, dtype=torch.float16)
    _ffi.call("ecd_mm_q4", xt.data_ptr(), K, None, 0.0, wp.codes_ptr, wp.scales_ptr, zeros, group, None, 0, y.data_ptr(), cols, M, N, K,
              silu, plan, ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    want, tol = x64 @ w.T, bound(x64, w)
    check(y, *(silu_of(want, tol) if silu else (want, tol)), "kernel")
