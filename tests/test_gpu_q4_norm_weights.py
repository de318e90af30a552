"""Products with a norm whose weights go up to fp16's largest numbers, over rows with quiet parts, against float64."""
import numpy as np
import pytest

from helpers import randn16, rng
from test_gpu_q4 import H, _t, make, norm64, packed

pytestmark = pytest.mark.gpu


def inputs(seed, M, K):
    """Rows and weights of a norm with x' that fits fp16: weights over the range of fp16, channels the quieter the larger their weight,
    and rows of which a part holds a single small value under a large weight."""
    g = rng(seed)
    nw = np.exp(g.uniform(np.log(1e-3), np.log(6e4), K)) * np.where(g.random(K) < 0.5, -1, 1)
    x = g.standard_normal((M, K)) * np.minimum(1.0, 30 / np.abs(nw))
    part = max(32, K // 8)
    for r in range(0, M, 2):
        x[r, :part] = 0
        x[r, g.integers(0, part)] = 0.0156
    nw[:part] = np.sign(nw[:part]) * np.maximum(np.abs(nw[:part]), 4000)
    return x.astype(np.float16), nw.astype(np.float16)


def tolerance(x, nw, w, few, once):
    """For each output, what fp32 sums, x' in two fp16 parts (few) or rounded, and the norm's fp32 roundings can add up to.

    few: x times a power of two up to 2 / rms of a part, 256 channels at least, so of 2 sqrt(K / 256) / rms of the row back; a
    rounding among the subnormal numbers is 2^-25 at most: of x times its weight, of the weight in units of 2^-5 (65504 times the 20 that
    a part's largest value can be has to fit) times 20, and of the second part."""
    xn = np.abs(norm64(x, nw))
    K = x.shape[1]
    A = xn @ np.abs(w).T
    tol = (2.0 ** -23 * (64 + K // 64 + 32) + K / 16 * 1.25 * 2.0 ** -22 + 2.0 ** -21) * A
    if few:
        err = 2.0 ** -25 * np.abs(nw.astype(np.float64)) + 2.0 ** -25 * 2.0 ** 5 * 21
        return tol + 2 * np.sqrt(K / 256 + 1) * (np.abs(w) @ err)
    return tol + (H * A if once else 0) + 2.0 ** -25 * np.abs(w).sum(1)


def silu_of(y, t, F):
    a, b, ta, tb = y[:, :F], y[:, F:], t[:, :F], t[:, F:]
    f = a / (1 + np.exp(-a))
    return f * b, (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb


def check(got, want, tol):
    """Results are fp16: from 65520 on they are infinities, and either where the bound reaches across."""
    got = got.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25
    past = (got == np.copysign(np.inf, want)) & (np.abs(want) + tol >= 65520)
    bad = ~(near & (np.abs(want) - tol < 65520) | past)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, {np.isnan(got).sum()} no numbers, first at {np.argwhere(bad)[0]}"


def test_one_small_value_under_a_large_weight(dev):
    """x = 0.0156 under a weight of 4500 in an otherwise empty part of the row: x' = 75."""
    from estudiocanciones_amd.kernels import mm_q4
    N, K = 48, 3072
    q, s, z, w = make(1, N, K, 128, False)
    for M in (1, 4, 8, 16):
        x = np.ones((M, K), np.float16)
        x[0, :] = [0 if k // 128 % 8 == 0 else 1 for k in range(K)]
        x[0, 5] = 0.0156
        nw = np.ones(K, np.float16)
        nw[5] = 4500
        xn = norm64(x, nw)
        assert 70 < xn[0, 5] < 80
        check(mm_q4(_t(x, dev), packed(dev, q, s, z), nw=_t(nw, dev)), xn @ w.T, tolerance(x, nw, w, True, False))


@pytest.mark.parametrize("M", [1, 4, 8, 16, 40])
@pytest.mark.parametrize("K", [256, 1024, 3072, 8192])
@pytest.mark.parametrize("weight", [3400, 20000, 65504])
def test_quiet_parts_under_large_weights(dev, M, K, weight):
    """Row r is empty in every eighth 128 channels from 128 (r % 8) on (a wave's, or all those of a shorter row) but for 60 / weight under the large
    weight: by the calls and by each form of the few-row kernel."""
    import torch
    from estudiocanciones_amd import _ffi
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    N = 128
    q, s, z, w = make(K + M, N, K, 64, True)
    x = randn16(M + K, M, K)
    nw = (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    for r in range(M):
        part = np.arange(K) // 128 % 8 == r % max(1, min(8, K // 128))
        x[r, part] = 0
        k = np.flatnonzero(part)[5 + r]
        x[r, k] = 60 / weight
        nw[k] = -weight
    other = np.abs(nw) > 3000  # (of other rows: small there)
    for r in range(M):
        x[r, other] = np.where(np.abs(x[r, other]) > 100 / weight, x[r, other] * np.float16(20 / weight), x[r, other])
    xn = norm64(x, nw)
    assert np.abs(xn).max() < 2000
    few, once, both = (tolerance(x, nw, w, *a) for a in ((True, False), (False, True), (False, False)))
    xt, nt, wp, wi = _t(x, dev), _t(nw, dev), packed(dev, q, s, z), packed(dev, q, s, z, True)
    check(mm_q4(xt, wp, nw=nt), xn @ w.T, few if M <= 16 else few + once)
    check(mm_q4_silu(xt, wi, nw=nt), *silu_of(xn @ w.T, few if M <= 16 else few + both, N // 2))
    for form in (1, 2, 3):
        y = torch.full((M, N), 7.0, device=dev, dtype=torch.float16)
        _ffi.call("ecd_mm_q4", xt.data_ptr(), K, nt.data_ptr(), 1e-5, wp.codes_ptr, wp.scales_ptr, True, 64, None, 0, y.data_ptr(),
                  N, M, N, K, False, 32 + 16 + form + 256, None, torch.cuda.current_stream().cuda_stream)
        check(y, xn @ w.T, few)


@pytest.mark.parametrize("M", [1, 4, 8, 16, 40])
@pytest.mark.parametrize("N,K,group,zeros", [(70, 64, 64, False), (50, 1088, 32, True), (512, 3072, 128, False), (1024, 3072, 64, True),
                                             (96, 8192, 128, True)])
def test_weights_over_the_range_of_fp16(dev, M, N, K, group, zeros):
    import torch
    from estudiocanciones_amd import _ffi
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    q, s, z, w = make(M + N + K, N, K, group, zeros)
    x, nw = inputs(M + K, M, K)
    assert np.abs(norm64(x, nw)).max() < 65504
    xt, nt, F = _t(x, dev), _t(nw, dev), N // 2
    wp, wi = packed(dev, q, s, z), packed(dev, q, s, z, True)
    xn = norm64(x, nw)
    few, rounded = tolerance(x, nw, w, True, False), tolerance(x, nw, w, False, True)
    check(mm_q4(xt, wp, nw=nt), xn @ w.T, few if M <= 16 else few + rounded)
    check(mm_q4_silu(xt, wi, nw=nt), *silu_of(xn @ w.T, few if M <= 16 else few + tolerance(x, nw, w, False, False), F))
    for form in (1, 2, 3) if M > 16 else ():
        y = torch.full((M, N), 7.0, device=dev, dtype=torch.float16)
        _ffi.call("ecd_mm_q4", xt.data_ptr(), K, nt.data_ptr(), 1e-5, wp.codes_ptr, wp.scales_ptr, zeros, group, None, 0, y.data_ptr(),
                  N, M, N, K, False, 32 + 16 + form + 256, None, torch.cuda.current_stream().cuda_stream)
        check(y, xn @ w.T, few)


@pytest.mark.parametrize("M", [1, 8, 16])
def test_ordinary_weights_beside_a_large_one(dev, M):
    """One weight of 65504 over a channel that is nearly empty: the others' products keep their precision (one rounding, H / sqrt(3)
    of the result in the mean, and little beside it)."""
    from estudiocanciones_amd.kernels import mm_q4
    N, K = 2048, 1024
    q, s, z, w = make(M, N, K, 128, True)
    x = randn16(M, M, K)
    nw = (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    nw[77] = 65504
    x[:, 77] *= np.float16(2.0 ** -17)
    want = norm64(x, nw) @ w.T
    got = mm_q4(_t(x, dev), packed(dev, q, s, z), nw=_t(nw, dev))
    check(got, want, tolerance(x, nw, w, True, False))
    assert np.sqrt(((got.double().cpu().numpy() - want) ** 2).mean()) <= 0.7 * H * np.sqrt((want ** 2).mean())
