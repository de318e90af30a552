"""4-bit weights: q4_rows, pack_q4, mm_q4 and mm_q4_silu against float64."""
import numpy as np
import pytest

from helpers import randn16, rng

pytestmark = pytest.mark.gpu

H = 2.0 ** -11  # half a step of fp16, relative


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def make(seed, N, K, group, zeros):
    """Random codes, scales and zero points, and the float64 matrix that they stand for."""
    g = rng(seed)
    ng = -(-K // group)
    u = g.integers(0, 16, (N, K)).astype(np.uint8)
    s = (0.004 * (0.5 + g.random((N, ng)))).astype(np.float16)
    z = g.integers(0, 16, (N, ng)).astype(np.uint8) if zeros else None
    zz = 8.0 if z is None else np.repeat(z, group, 1)[:, :K].astype(np.float64)
    w = (u.astype(np.float64) - zz) * np.repeat(s.astype(np.float64), group, 1)[:, :K]
    return u[:, 0::2] | (u[:, 1::2] << 4), s, z, w


def packed(dev, q, s, z, interleave=False):
    from estudiocanciones_amd.kernels import pack_q4
    return pack_q4(_t(q, dev), _t(s, dev), None if z is None else _t(z, dev), interleave)


def norm64(x, nw, eps=1e-5):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * nw.astype(np.float64)


def sums_tol(x, w, norm):
    """What fp32 sums and the roundings of operands can add up to, for each output.

    Sums: products of an fp16 and a code are exact in fp32; a sum passes at most 64 additions within a chunk of k and one for
    each chunk and partial sum, of an error of at most 2^-23 (a truncating adder) times the sum of magnitudes A.  Operands:
    one rounding of the weights to fp16 (many rows) and, with a norm, two of x' (H each, times A)."""
    A = np.abs(x) @ np.abs(w).T
    return (2.0 ** -23 * (64 + x.shape[1] // 64 + 32) + H * (3 if norm else 1)) * A


def check(got, want, tol, what="", floor=0.0):
    got = got.double().cpu().numpy()
    err = np.abs(got - want)
    bad = ~(err <= tol + H * (np.abs(want) + tol) + 2.0 ** -25)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(err)} at {np.argwhere(bad)[0]}"
    if want.size >= 2000:
        # at most four independent roundings of H / sqrt(3) each on the average value; among the subnormal numbers a rounding is
        # 2^-25 at most whatever the value (the output's here, the operands' in `floor`)
        rms = np.sqrt((err ** 2).mean())
        assert rms <= 1.25 * H * np.sqrt((want ** 2).mean()) + 2.0 ** -25 + floor, f"{what}: rms {rms}"


# ---------------------------------------------------------------- the quantiser
def _round_even(x):
    return np.rint(x)


def quant64(w, group, zeros):
    """The definition, with exact quotients (float64 of fp32 or narrower values: no tie is made or lost)."""
    N, K = w.shape
    ng = -(-K // group)
    pad = np.zeros((N, ng * group))
    pad[:, :K] = w
    p = pad.reshape(N, ng, group)
    if zeros:
        lo, hi = np.minimum(p.min(2), 0), np.maximum(p.max(2), 0)
        s = ((hi.astype(np.float32) - lo.astype(np.float32)) / np.float32(15)).astype(np.float16)
    else:
        s = (np.abs(p).max(2).astype(np.float32) / np.float32(7)).astype(np.float16)
    sd = s.astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        z = np.where(sd > 0, np.clip(_round_even(-lo / sd), 0, 15), 0) if zeros else np.full((N, ng), 8)
        u = np.where(sd[..., None] > 0, _round_even(p / sd[..., None]) + z[..., None], z[..., None])
    u = np.clip(u, 0, 15).astype(np.uint8).reshape(N, -1)[:, :K]
    return u[:, 0::2] | (u[:, 1::2] << 4), s, z.astype(np.uint8)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K,group", [(1, 64, 64), (3, 64, 128), (5, 192, 128), (33, 192, 32), (7, 3072, 128), (1001, 320, 64)])
def test_quantiser_gives_the_nearest_codes(dev, dtype, zeros, N, K, group):
    import torch
    from estudiocanciones_amd.quant import q4_rows
    t = (torch.randn(N, K, generator=torch.Generator().manual_seed(N + K)) * 0.02).to(getattr(torch, dtype))
    t[0, :32] = torch.arange(32).to(t.dtype) * 0.5 - 8  # quotients that are ties
    t[-1, 32:64] = 0
    t[N // 2] *= 2.0 ** -12  # scales in the subnormal numbers
    q, s, z = q4_rows(t.to(dev), group, zeros)
    wq, ws, wz = quant64(t.double().numpy(), group, zeros)
    assert np.array_equal(s.cpu().numpy().view(np.uint16), ws.view(np.uint16))
    assert np.array_equal(q.cpu().numpy(), wq)
    assert z is None if not zeros else np.array_equal(z.cpu().numpy(), wz)


def test_quantiser_ties(dev):
    """Every half step of scale 2^-4 on both sides of 0: ties to the even integer."""
    import torch
    from estudiocanciones_amd.quant import q4_rows
    t = torch.zeros(1, 64)
    t[0, :29] = (torch.arange(29) - 14) / 32.0  # -7 .. 7 by halves of the scale 1 / 16
    q, s, _ = q4_rows(t.to(dev), 64)
    assert s.item() == 1 / 16
    assert np.array_equal(q.cpu().numpy(), quant64(t.double().numpy(), 64, False)[0])


def test_quantiser_rows_of_zeros_and_no_numbers(dev):
    import torch
    from estudiocanciones_amd.quant import q4_rows
    t = torch.randn(6, 128, generator=torch.Generator().manual_seed(1))
    t[0] = 0
    t[1, 5] = float("inf")
    t[2, 70] = float("nan")
    t[3, 9] = -3e6  # a scale past fp16
    for zeros in (False, True):
        q, s, z = q4_rows(t.to(dev), 64, zeros)
        s = s.cpu().numpy()
        assert (s[0] == 0).all() and np.isnan(s[1, 0]) and np.isnan(s[2, 1]) and np.isnan(s[3, 0])
        assert np.isfinite(s[[1, 2, 3], [1, 0, 1]]).all() and np.isfinite(s[4:]).all()
        if not zeros:
            assert (q[0].cpu().numpy() == 0x88).all()


def test_quantiser_takes_views(dev):
    """Rows of a wider tensor, and a view whose start is not aligned."""
    import torch
    from estudiocanciones_amd.quant import q4_rows
    big = torch.randn(9, 200, generator=torch.Generator().manual_seed(2)).to(dev)
    flat = torch.randn(3 * 64 + 1, generator=torch.Generator().manual_seed(3)).to(dev)[1:].view(3, 64)
    for t in (big[:, 3:131], flat):
        q, s, _ = q4_rows(t, 32)
        wq, ws, _ = quant64(t.double().cpu().numpy(), 32, False)
        assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)


# ---------------------------------------------------------------- products
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [5, 13, 40, 192])
def test_single_weights_come_out_exactly(dev, M, group, zeros):
    """Rows that hold one 1 give single weights s (u - z), rounded to fp16 once: the nearest fp16, or with many rows its other
    neighbour where the weight (of 16 bits) lies so near the middle that the quotients of scales (K / 32 at most, each off by
    2^-22 with its reciprocal, and a product each) pass it."""
    from estudiocanciones_amd.kernels import mm_q4
    N, K = 75, 192
    q, s, z, w = make(M + group, N, K, group, zeros)
    wp = packed(dev, q, s, z)
    for k0 in range(0, K, M):
        x = np.zeros((M, K), np.float16)
        ks = np.arange(k0, min(k0 + M, K))
        x[np.arange(len(ks)), ks] = 1
        y = mm_q4(_t(x, dev), wp).cpu().numpy()
        want = np.zeros((M, N))
        want[:len(ks)] = w[:, ks].T
        if M <= 16:
            assert np.array_equal(y, want.astype(np.float16))
        else:
            # half a step at the magnitude of the weight (2^-11 of its power of two), widened by the quotients' 6 (2^-22 + 2^-24)
            step = 2.0 ** np.floor(np.log2(np.maximum(np.abs(want), 2.0 ** -14))) * H
            assert (np.abs(y.astype(np.float64) - want) <= step + 2.0 ** -19 * np.abs(want)).all()


SHAPES = [(1, 1, 64), (1, 33, 64), (2, 1001, 192), (7, 31, 320), (8, 512, 1024), (9, 77, 8192), (16, 1024, 448), (17, 40, 64),
          (31, 96, 1024), (32, 250, 192), (33, 64, 2048), (48, 3072, 128), (64, 65, 320), (65, 130, 1024), (100, 1001, 192),
          (128, 256, 512), (129, 70, 8192), (187, 512, 1024), (257, 1032, 320), (300, 3, 64), (512, 384, 192)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, True), (128, False), (128, True)])
def test_products(dev, M, N, K, group, zeros):
    from estudiocanciones_amd.kernels import mm_q4
    q, s, z, w = make(M + N + K, N, K, group, zeros)
    x, res = randn16(M, M, K), randn16(M + 1, M, N)
    wp = packed(dev, q, s, z)
    x64 = x.astype(np.float64)
    tol = sums_tol(x64, w, False)
    check(mm_q4(_t(x, dev), wp), x64 @ w.T, tol, "plain")
    check(mm_q4(_t(x, dev), wp, res=_t(res, dev)), x64 @ w.T + res, tol, "residual")
    nw = (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    xn = norm64(x * np.float16(3), nw)
    check(mm_q4(_t(x * np.float16(3), dev), wp, nw=_t(nw, dev)), xn @ w.T, sums_tol(xn, w, True), "norm")


@pytest.mark.parametrize("tile", range(1, 7))
@pytest.mark.parametrize("M,N,K,ks", [(5, 40, 64, 1), (37, 300, 320, 1), (37, 300, 320, 3), (150, 129, 1088, 1), (150, 129, 1088, 5),
                                      (300, 520, 192, 2), (8, 64, 832, 13)])
@pytest.mark.parametrize("group,zeros,silu", [(32, True, False), (64, False, True), (128, True, True), (128, False, False)])
def test_every_tile(dev, tile, M, N, K, ks, group, zeros, silu):
    """The kernels of many rows that the sizes' own plan need not choose: K of an odd number of chunks, split in uneven parts."""
    import torch
    from estudiocanciones_amd import _ffi
    q, s, z, w = make(M + N + K, N, K, group, zeros)
    wp = packed(dev, q, s, z, silu and N % 2 == 0)
    silu = wp.interleave
    x, nw = randn16(M, M, K), (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    cols = N // 2 if silu else N
    xt, nt, st = _t(x, dev), _t(nw, dev), torch.cuda.current_stream().cuda_stream
    plan = tile + 256 * ks
    ws = torch.full((_ffi.lib().ecd_mm_q4_ws_bytes(M, N, K, plan, 1) // 4,), float("nan"), device=dev)
    for norm in (False, True):
        y = torch.full((M + 1, cols), 7.0, device=dev, dtype=torch.float16)
        _ffi.call("ecd_mm_q4", xt.data_ptr(), K, nt.data_ptr() if norm else None, 1e-5, wp.codes_ptr, wp.scales_ptr, zeros, group,
                  None, 0, y.data_ptr(), cols, M, N, K, silu, plan, ws.data_ptr(), st)
        xn = norm64(x, nw) if norm else x.astype(np.float64)
        want, tol = xn @ w.T, sums_tol(xn, w, norm)
        if silu:
            a, b, ta, tb = want[:, :cols], want[:, cols:], tol[:, :cols], tol[:, cols:]
            f = a / (1 + np.exp(-a))
            want, tol = f * b, (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb
        got = y[:M].double().cpu().numpy()
        bad = ~(np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25)
        assert not bad.any(), (norm, bad.sum(), np.argwhere(bad)[0])
        assert (y[M] == 7.0).all()


@pytest.mark.parametrize("form", [1, 2, 3])
@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (4, 129, 192), (17, 300, 320), (40, 66, 1088), (150, 129, 2176), (33, 520, 128)])
@pytest.mark.parametrize("group,zeros,silu", [(32, True, False), (32, False, True), (64, True, True), (64, False, False),
                                              (128, True, True), (128, False, False)])
def test_few_rows_at_a_time(dev, form, M, N, K, group, zeros, silu):
    """The few-row kernel over blocks of rows, 16, 32 or 64 features a workgroup, with residual, norm and SiLU, into rows of a
    larger matrix: the same values as without a plan, of which it changes nothing else."""
    import torch
    from estudiocanciones_amd import _ffi
    q, s, z, w = make(M + N + K, N, K, group, zeros)
    wp = packed(dev, q, s, z, silu and N % 2 == 0)
    silu = wp.interleave
    x, nw = randn16(M, M, K), (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    cols = N // 2 if silu else N
    res = None if silu else randn16(M + 1, M, cols)
    xt, nt, rt, st = _t(x, dev), _t(nw, dev), None if silu else _t(res, dev), torch.cuda.current_stream().cuda_stream
    ws = torch.full((M * K,), float("nan"), device=dev, dtype=torch.float16)
    for norm in (False, True):
        y = torch.full((M + 1, cols + 8), 7.0, device=dev, dtype=torch.float16)
        _ffi.call("ecd_mm_q4", xt.data_ptr(), K, nt.data_ptr() if norm else None, 1e-5, wp.codes_ptr, wp.scales_ptr, zeros, group,
                  None if silu else rt.data_ptr(), cols, y.data_ptr(), cols + 8, M, N, K, silu, 16 + form + 256,
                  ws.data_ptr() if norm else None, st)
        xn = norm64(x, nw) if norm else x.astype(np.float64)
        want, tol = xn @ w.T, sums_tol(xn, w, norm)
        if silu:
            a, b, ta, tb = want[:, :cols], want[:, cols:], tol[:, :cols], tol[:, cols:]
            f = a / (1 + np.exp(-a))
            want, tol = f * b, (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb
        else:
            want = want + res
        got = y[:M, :cols].double().cpu().numpy()
        bad = ~(np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25)
        assert not bad.any(), (norm, bad.sum(), np.argwhere(bad)[0])
        assert (y[M] == 7.0).all() and (y[:, cols:] == 7.0).all()


@pytest.mark.parametrize("plan", [1, 2 + 256, 3 + 512, 4, 5 + 512, 6 + 256, 17, 18, 19])
@pytest.mark.parametrize("M,F,K", [(5, 20, 192), (37, 150, 320), (150, 65, 1088), (300, 260, 256)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
def test_norm_in_two_parts(dev, plan, M, F, K, group, zeros):
    """The norm before a SiLU in two fp16 parts, by the tiles (K whole and split, of odd and even numbers of chunks) and by the
    few-row kernel: x' counts with 2^-22 of its value (what is left of the second part, 2^-25 of it where that is subnormal) and
    the fp32 roundings of the norm (four of 2^-24), not with half a step of fp16."""
    import torch
    from estudiocanciones_amd import _ffi
    tile, ks = plan & 255, 1 + (plan >> 8)
    q, s, z, w = make(M + F + K, 2 * F, K, group, zeros)
    wp = packed(dev, q, s, z, True)
    x, nw = randn16(M, M, K), (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16)
    xt, nt, st = _t(x, dev), _t(nw, dev), torch.cuda.current_stream().cuda_stream
    plan = 32 + tile + 256 * ks
    nb = _ffi.lib().ecd_mm_q4_ws_bytes(M, 2 * F, K, plan, 1)
    assert nb == (0 if tile > 6 else 4 * M * K + (ks * M * (-(-2 * F // 8) * 8) * 4 if ks > 1 else 0))
    ws = torch.full((nb // 4 + 64,), float("nan"), device=dev)
    y = torch.full((M + 1, F), 7.0, device=dev, dtype=torch.float16)
    _ffi.call("ecd_mm_q4", xt.data_ptr(), K, nt.data_ptr(), 1e-5, wp.codes_ptr, wp.scales_ptr, zeros, group, None, 0,
              y.data_ptr(), F, M, 2 * F, K, True, plan, ws.data_ptr(), st)
    xn = norm64(x, nw)
    A = np.abs(xn) @ np.abs(w).T
    want = xn @ w.T
    # sums as in sums_tol (twice the additions), the quotients of scales (K / 16 at most, 2^-22 + 2^-24 each), and x'
    tol = (2.0 ** -23 * (2 * 64 + 2 * K // 64 + 32) + K / 16 * 1.25 * 2.0 ** -22 + 2.0 ** -22 + 2.0 ** -22) * A
    tol += 2.0 ** -25 * np.abs(w).sum(1)
    a, b, ta, tb = want[:, :F], want[:, F:], tol[:, :F], tol[:, F:]
    f = a / (1 + np.exp(-a))
    want, tol = f * b, (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb
    got = y[:M].double().cpu().numpy()
    err = np.abs(got - want)
    bad = ~(err <= tol + H * (np.abs(want) + tol) + 2.0 ** -25)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[0])
    assert (y[M] == 7.0).all() and torch.isnan(ws[nb // 4:]).all()
    if want.size >= 2000:  # one rounding, of H / sqrt(3) at most in the mean (an x' rounded once adds as much twice)
        assert np.sqrt((err ** 2).mean()) <= 0.6 * H * np.sqrt((want ** 2).mean()) + 2.0 ** -25


@pytest.mark.parametrize("M,F,K", [(1, 1, 64), (1, 4099, 192), (3, 17, 192), (8, 512, 1024), (16, 40, 320), (30, 33, 64), (33, 500, 192),
                                   (64, 64, 128), (70, 65, 1024), (187, 1001, 320), (300, 256, 512)])
@pytest.mark.parametrize("group,zeros,norm", [(32, True, True), (64, False, False), (128, False, True), (128, True, False)])
def test_silu(dev, M, F, K, group, zeros, norm):
    from estudiocanciones_amd.kernels import mm_q4_silu
    q, s, z, w = make(M + F + K, 2 * F, K, group, zeros)
    x = randn16(M, M, K, std=2.0)
    nw = (1 + 0.1 * rng(K).standard_normal(K)).astype(np.float16) if norm else None
    xn = norm64(x, nw) if norm else x.astype(np.float64)
    y = xn @ w.T
    t = sums_tol(xn, w, norm) + 2.0 ** -22 * np.abs(y)
    a, b, ta, tb = y[:, :F], y[:, F:], t[:, :F], t[:, F:]
    if M > 64:  # (many rows: a and b may be rounded to fp16 before the SiLU)
        ta, tb = ta + H * np.abs(a) + 2.0 ** -25, tb + H * np.abs(b) + 2.0 ** -25
    f = a / (1 + np.exp(-a))
    # |silu'| <= 1.1; the exponential's and the quotient's few fp32 roundings relative to silu(a)
    tol = (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb
    if M > 64:
        tol += H * np.abs(f) * np.abs(b)
    got = mm_q4_silu(_t(x, dev), packed(dev, q, s, z, True), nw=None if nw is None else _t(nw, dev)).double().cpu().numpy()
    bad = ~(np.abs(got - f * b) <= tol + H * (np.abs(f * b) + tol) + 2.0 ** -25)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[0])


@pytest.mark.parametrize("M", [1, 8, 20, 50, 200])
def test_strided_rows_and_results_in_place(dev, M):
    """x, res and out as parts of wider tensors (out rows of any alignment), res as out; what lies beside out stays."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4
    N, K = 203, 320
    q, s, z, w = make(M, N, K, 64, True)
    wp = packed(dev, q, s, z)
    xw = _t(randn16(M, M + 2, K + 40), dev)
    x = xw[1:M + 1, 8:8 + K]
    wide = _t(randn16(M + 1, M + 3, N + 9), dev)
    before = wide.clone()
    out = wide[1:M + 1, 3:3 + N]
    res = out.clone()
    x64 = x.double().cpu().numpy()
    want = x64 @ w.T + res.double().cpu().numpy()
    same = mm_q4(x, wp, res=res)
    mm_q4(x, wp, res=out, out=out)
    check(out, want, sums_tol(x64, w, False))
    assert torch.equal(out, same)
    before[1:M + 1, 3:3 + N] = out
    assert torch.equal(before, wide)


@pytest.mark.parametrize("M", [2, 9, 40, 130])
def test_rows_do_not_mix(dev, M):
    """NaN and infinite rows leave the others' bits alone; so does garbage in rows of x that the call does not have."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4
    q, s, z, w = make(M, 100, 256, 128, False)
    wp = packed(dev, q, s, z)
    x = _t(randn16(M, M + 1, 256), dev)
    x[M] = float("nan")
    nw = torch.ones(256, device=dev, dtype=torch.float16)
    for kw in ({}, {"nw": nw}):
        clean = mm_q4(x[:M], wp, **kw)
        assert torch.isfinite(clean).all()
        y = x.clone()
        y[0, 3] = float("nan")
        y[1, 7] = float("inf")
        dirty = mm_q4(y[:M], wp, **kw)
        assert not torch.isfinite(dirty[:2]).any()
        assert torch.equal(dirty[2:], clean[2:])


@pytest.mark.parametrize("M", [3, 20, 100])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -24, 1e-3, 1.0, 2e4])
def test_norm_over_the_range_of_fp16(dev, M, scale):
    from estudiocanciones_amd.kernels import mm_q4
    q, s, z, w = make(M, 96, 512, 64, True)
    x = np.clip(np.round(randn16(M, M, 512).astype(np.float32) * 4) * (scale / 4 if scale > 1e-6 else scale), -65504, 65504).astype(np.float16)
    nw = (1 + 0.1 * rng(M).standard_normal(512)).astype(np.float16)
    xn = norm64(x, nw, 1e-5)
    # operands among the subnormal numbers: two roundings of 2^-25 (or one, times a factor below 2) for each
    tol = sums_tol(xn, w, True) + 2.0 ** -24 * np.abs(w).sum(1)
    check(mm_q4(_t(x, dev), packed(dev, q, s, z), nw=_t(nw, dev)), xn @ w.T, tol, floor=2.0 ** -24 * np.sqrt((w * w).sum(1).max()))


@pytest.mark.parametrize("M", [1, 8, 40, 190])
def test_graph_replays_and_streams(dev, M):
    """A captured call follows its inputs over replays with eager work between; calls on two streams do not disturb each other."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    q, s, z, w = make(M, 512, 2048, 128, False)
    wp, wi = packed(dev, q, s, z), packed(dev, q, s, z, True)
    nw = torch.ones(2048, device=dev, dtype=torch.float16)
    xs = [_t(randn16(i, M, 2048), dev) for i in range(4)]
    eager = [(mm_q4(x, wp, nw=nw), mm_q4_silu(x, wi)) for x in xs]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mm_q4(x, wp, nw=nw), mm_q4_silu(x, wi)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = mm_q4(x, wp, nw=nw), mm_q4_silu(x, wi)
    for i in (1, 2, 3, 0, 2):
        x.copy_(xs[i])
        g.replay()
        mm_q4(xs[(i + 1) % 4], wp)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(a, eager[i][0]) and torch.equal(b, eager[i][1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for r in range(8):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(mm_q4(xs[(r + k) % 4], wp, nw=nw))
    torch.cuda.synchronize()
    for k in range(2):
        for r in range(8):
            assert torch.equal(got[k][r], eager[(r + k) % 4][0])


def test_no_rows(dev):
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    q, s, z, _ = make(0, 64, 64, 64, False)
    x = torch.empty(0, 64, device=dev, dtype=torch.float16)
    assert mm_q4(x, packed(dev, q, s, z)).shape == (0, 64)
    assert mm_q4_silu(x, packed(dev, q, s, z, True)).shape == (0, 32)


def test_refusals(dev):
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu, pack_q4
    from estudiocanciones_amd.quant import q4_rows
    q, s, z, _ = make(0, 64, 128, 64, True)
    q, s, z = _t(q, dev), _t(s, dev), _t(z, dev)
    w, wi = pack_q4(q, s, z), pack_q4(q, s, z, True)
    x = torch.zeros(4, 128, device=dev, dtype=torch.float16)
    e = torch.empty
    f16 = dict(device=dev, dtype=torch.float16)
    for err, call in [
        (TypeError, lambda: mm_q4(x.float(), w)),
        (ValueError, lambda: mm_q4(x[:, :64], w)),                      # another K
        (ValueError, lambda: mm_q4(e(4, 132, **f16)[:, 4:], w)),        # rows not 16-byte aligned
        (ValueError, lambda: mm_q4(x.t().contiguous().t(), w)),         # columns not contiguous
        (RuntimeError, lambda: mm_q4(x.cpu(), w)),
        (ValueError, lambda: mm_q4(x, wi)),
        (ValueError, lambda: mm_q4_silu(x, w)),
        (ValueError, lambda: mm_q4(x, w, res=e(4, 63, **f16))),
        (ValueError, lambda: mm_q4(x, w, res=e(4, 64, device=dev))),
        (ValueError, lambda: mm_q4(x, w, out=e(5, 64, **f16))),
        (ValueError, lambda: mm_q4(x, w, out=e(64, 4, **f16).t())),
        (ValueError, lambda: mm_q4(x, w, res=e(4, 64, dtype=torch.float16))),  # on the CPU
        (ValueError, lambda: mm_q4(x, w, out=x[:, :64])),               # over its own input
        (TypeError, lambda: mm_q4(x, w, nw=e(128, device=dev))),
        (ValueError, lambda: mm_q4(x, w, nw=e(64, **f16))),
        (ValueError, lambda: mm_q4(x, w, nw=e(132, **f16)[4:])),        # not 16-byte aligned
        (ValueError, lambda: mm_q4(x, w, nw=e(128, **f16), eps=-1.0)),
        (ValueError, lambda: mm_q4(x, w, nw=e(128, **f16), eps=float("nan"))),
        (ValueError, lambda: pack_q4(q[:63], s[:63], z[:63], True)),    # an odd number of rows to interleave
        (ValueError, lambda: pack_q4(q, s[:, :1].repeat(1, 3))),        # three groups of 128
        (ValueError, lambda: pack_q4(q[:, :40], s)),                    # K = 80
        (TypeError, lambda: pack_q4(q.to(torch.int8), s)),
        (TypeError, lambda: pack_q4(q, s.float())),
        (TypeError, lambda: pack_q4(q, s, z.int())),
        (RuntimeError, lambda: pack_q4(q.cpu(), s.cpu())),
        (TypeError, lambda: q4_rows(torch.zeros(4, 64, device=dev, dtype=torch.float64))),
        (ValueError, lambda: q4_rows(torch.zeros(4, 96, device=dev))),
        (ValueError, lambda: q4_rows(torch.zeros(4, 64, device=dev), group=16)),
        (RuntimeError, lambda: q4_rows(torch.zeros(4, 64))),
    ]:
        with pytest.raises(err):
            call()


def test_out_and_res(dev):
    """The sum may take the residual's place, or lie apart from it (between its rows too where ranges do not meet); other overlaps
    are refused, as one thread would write what another has yet to read."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4
    for M in (1, 8, 40):
        N, K = 64, 128
        q, s, z, w = make(M, N, K, 64, False)
        wp = packed(dev, q, s, z)
        x, res = _t(randn16(M, M, K), dev), _t(randn16(M + 1, M + 2, N), dev)
        want = mm_q4(x, wp, res=res[:M])
        buf = res.clone()
        assert mm_q4(x, wp, res=buf[:M], out=buf[:M]).data_ptr() == buf.data_ptr() and torch.equal(buf[:M], want)
        assert torch.equal(buf[M:], res[M:])
        for a, b in ((slice(1, M + 1), slice(0, M)), (slice(0, M), slice(1, M + 1))):
            buf = res.clone()
            if M == 1:  # (rows next to each other)
                assert torch.equal(mm_q4(x, wp, res=buf[a], out=buf[b]), mm_q4(x, wp, res=res[a]))
                continue
            with pytest.raises(ValueError, match="res"):
                mm_q4(x, wp, res=buf[a], out=buf[b])
            assert torch.equal(buf, res)
        flat = torch.zeros((M + 1) * N, device=dev, dtype=torch.float16)
        with pytest.raises(ValueError, match="res"):
            mm_q4(x, wp, res=flat[:M * N].view(M, N), out=flat[8:8 + M * N].view(M, N))


def test_one_row_of_any_stride(dev):
    """A row's stride says nothing where there is one row, as of a transposed column."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    N, K = 70, 192
    q, s, z, w = make(3, N, K, 32, True)
    for il, f in ((False, mm_q4), (True, mm_q4_silu)):
        wp = packed(dev, q, s, z, il)
        x = _t(randn16(5, 1, K), dev)
        col = x.reshape(K, 1).clone().t()
        assert col.stride(0) == 1
        assert torch.equal(f(col, wp), f(x, wp)) and torch.equal(f(x.as_strided((1, K), (3, 1)), wp), f(x, wp))
        assert torch.equal(f(x.as_strided((1, K), (8, 1)), wp), f(x, wp))


@pytest.mark.parametrize("M", [12, 40, 700])
def test_two_graphs_of_the_same_weights(dev, M):
    """Two captured calls with a norm before a SiLU (with a workspace each, where many rows take one), replayed in turn, and an eager
    call between them."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4_silu
    q, s, z, w = make(M, 256, 1024, 64, True)
    wi = packed(dev, q, s, z, True)
    nw = _t((1 + 0.1 * rng(M).standard_normal(1024)).astype(np.float16), dev)
    xs = [_t(randn16(i, M, 1024), dev) for i in range(3)]
    want = [mm_q4_silu(x, wi, nw=nw) for x in xs]
    ins, graphs, outs = [xs[0].clone(), xs[0].clone()], [], []
    torch.cuda.synchronize()
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mm_q4_silu(x, wi, nw=nw))
        graphs.append(g)
    for i in range(6):
        for k in range(2):
            ins[k].copy_(xs[(i + k) % 3])
        graphs[0].replay()
        assert torch.equal(mm_q4_silu(xs[2], wi, nw=nw), want[2])
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[k], want[(i + k) % 3]) for k in range(2))

