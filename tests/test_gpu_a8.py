"""int8 activations: quant_a8, gemm_a8_packed and gemm_a8_silu_packed against float64 and integer sums."""
import numpy as np
import pytest

from helpers import randn16, rng

pytestmark = pytest.mark.gpu


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _codes_np(y):
    """float64 rows -> (codes, scales) of the definition."""
    top = np.abs(y).max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        c = np.where(top > 0, np.rint(y * 127 / top), 0)
    return c, top[:, 0] / 127


@pytest.mark.parametrize("M,K", [(1, 64), (3, 192), (8, 3072), (5, 8192), (37, 1024), (2, 2112), (4, 64 * 300)])
def test_codes_are_the_nearest(dev, M, K):
    """Codes equal those of exact quotients; the scale within two fp32 roundings."""
    from estudiocanciones_amd.kernels import quant_a8
    x = randn16(M + K, M, K, std=3.0)
    x[0, ::7] = (np.arange(len(x[0, ::7])) % 33 - 16) / 2  # quotients that are ties
    x[0, 1] = 8
    x[-1, 3] = 60000  # one large value: most codes 0
    c, s = quant_a8(_t(x, dev))
    want, sw = _codes_np(x.astype(np.float64))
    assert np.array_equal(c.cpu().numpy(), want)
    assert (np.abs(s.cpu().numpy() - sw) <= 2.0 ** -23 * sw).all()
    pad = c.as_strided((M, c.stride(0)), (c.stride(0), 1))[:, K:]
    assert (pad == 0).all() and c.stride(0) % 128 == 0


def test_codes_of_every_value(dev):
    """Rows of all positive fp16 values up to a largest one, and their negatives: every code is the nearest integer."""
    from estudiocanciones_amd.kernels import quant_a8
    every = np.arange(0, 0x7C00, dtype=np.uint16).view(np.float16)
    tops = [1, 2, 3, 1023, 1024, 2047, 0x3C00, 0x3BFF, 0x3F80, 0x57F0, 0x57F1, 0x7BFF] + rng(1).integers(1, 0x7C00, 100).tolist()
    K = -(-len(every) // 64) * 64
    x = np.zeros((len(tops), K), np.float16)
    for r, t in enumerate(tops):
        x[r, :t + 1] = every[:t + 1] * np.float16(-1 if r % 2 else 1)
    c, _ = quant_a8(_t(x, dev))
    want, _ = _codes_np(x.astype(np.float64))
    assert np.array_equal(c.cpu().numpy(), want)


def test_rows_of_zeros_tiny_and_no_numbers(dev):
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, quant_a8
    x = randn16(1, 6, 128)
    x[0] = 0
    x[1] = 2.0 ** -24 * np.sign(x[1].astype(np.float32))  # the least subnormal
    x[2, 100] = np.inf
    x[3, 5] = np.nan
    x[4, 7] = -65504
    c, s = quant_a8(_t(x, dev))
    cn, sn = c.cpu().numpy(), s.cpu().numpy()
    assert (cn[0] == 0).all() and sn[0] == 0
    assert np.array_equal(cn[1], 127 * np.sign(x[1].astype(np.float32)))
    assert np.isnan(sn[[2, 3]]).all() and not np.isnan(sn[[0, 1, 4, 5]]).any()
    w = _t(rng(2).integers(-127, 128, (20, 128)).astype(np.int8), dev)
    y = gemm_a8_packed(c, s, pack_i8(w), _t(np.full(20, 0.01, np.float16), dev), 20, 128).cpu().numpy()
    assert np.isnan(y[[2, 3]]).all() and (y[0] == 0).all()
    # row 4 passes fp16's largest value where |w| > 100 (65504 |w| 0.01 > 65519): those round to infinity, no others do
    z = cn.astype(np.float64) @ w.cpu().numpy().T * sn[:, None] * float(np.float16(0.01))
    rows = [1, 4, 5]
    assert np.array_equal(np.isfinite(y[rows]), np.abs(z[rows]) < 65520) and np.isinf(y[4]).any()


@pytest.mark.parametrize("M,K", [(1, 64), (9, 3072), (4, 8192), (33, 192)])
def test_codes_of_normed_rows(dev, M, K):
    """The norm is in fp32: a code differs from float64's only where the quotient lies within its error of a tie."""
    from estudiocanciones_amd.kernels import quant_a8
    x, w = randn16(3, M, K, std=2.0), (1 + 0.1 * randn16(4, K)).astype(np.float16)
    c, s = quant_a8(_t(x, dev), _t(w, dev), 1e-5)
    xd = x.astype(np.float64)
    y = xd / np.sqrt((xd ** 2).mean(1, keepdims=True) + 1e-5) * w.astype(np.float64)
    quot = y * 127 / np.abs(y).max(1, keepdims=True)
    # squares, their sum (at most 8 terms a thread and pass, then a tree), root, reciprocal, products, quotient
    eps = (K / 256 + 24) * 2.0 ** -24
    far = np.abs(c.cpu().numpy() - quot) > 0.5 + 2 * eps * np.abs(quot)
    assert not far.any()
    sw = np.abs(y).max(1) / 127
    assert (np.abs(s.cpu().numpy() - sw) <= eps * sw).all()


def _weights(N, K, seed=5):
    g = rng(seed)
    w = np.clip(np.rint(g.standard_normal((N, K)) * 40), -127, 127).astype(np.int8)
    s = (0.001 * (1 + 0.3 * g.random(N))).astype(np.float16)
    return w, s


SHAPES = [(1, 16, 64), (1, 5120, 1024), (2, 17, 192), (7, 33, 128), (8, 3072, 3072), (16, 1001, 320), (17, 64, 8192),
          (31, 515, 256), (33, 8197, 1024), (64, 48, 64), (65, 130, 448), (127, 256, 512), (129, 300, 1024),
          (187, 3072, 512), (257, 1001, 192), (300, 2050, 320), (1000, 520, 256), (2100, 1030, 192)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("res", [False, True])
def test_product(dev, M, N, K, res):
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, quant_a8
    x, (w, s) = randn16(M, M, K), _weights(N, K)
    r = randn16(7, M, N) if res else None
    c, sx = quant_a8(_t(x, dev))
    got = gemm_a8_packed(c, sx, pack_i8(_t(w, dev)), _t(s, dev), N, K, None if r is None else _t(r, dev))
    z = (c.cpu().numpy().astype(np.float64) @ w.T.astype(np.float64)) * sx.cpu().numpy().astype(np.float64)[:, None] * s.astype(np.float64)
    want = z + r if res else z
    # the sum to fp32, the product of the scales, their product, the residual: 2^-24 each; one fp16 rounding
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * (np.abs(z) + np.abs(want)) + 2.0 ** -25
    err = np.abs(got.cpu().numpy().astype(np.float64) - want)
    assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:4])


@pytest.mark.parametrize("M,F,K", [(1, 8, 64), (1, 1001, 1024), (8, 8192, 3072), (5, 17, 192), (40, 130, 128),
                                   (187, 1030, 256), (300, 515, 320), (1100, 520, 192)])
def test_silu_product(dev, M, F, K):
    import torch
    from estudiocanciones_amd.kernels import gemm_a8_silu_packed, pack_i8, quant_a8
    x, (w, s) = randn16(M, M, K, std=4.0), _weights(2 * F, K)
    c, sx = quant_a8(_t(x, dev))
    sd = _t(s, dev)
    got = gemm_a8_silu_packed(c, sx, pack_i8(_t(w, dev), interleave=True), torch.stack([sd[:F], sd[F:]], 1).reshape(-1).contiguous(), F, K)
    z = (c.cpu().numpy().astype(np.float64) @ w.T.astype(np.float64)) * sx.cpu().numpy().astype(np.float64)[:, None] * s.astype(np.float64)
    a, b = z[:, :F], z[:, F:]
    want = a / (1 + np.exp(-a)) * b
    # z within 2^-22; the exponential within (|a| + 2) 2^-23, the reciprocal and the products 2^-22; one fp16 rounding
    tol = 2.0 ** -11 * np.abs(want) + np.abs(want) * (np.abs(a) + 8) * 2.0 ** -21 + 2.0 ** -25
    err = np.abs(got.cpu().numpy().astype(np.float64) - want)
    assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:4])


def test_silu_of_large_products(dev):
    """Where exp(-a) overflows the result is 0, where it vanishes a b."""
    from estudiocanciones_amd.kernels import gemm_a8_silu_packed, pack_i8, quant_a8
    x = np.ones((2, 64), np.float16)
    x[1] = -1
    w = np.full((16, 64), 127, np.int8)
    s = np.full(16, 4.0, np.float16)  # a = +-(1 / 127) 4 (64 127 127) = +-32512, b = +-64 127 / 2^13
    s[1::2] = 2.0 ** -13
    c, sx = quant_a8(_t(x, dev))
    wp = pack_i8(_t(w, dev))  # rows are (a, b) pairs as they stand
    y = gemm_a8_silu_packed(c, sx, wp, _t(s, dev), 8, 64).float().cpu().numpy()
    assert np.allclose(y[0], 32512 * 64 * 127 * 2.0 ** -13, rtol=2.0 ** -10) and (y[1] == 0).all()


def test_a_rows_bits_do_not_depend_on_the_call(dev):
    """The sum is an integer: any number of rows, tile and split gives the same bits."""
    import torch
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, quant_a8
    N, K = 1040, 1344
    w, s = _weights(N, K)
    wp, sd, x = pack_i8(_t(w, dev)), _t(s, dev), _t(randn16(3, 600, K), dev)
    c, sx = quant_a8(x)
    whole = gemm_a8_packed(c, sx, wp, sd, N, K)
    for M in (1, 5, 16, 17, 40, 64, 100, 200, 400):
        cm, sm = quant_a8(x[600 - M:])
        assert torch.equal(gemm_a8_packed(cm, sm, wp, sd, N, K), whole[600 - M:]), M


def test_extreme_codes(dev):
    """-128 as a weight, the longest K: the sum stays within 32 bits."""
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, quant_a8
    K = 1 << 17
    x = np.ones((3, K), np.float16)
    x[1] = -1
    w = np.full((16, K), -128, np.int8)
    c, sx = quant_a8(_t(x, dev))
    y = gemm_a8_packed(c, sx, pack_i8(_t(w, dev)), _t(np.full(16, 2.0 ** -14, np.float16), dev), 16, K).float().cpu().numpy()
    assert (y[[0, 2]] == -1024).all() and (y[1] == 1024).all()


def test_strides_and_destinations(dev):
    import torch
    from estudiocanciones_amd.kernels import gemm_a8_packed, gemm_a8_silu_packed, pack_i8, quant_a8
    M, N, K = 70, 130, 192
    w, s = _weights(N, K)
    wp, sd = pack_i8(_t(w, dev)), _t(s, dev)
    wide = _t(randn16(3, M, K + 40), dev)
    c, sx = quant_a8(wide[:, 8:8 + K])
    c2, sx2 = quant_a8(wide[:, 8:8 + K].contiguous())
    assert torch.equal(c, c2) and torch.equal(sx, sx2)
    res = _t(randn16(4, M, N + 3), dev)[:, 1:N + 1]  # rows that are not 16-byte aligned
    out = torch.full((M, N + 7), 5.0, dtype=torch.float16, device=dev)
    got = gemm_a8_packed(c, sx, wp, sd, N, K, res, out=out[:, 2:2 + N])
    assert torch.equal(got, gemm_a8_packed(c2, sx2, wp, sd, N, K, res.contiguous()))
    assert (out[:, :2] == 5).all() and (out[:, 2 + N:] == 5).all()
    mm = torch.full((M, N // 2 + 3), 5.0, dtype=torch.float16, device=dev)
    got = gemm_a8_silu_packed(c, sx, wp, sd, N // 2, K, out=mm[:, 1:1 + N // 2])
    assert torch.equal(got, gemm_a8_silu_packed(c, sx, wp, sd, N // 2, K))
    assert (mm[:, 0] == 5).all() and (mm[:, 1 + N // 2:] == 5).all()


@pytest.mark.parametrize("M", [5, 40, 300, 600])
def test_a_part_of_the_columns(dev, M):
    """Codes of a longer row, from one column to another: the columns behind K do not count, whatever they hold."""
    from estudiocanciones_amd._ffi import call
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, stream_ptr
    import torch
    g = rng(31)
    whole = _t(g.integers(-127, 128, (M, 512)).astype(np.int8), dev)
    N = 300
    s, sx = _t((0.01 * (1 + g.random(N))).astype(np.float16), dev), _t((0.01 * (1 + g.random(M))).astype(np.float32), dev)
    for a, b in ((0, 192), (64, 512), (320, 384), (192, 512), (16, 208), (432, 496)):
        w = _t(g.integers(-127, 128, (N, b - a)).astype(np.int8), dev)
        wp, c = pack_i8(w), whole[:, a:b]
        got = gemm_a8_packed(c, sx, wp, s, N, b - a)
        want = (c.double() @ w.double().T) * sx.double()[:, None] * s.double()
        # |sum| < 2^24 is a value of fp32; two products in fp32, one rounding to fp16 (2^-24 absolute where it is subnormal)
        assert ((got.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -22) * want.abs() + 2.0 ** -25).all()
        for cfg in range(2, 9):
            y = torch.empty_like(got)
            call("ecd_gemm_a8_tuned", c.data_ptr(), 512, sx.data_ptr(), wp.data_ptr(), s.data_ptr(), None, 0, y.data_ptr(), N,
                 M, N, b - a, cfg, stream_ptr(y.device))
            assert torch.equal(y, got)


@pytest.mark.parametrize("M,N", [(3, 40), (12, 300), (90, 1001), (600, 520)])
def test_residual_in_place(dev, M, N):
    """The residual's rows may be the result's."""
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, quant_a8
    import torch
    g = rng(32)
    K = 320
    c, sx = quant_a8(_t(g.standard_normal((M, K)).astype(np.float16), dev))
    wp = pack_i8(_t(g.integers(-127, 128, (N, K)).astype(np.int8), dev))
    s = _t((0.001 * (1 + g.random(N))).astype(np.float16), dev)
    wide = _t(g.standard_normal((M, N + 13)).astype(np.float16), dev)
    y = wide[:, 3:3 + N]
    keep = wide.clone()
    want = gemm_a8_packed(c, sx, wp, s, N, K, res=y.clone())
    gemm_a8_packed(c, sx, wp, s, N, K, res=y, out=y)
    assert torch.equal(y, want)
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 3 + N:], keep[:, 3 + N:])


@pytest.mark.parametrize("M,N,K", [(262200, 8200, 64), (33000, 40, 131072)])
def test_offsets_past_32_bits(dev, M, N, K):
    """More than 2^31 results, more than 2^32 bytes of codes: the last rows have the bits that they have by themselves."""
    from estudiocanciones_amd.kernels import gemm_a8_packed, gemm_a8_silu_packed, pack_i8, quant_a8
    import torch
    g = rng(33)
    x = _t(g.standard_normal((64, K)).astype(np.float16), dev).repeat(-(-M // 64), 1)[:M]
    wp = pack_i8(_t(g.integers(-127, 128, (N, K)).astype(np.int8), dev))
    s = _t((0.001 * (1 + g.random(N))).astype(np.float16), dev)
    c, sx = quant_a8(x)
    y = gemm_a8_packed(c, sx, wp, s, N, K, res=None)
    z = gemm_a8_silu_packed(c, sx, wp, s, N // 2, K)
    for r in (0, M // 2 // 64 * 64, M - 70):
        c1, sx1 = quant_a8(x[r:r + 70])
        assert torch.equal(c1, c[r:r + 70]) and torch.equal(sx1, sx[r:r + 70])
        assert torch.equal(gemm_a8_packed(c1, sx1, wp, s, N, K), y[r:r + 70])
        assert torch.equal(gemm_a8_silu_packed(c1, sx1, wp, s, N // 2, K), z[r:r + 70])
    assert torch.equal(y[:64], y[(M // 64 - 1) * 64:M // 64 * 64])


def test_no_rows(dev):
    import torch
    from estudiocanciones_amd.kernels import gemm_a8_packed, pack_i8, quant_a8
    w, s = _weights(32, 64)
    c, sx = quant_a8(torch.empty(0, 64, dtype=torch.float16, device=dev))
    assert gemm_a8_packed(c, sx, pack_i8(_t(w, dev)), _t(s, dev), 32, 64).shape == (0, 32)


@pytest.mark.parametrize("M,N,K", [(1, 16, 64), (9, 1001, 192), (40, 33, 128), (70, 300, 1344), (130, 260, 448), (300, 1030, 320)])
def test_every_kernel_gives_the_same_bits(dev, M, N, K):
    """All kernels that ecd_gemm_a8 chooses from, on shapes with fewer and more chunks of k than stages and K groups."""
    import torch
    from estudiocanciones_amd import _ffi
    from estudiocanciones_amd.kernels import pack_i8, quant_a8, stream_ptr
    w, s = _weights(N, K)
    c, sx = quant_a8(_t(randn16(M, M, K), dev))
    wp, sd, res = pack_i8(_t(w, dev)), _t(s, dev), _t(randn16(7, M, N), dev)
    ys = []
    for cfg in range(1, 9):
        y = torch.full((M, N), float("nan"), dtype=torch.float16, device=dev)
        _ffi.call("ecd_gemm_a8_tuned", c.data_ptr(), c.stride(0), sx.data_ptr(), wp.data_ptr(), sd.data_ptr(), res.data_ptr(), N,
                  y.data_ptr(), N, M, N, K, cfg, stream_ptr(dev))
        ys.append(y)
    z = (c.cpu().numpy().astype(np.int64) @ w.T.astype(np.int64)) * sx.cpu().numpy().astype(np.float64)[:, None] * s.astype(np.float64)
    want = z + res.cpu().numpy()
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * (np.abs(z) + np.abs(want)) + 2.0 ** -25
    assert (np.abs(ys[0].cpu().numpy() - want) <= tol).all()
    for k, y in enumerate(ys):
        assert torch.equal(y, ys[0]), k + 1


def test_refusals(dev):
    import torch
    from estudiocanciones_amd.kernels import gemm_a8_packed, gemm_a8_silu_packed, pack_i8, quant_a8
    x = _t(randn16(1, 4, 128), dev)
    for bad in (x[:, :96], x[:, ::2], x.reshape(-1)[4:4 + 64 * 7].reshape(7, 64), x[0]):
        with pytest.raises(ValueError):
            quant_a8(bad)
    with pytest.raises(TypeError):
        quant_a8(x.float())
    with pytest.raises(ValueError):
        quant_a8(x, _t(randn16(2, 64), dev))
    w, s = _weights(32, 128)
    wp, sd = pack_i8(_t(w, dev)), _t(s, dev)
    c, sx = quant_a8(x)
    for a in ((c, sx, wp, sd, 48, 128), (c, sx, wp, sd, 32, 64), (c[:, ::2], sx, wp, sd, 32, 64), (c, sx[:3], wp, sd, 32, 128),
              (c, sx, wp[:100], sd, 32, 128), (c, sx, wp, sd[:16], 32, 128), (c.float(), sx, wp, sd, 32, 128)):
        with pytest.raises(ValueError):
            gemm_a8_packed(*a)
    with pytest.raises(ValueError):
        gemm_a8_packed(c, sx, wp, sd, 32, 128, res=x[:, :32].t())
    with pytest.raises(ValueError):
        gemm_a8_silu_packed(c, sx, wp, sd, 16, 128, out=torch.empty(4, 32, dtype=torch.float16, device=dev))
