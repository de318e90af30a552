"""4-bit products of views and of sizes past 31 bits."""
import numpy as np
import pytest

from helpers import randn16
from test_gpu_q4 import H, _t, make, packed

pytestmark = pytest.mark.gpu


def wide(dev, rows, ld, K, seed):
    """[rows, K] of rows ld apart, in memory of which the rest is NaN around them."""
    import torch
    flat = torch.empty((rows - 1) * ld + K + 64, device=dev, dtype=torch.float16)
    x = flat.as_strided((rows, K), (ld, 1))
    flat.as_strided((rows, K + 64), (ld, 1)).fill_(float("nan"))
    x.copy_(_t(randn16(seed, rows, K), dev))
    return x


@pytest.mark.parametrize("M", [2, 16, 17, 40, 130])
@pytest.mark.parametrize("ld", [(1 << 23) + 8, (1 << 24) + 8])
def test_rows_far_apart(dev, M, ld):
    """Row strides that 32 bits of a tile's offsets do not reach: the values of a compact copy, within the kernels' sums."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4
    for N, K, group in ((70, 192, 64), (3000, 128, 128)):
        q, s, z, w = make(M, N, K, group, True)
        wp = packed(dev, q, s, z)
        x = wide(dev, M, ld, K, M)
        res, nw = _t(randn16(M + 1, M, N), dev), torch.ones(K, device=dev, dtype=torch.float16)
        x64 = x.double().cpu().numpy()
        A = np.abs(x64) @ np.abs(w).T
        tol = (2.0 ** -23 * (64 + K // 64 + 32) + K / 32 * 1.25 * 2.0 ** -22) * A
        want = x64 @ w.T + res.double().cpu().numpy()
        got = mm_q4(x, wp, res=res).double().cpu().numpy()
        assert (np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25).all()
        assert torch.equal(mm_q4(x, wp, nw=nw), mm_q4(x.contiguous(), wp, nw=nw))
        del x


@pytest.mark.parametrize("M,N,K", [(130, 16384, 192), (200, 5120, 1024), (400, 8197, 1024)])
def test_rows_too_far_apart_for_the_tiles(dev, M, N, K):
    """Sizes that go by tiles where rows are close together."""
    import torch
    from estudiocanciones_amd import _ffi
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    assert 1 <= _ffi.lib().ecd_mm_q4_choice(M, N, K) & 255 <= 6
    q, s, z, w = make(M, N, K, 128, True)
    x = wide(dev, M, (1 << 24) + 8, K, M)
    x64 = x.double().cpu().numpy()
    want = x64 @ w.T
    tol = (2.0 ** -23 * (64 + K // 64 + 32) + K / 32 * 1.25 * 2.0 ** -22) * (np.abs(x64) @ np.abs(w).T)
    got = mm_q4(x, packed(dev, q, s, z)).double().cpu().numpy()
    assert (np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25).all()
    if N % 2 == 0:
        a, b, ta, tb = want[:, :N // 2], want[:, N // 2:], tol[:, :N // 2], tol[:, N // 2:]
        f = a / (1 + np.exp(-a))
        want, tol = f * b, (1.1 * ta + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb
        wi, nw = packed(dev, q, s, z, True), torch.ones(K, device=dev, dtype=torch.float16)
        got = mm_q4_silu(x, wi).double().cpu().numpy()
        assert (np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25).all()
        assert torch.equal(mm_q4_silu(x, wi, nw=nw), mm_q4_silu(x.contiguous(), wi, nw=nw))


def test_one_row_however_far_the_next(dev):
    """A row's stride says nothing where there is one row: as of a view of a wide tensor."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    N, K = 70, 192
    q, s, z, w = make(3, N, K, 32, True)
    x = _t(randn16(5, 1, K), dev)
    for il, f in ((False, mm_q4), (True, mm_q4_silu)):
        wp = packed(dev, q, s, z, il)
        for ld in (1 << 26, (1 << 26) + 8, 1 << 27, 1 << 40, (1 << 40) + 3):
            assert torch.equal(f(x.as_strided((1, K), (ld, 1)), wp), f(x, wp))


@pytest.mark.parametrize("silu", [False, True])
def test_more_rows_than_blocks_of_a_launch(dev, silu):
    """1.1 million rows (of more than 2^31 bytes): the first, the last and some between them."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    M, N, K = 1_100_003, 16, 1024
    q, s, z, w = make(1, N, K, 128, False)
    wp = packed(dev, q, s, z, silu)
    x = torch.empty(M, K, device=dev, dtype=torch.float16)
    x.normal_(generator=torch.Generator(device=dev).manual_seed(1))
    y = (mm_q4_silu if silu else mm_q4)(x, wp)
    for a in (0, 524288, M - 700):
        x64 = x[a:a + 700].double().cpu().numpy()
        A, want = np.abs(x64) @ np.abs(w).T, x64 @ w.T
        tol = (2.0 ** -23 * (64 + K // 64 + 32) + K / 32 * 1.25 * 2.0 ** -22) * A
        if silu:
            g, b, tg, tb = want[:, :8], want[:, 8:], tol[:, :8], tol[:, 8:]
            f = g / (1 + np.exp(-g))
            want, tol = f * b, (1.1 * tg + 2.0 ** -20 * np.abs(f)) * (np.abs(b) + tb) + np.abs(f) * tb
        got = y[a:a + 700].double().cpu().numpy()
        assert (np.abs(got - want) <= tol + H * (np.abs(want) + tol) + 2.0 ** -25).all()


@pytest.mark.parametrize("M", [1, 3, 12, 40, 200])
def test_results_beside_their_inputs(dev, M):
    """out in columns of the same wide rows as x or res, which do not meet; columns that do are refused, and nothing is written."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4, process_logits
    N, K = 72, 192
    q, s, z, w = make(M, N, K, 64, True)
    wp = packed(dev, q, s, z)
    for at in (0, N, K):  # out before x, behind it, and res behind out
        room = torch.full((M, K + 2 * N + 8), 7.0, device=dev, dtype=torch.float16)
        cols = {"x": K, "out": N, "res": N}
        order = {0: ["out", "x", "res"], N: ["x", "out", "res"], K: ["res", "x", "out"]}[at]
        v, c = {}, 0
        for n in order:
            v[n] = room[:, c:c + cols[n]]
            c += cols[n]
        v["x"].copy_(_t(randn16(M, M, K), dev))
        v["res"].copy_(_t(randn16(M + 1, M, N), dev))
        x, res = v["x"].clone(), v["res"].clone()
        mm_q4(v["x"], wp, res=v["res"], out=v["out"])
        assert torch.equal(v["out"], mm_q4(x, wp, res=res))
        assert torch.equal(v["x"], x) and torch.equal(v["res"], res) and (room[:, c:] == 7.0).all()
    if M > 1:
        before = room.clone()
        for out in (room[:, 1:1 + N], room[:, 100:100 + N], room[:, K + N - 1:K + 2 * N - 1]):
            with pytest.raises(ValueError):
                mm_q4(v["x"], wp, res=v["res"], out=out)
        assert torch.equal(room, before)
    lg = torch.full((2 * M, 300), 7.0, device=dev, dtype=torch.float16)
    lg[:, :100] = _t(randn16(3, 2 * M, 100), dev)
    src = lg[:, :100].clone()
    process_logits(lg[:, :100], cfg=1.5, out=lg[:M, 100:200])
    assert torch.equal(lg[:M, 100:200], process_logits(src, cfg=1.5))
    assert torch.equal(lg[:, :100], src) and (lg[:, 200:] == 7.0).all() and (lg[M:, 100:] == 7.0).all()
    for out in (lg[:M, 99:199], lg[M:, :100], lg[:M, 200:].as_strided((M, 100), (299, 1))):
        if M > 1 or out.data_ptr() < lg[1].data_ptr() + 200 and out.storage_offset() % 300 < 100:
            with pytest.raises(ValueError):
                process_logits(lg[:, :100], cfg=1.5, out=out)


@pytest.mark.parametrize("silu", [False, True])
def test_results_past_31_bits(dev, silu):
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu
    M, N, K = 66001, 32800 if silu else 16400, 64
    cols = N // 2 if silu else N
    q, s, z, w = make(2, N, K, 32, True)
    wp = packed(dev, q, s, z, silu)
    x = _t(randn16(1, M, K), dev)
    y = (mm_q4_silu if silu else mm_q4)(x, wp)
    assert y.numel() * 2 > 2 ** 31
    wt, aw = _t(w.T, dev), _t(np.abs(w).T, dev)
    for a in (0, 32768, M - 999):
        x64 = x[a:a + 999].double()
        want, A = x64 @ wt, x64.abs() @ aw
        tol = (2.0 ** -23 * (64 + K // 64 + 32) + K / 32 * 1.25 * 2.0 ** -22) * A
        if silu:
            g, b, tg, tb = want[:, :cols], want[:, cols:], tol[:, :cols], tol[:, cols:]
            f = g / (1 + (-g).exp())
            want, tol = f * b, (1.1 * tg + 2.0 ** -20 * f.abs()) * (b.abs() + tb) + f.abs() * tb
        assert ((y[a:a + 999].double() - want).abs() <= tol + H * (want.abs() + tol) + 2.0 ** -25).all()


@pytest.mark.parametrize("silu", [False, True])
def test_weights_past_31_bits(dev, silu):
    """Weights to quantise, codes and packed codes of more than 2^31 bytes: the last features come out as on their own."""
    import torch
    from estudiocanciones_amd.kernels import mm_q4, mm_q4_silu, pack_q4
    from estudiocanciones_amd.quant import q4_rows
    N, K = 1_050_004, 4096
    g = torch.Generator(device=dev).manual_seed(2)
    t = torch.empty(N, K, device=dev, dtype=torch.bfloat16)
    t.normal_(generator=g)
    q, s, z = q4_rows(t, 128, True)
    del t
    assert q.numel() > 2 ** 31
    w, half = pack_q4(q, s, z, silu), N // 2
    for M in (3, 40):
        x = _t(randn16(M, M, K), dev)
        y = (mm_q4_silu if silu else mm_q4)(x, w)
        for a in (0, half - 600, N - 600) if not silu else (0, half - 600):
            rows = torch.arange(a, a + 600, device=dev)
            rows = torch.cat([rows, rows + half]) if silu else rows
            u = torch.stack([q[rows] & 15, q[rows] >> 4], -1).flatten(1).double()
            wd = (u - z[rows].double().repeat_interleave(128, 1)) * s[rows].double().repeat_interleave(128, 1)
            x64 = x.double()
            want, A = x64 @ wd.t().contiguous(), x64.abs() @ wd.abs().t().contiguous()
            tol = (2.0 ** -23 * (64 + K // 64 + 32) + K / 32 * 1.25 * 2.0 ** -22) * A
            if silu:
                ga, b, tg, tb = want[:, :600], want[:, 600:], tol[:, :600], tol[:, 600:]
                f = ga / (1 + (-ga).exp())
                want, tol = f * b, (1.1 * tg + 2.0 ** -20 * f.abs()) * (b.abs() + tb) + f.abs() * tb
            assert ((y[:, a:a + 600].double() - want).abs() <= tol + H * (want.abs() + tol) + 2.0 ** -25).all()
        assert y.shape[1] == (half if silu else N)
    assert torch.equal(q4_rows(torch.zeros(1, K, device=dev), 128, True)[0], torch.zeros(1, K // 2, device=dev, dtype=torch.uint8))
