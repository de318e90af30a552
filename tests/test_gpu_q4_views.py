"""4-bit products of views and of sizes past 31 bits."""
import numpy as np
import pytest

from helpers import randn16
from test_gpu_q4 import H, _t, make, packed

pytestmark = pytest.mark.gpu


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
