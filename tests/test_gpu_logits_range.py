"""process_logits where values leave fp16: above, a finite one stops at the largest number, so that a sampler's softmax has no infinity to
subtract; below, it is -inf, which draws nothing."""
import numpy as np
import pytest

from helpers import randn16, rng
from test_gpu_logits import _t, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [5, 100, 8197])
@pytest.mark.parametrize("way", ["bias", "presence", "frequency", "repetition", "guidance"])
def test_values_above_the_range_stop_at_the_largest(dev, V, way):
    import torch
    from estudiocanciones_amd.kernels import process_logits, sample_topk
    N = 3
    x = randn16(V, 2 * N, V)
    hot = np.array([1, V - 1, V // 2])
    x[np.arange(N), hot] = 2
    x[np.arange(N, 2 * N), hot] = -2
    hist = np.repeat(hot[:, None], 2, 1)
    one = lambda v: _t(np.float32([v]), dev)  # noqa: E731
    bias = np.zeros((N, V), np.float32)
    bias[np.arange(N), hot] = [65504, 1e5, 3e38]
    kw = {"bias": dict(bias=_t(bias, dev)), "presence": dict(hist=_t(hist, dev), presence=one(-1e5)),
          "frequency": dict(hist=_t(hist, dev), frequency=one(-1e30)), "repetition": dict(hist=_t(hist, dev), repetition=one(1e-30)),
          "guidance": dict(cfg=1e5)}[way]
    out = process_logits(_t(x if way == "guidance" else x[:N], dev), **kw)
    got = out.cpu().numpy()
    assert (got[np.arange(N), hot] == 65504).all()
    if way != "guidance":  # the others as they were
        keep = np.ones((N, V), bool)
        keep[np.arange(N), hot] = False
        assert np.array_equal(got[keep], x[:N][keep])
        tok = torch.full((N, 1), -1, device=dev, dtype=torch.int64)
        for p in range(4):
            sample_topk(out, N, 1.0, 1.0, 3, tok[:, 0], seed=torch.tensor([5], device=dev), pos=torch.tensor([p], device=dev))
            assert np.array_equal(tok[:, 0].cpu().numpy(), hot)


def test_what_is_infinite_stays_so(dev):
    """Infinite logits and biases and NaN pass through; values below the range are -inf; a mask still takes everything."""
    from estudiocanciones_amd.kernels import process_logits
    x = np.float16([[np.inf, 1, np.nan, 2, -65504, 65504, 65504, 65504, np.inf, 3]])
    bias = np.float32([[0, np.inf, 0, -1e5, -100, 15, 16, 1e30, 0, 1e5]])
    keep = np.ones((1, 10), bool)
    keep[0, 8:] = False
    got = process_logits(_t(x, dev), bias=_t(bias, dev), allowed=_t(words(keep), dev)).cpu().numpy()
    want = np.float16([[np.inf, np.inf, np.nan, -np.inf, -np.inf, 65504, 65504, 65504, -np.inf, -np.inf]])
    assert np.array_equal(got, want, equal_nan=True)


def test_rows_past_31_bits(dev):
    """Logits and results of more than 2^31 bytes: the last rows come out as on their own."""
    import torch
    from estudiocanciones_amd.kernels import process_logits
    N, V = 9000, 120001
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.empty(N, V, device=dev, dtype=torch.float16)
    x.normal_(generator=g)
    hist = torch.randint(0, V, (N, 7), device=dev, generator=g)
    rep = torch.full((N,), 1.5, device=dev)
    out = process_logits(x, hist, repetition=rep)
    assert (N - 1) * out.stride(0) * 2 > 2 ** 31 and (N - 1) * V * 2 > 2 ** 31
    for a in (slice(0, 2), slice(N - 3, N)):
        own = process_logits(x[a].clone(), hist[a].clone(), repetition=rep[a])
        assert torch.equal(out[a], own)
        seen = torch.zeros_like(own, dtype=torch.bool).scatter_(1, hist[a], True)
        l = x[a].float()
        assert torch.equal(own, torch.where(seen, torch.where(l > 0, l / 1.5, l * 1.5), l).half())
