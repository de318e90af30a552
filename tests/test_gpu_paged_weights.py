"""The weights of decode attention over pages: scores that are exact in fp32, so that what is left is how the kernel forms,
scales and sums the weights (float64 references)."""
import numpy as np
import pytest

from test_gpu_paged_attn import Batch

pytestmark = pytest.mark.gpu

HEADS = [(6, 2, 128), (24, 8, 128), (12, 2, 64), (8, 2, 256)]
SHARES = (True, False, None)


def _fill(b, slots, q, k, v):
    """The same few dims of k [slots, d], v [slots, HD] for every kv head and row, q [d] for every query head (the rest 0)."""
    Hq, Hk, HD, P = b.H
    b.q[:] = 0
    b.q.reshape(b.R, Hq, HD)[:, :, :len(q)] = q
    assert max(b.lens) <= slots
    for r, m in enumerate(b.lens):
        t = np.arange(m)
        page = b.table[r // b.S, t // P]
        full = np.zeros((m, HD), np.float16)
        full[:, :k.shape[1]] = k[:m]
        b.pool[0][page, :, t % P] = full[:, None]
        b.pool[1][page, :, t % P] = v[:m, None]


def _check(b, dev, s, v):
    """s [slots]: the exact scores (scale 1).  A weight is off by
      exponent: the difference to the maximum, its product with log2(e), log2(e) itself and the sum behind it, 2^-24 each of
        at most 14 + 1.5 |s - max|, times ln 2;
      the exponential itself 2^-22; what is left of it in two fp16 values 2^-20, or 2^-38 of the largest weight;
      fp32 sums over at most 9000 slots in chains of at most 300, and the joins: 2^-15 would be a chain of 512 roundings that
        all go one way; a mean of them is 2^-24 sqrt(512) < 2^-19;
    and the result is rounded to fp16 once."""
    HD = b.H[2]
    for share in SHARES:
        got = b.run(dev, scale=1.0, share=share).double().cpu().numpy().reshape(b.R, -1, HD)
        for r, m in enumerate(b.lens):
            if not m:
                assert (got[r] == 0).all()
                continue
            d = s[:m] - s[:m].max()
            p = np.exp(d)
            want = p @ v[:m].astype(np.float64) / p.sum()
            near = np.abs(d[p > 2.0 ** -40]).max()  # (smaller weights do not count)
            rel = 2.0 ** -24 * 4 * (14 + 1.5 * near) + 2.0 ** -22 + 2.0 ** -20 + 2.0 ** -18
            tol = 2.0 ** -11 * np.abs(want) + rel * (p @ np.abs(v[:m].astype(np.float64)) / p.sum()) \
                + 2.0 ** -38 * np.abs(v[:m].astype(np.float64)).sum(0) / p.sum() + 2.0 ** -25
            err = np.abs(got[r] - want)
            assert (err <= tol).all(), (share, r, m, float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("Hq,Hk,HD", HEADS)
def test_weights_that_cancel(dev, Hq, Hk, HD):
    """Values whose weighted sum nearly cancels: the result is a difference of weights, and fp16 weights (2^-11 each) show."""
    lens = [2, 3, 40, 64, 65, 200, 330, 331]
    b = Batch([(4, 0), (4, 65)], lens, Hq, Hk, HD, 16, seed=3)
    g = np.random.default_rng(5)
    k = g.integers(-40, 41, (331, 1)) / 32  # exact scores
    v = np.ones((331, HD), np.float16)
    v[1::2] = -1
    v[:, 1::2] *= np.float16(0.75)
    _fill(b, 331, np.array([1.0]), k.astype(np.float16), v)
    _check(b, dev, k[:, 0], v)


@pytest.mark.parametrize("Hq,Hk,HD", HEADS)
def test_many_small_weights_beside_a_large_one(dev, Hq, Hk, HD):
    """A slot in each of the first tiles takes nearly all of the weight; the others have e^-17.5 = 2^-25.2 of it each, below
    what fp16 holds, and there are enough of them to count."""
    n = 9000
    k = np.zeros((n, 1))
    k[:1024:32] = 17.5
    v = np.ones((n, HD), np.float16)
    v[:1024:32] = 0
    b = Batch([(1, 0), (2, 8000)], [n, 8000, 8500], Hq, Hk, HD, 64, seed=2)
    _fill(b, n, np.array([1.0]), k.astype(np.float16), v)
    _check(b, dev, k[:, 0], v)


@pytest.mark.parametrize("Hq,Hk,HD", HEADS)
def test_large_scores_that_rise(dev, Hq, Hk, HD):
    """Scores of 2^20 and more that differ by a few eighths, rising from tile to tile: the running maximum's changes must not
    scale the sums by anything but the weights' own factor."""
    n = 700
    k = np.stack([np.full(n, 1024.0), np.minimum(np.arange(n) // 16, 40), np.arange(n) * 7 % 5], 1)  # exact in fp16
    q = np.array([1024.0, 0.125, 0.125])
    v = np.random.default_rng(7).standard_normal((n, HD)).astype(np.float16)
    b = Batch([(2, 0), (3, 300)], [n, 33, 300, 640, 411], Hq, Hk, HD, 32, seed=6)
    _fill(b, n, q, k.astype(np.float16), v)
    s = k @ q
    assert s.max() < 2 ** 21 and (s * 8 == np.rint(s * 8)).all()  # at most 24 bits: exact in fp32 in any order
    _check(b, dev, s, v)


@pytest.mark.parametrize("Hq,Hk,HD", HEADS)
def test_an_infinite_value_that_is_attended(dev, Hq, Hk, HD):
    """An infinity in a slot of any weight that counts stays one, with its sign, and only in its dim."""
    n = 300
    k = (np.arange(n) % 7)[:, None] * 1.5
    v = np.random.default_rng(8).standard_normal((n, HD)).astype(np.float16)
    clean = v.copy()
    # scores 0 (e^-9 of the largest), 1.5, and the largest, whose weight is one fp16 value exactly
    v[21, 3], v[260, HD - 1], v[6, 5], v[13, 7] = np.inf, -np.inf, np.inf, -np.inf
    b = Batch([(2, 0), (3, 280)], [n, 300, 280, 300, 290], Hq, Hk, HD, 32, seed=6)
    _fill(b, n, np.array([1.0]), k.astype(np.float16), v)
    for share in SHARES:
        got = b.run(dev, scale=1.0, share=share).double().cpu().numpy().reshape(b.R, Hq, HD)
        assert (got[:, :, [3, 5]] == np.inf).all() and (got[:, :, [7, HD - 1]] == -np.inf).all()
        for r, m in enumerate(b.lens):
            p = np.exp(k[:m, 0] - 9.0)
            want = p @ clean[:m].astype(np.float64) / p.sum()
            rest = [d for d in range(HD) if d not in (3, 5, 7, HD - 1)]
            assert (np.abs(got[r] - want)[:, rest] <= 2.0 ** -10).all()
