"""process_logits against float64: guidance, penalties over a history, biases and masks."""
import numpy as np
import pytest

from helpers import randn16, rng

pytestmark = pytest.mark.gpu

H = 2.0 ** -11  # half a step of fp16, relative


def _t(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def words(keep):
    """bool [A, V] -> int32 [A, ceil(V / 32)], bit v % 32 of word v // 32."""
    A, V = keep.shape
    pad = np.zeros((A, -(-V // 32) * 32), bool)
    pad[:, :V] = keep
    return np.packbits(pad, axis=1, bitorder="little").view(np.int32)


def plain(logits, hist=None, length=None, window=0, rep=None, pres=None, freq=None, bias=None, keep=None, state=None, cfg=None):
    """(result, what fp32 roundings can add up to) in float64."""
    l = logits.astype(np.float64)
    mag = np.abs(l)
    if cfg is not None:
        N = len(l) // 2
        mag = np.abs(l[N:]) + np.abs(cfg) * (np.abs(l[:N]) + np.abs(l[N:]))
        l = l[N:] + (l[:N] - l[N:]) * cfg
    N, V = l.shape
    one = lambda v, d: np.full(N, d) if v is None else np.broadcast_to(v.astype(np.float64), N)  # noqa: E731
    rep, pres, freq = one(rep, 1.0), one(pres, 0.0), one(freq, 0.0)
    for r in range(N):
        if hist is not None:
            n = len(hist[r]) if length is None else int(np.clip(length[r], 0, len(hist[r])))
            seen = hist[r, max(0, n - window) if window else 0:n]
            c = np.bincount(seen[(seen >= 0) & (seen < V)], minlength=V)
            t = c > 0
            l[r, t] = np.where(l[r, t] > 0, l[r, t] / rep[r], l[r, t] * rep[r])
            p = pres[r] + freq[r] * c[t]
            mag[r, t] = mag[r, t] * max(rep[r], 1 / rep[r]) + 2 * (np.abs(pres[r]) + np.abs(freq[r]) * c[t])
            l[r, t] -= p
        if bias is not None:
            b = bias[r] if bias.ndim == 2 else bias
            l[r] += b
            mag[r] += np.abs(b)
        if keep is not None:
            s = (0 if len(keep) == 1 else r) if state is None else state[r]
            if s >= len(keep) or s < -1:
                l[r] = -np.inf
            elif s >= 0:
                l[r, ~keep[s]] = -np.inf
    return l, 8 * 2.0 ** -24 * mag  # (eight fp32 roundings at most)


def check(out, want, tol):
    got = out.double().cpu().numpy()
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    f = np.isfinite(want)
    err = np.abs(got[f] - want[f])
    assert (err <= tol[f] + H * (np.abs(want[f]) + tol[f]) + 2.0 ** -25).all(), err.max()
    assert np.array_equal(got[~f], want[~f], equal_nan=True)


@pytest.mark.parametrize("V", [1, 7, 31, 33, 2048, 2049, 8197, 40003])
@pytest.mark.parametrize("N,T,window", [(1, 1, 0), (3, 300, 0), (5, 1000, 64), (2, 257, 1000)])
@pytest.mark.parametrize("guided", [False, True])
def test_everything_together(dev, V, N, T, window, guided):
    from estudiocanciones_amd.kernels import process_logits
    g = rng(V + T)
    x = randn16(V + N, 2 * N if guided else N, V, std=4.0)
    hist = (V * g.random((N, T)) ** 2).astype(np.int64)
    length = g.integers(0, T + 1, N)
    rep, pres, freq = ((a + b * g.random(N)).astype(np.float32) for a, b in ((1.05, 0.5), (0.1, 1.0), (0.01, 0.2)))
    bias = np.where(g.random((N, V)) < 0.2, 3 * g.standard_normal((N, V)), 0).astype(np.float32)
    keep = g.random((4, V)) < 0.7
    state = g.integers(-1, 4, N).astype(np.int32)
    cfg = 1.5 if guided else None
    out = process_logits(_t(x, dev), _t(hist, dev), _t(length, dev), window, _t(rep, dev), _t(pres, dev), _t(freq, dev),
                         _t(bias, dev), _t(words(keep), dev), _t(state, dev), cfg)
    check(out, *plain(x, hist, length, window, rep, pres, freq, bias, keep, state, cfg))


@pytest.mark.parametrize("which", range(8))
def test_each_part_alone(dev, which):
    import torch
    from estudiocanciones_amd.kernels import process_logits
    g = rng(which)
    N, V, T = 4, 3001, 200
    x = randn16(which, N, V, std=4.0)
    hist = g.integers(0, V, (N, T))
    one = lambda v: np.array([v], np.float32)  # noqa: E731
    kw = [{}, {"hist": hist}, {"hist": hist, "rep": one(1.3)}, {"hist": hist, "pres": np.float32([0.5, 0, 1, 2])},
          {"hist": hist, "freq": one(0.25)}, {"bias": g.standard_normal(V).astype(np.float32)},
          {"keep": g.random((1, V)) < 0.5}, {"keep": g.random((N, V)) < 0.5}][which]
    names = {"rep": "repetition", "pres": "presence", "freq": "frequency", "keep": "allowed"}
    args = {names.get(k, k): _t(words(v) if k == "keep" else v, dev) for k, v in kw.items()}
    out = process_logits(_t(x, dev), **args)
    check(out, *plain(x, **kw))
    if which < 2:
        assert torch.equal(out, _t(x, dev))  # nothing to change


def test_masked_tokens_hold_anything(dev):
    """Infinities and NaN under a mask; a row whose mask leaves nothing; states outside the masks; tokens outside the
    vocabulary in a history; lengths below 0 and past T."""
    from estudiocanciones_amd.kernels import process_logits
    g = rng(5)
    N, V, T = 6, 500, 40
    x = randn16(1, 2 * N, V)
    keep = g.random((3, V)) < 0.5
    keep[2] = False
    for r in range(2 * N):
        x[r, ~keep[0] & ~keep[1]] = [np.inf, -np.inf, np.nan, 65504][r % 4]
    hist = g.integers(-3, V + 3, (N, T))
    hist[0, :5] = [-2 ** 63, 2 ** 63 - 1, 2 ** 32, -1, V]
    length = np.array([T, -5, T + 9, 0, 2 ** 62, 7])
    state = np.array([0, 1, 2, 0, 3, 1], np.int32)
    rep, freq = np.float32([1.2]), np.float32([0.1])
    out = process_logits(_t(x, dev), _t(hist, dev), _t(length, dev), repetition=_t(rep, dev), frequency=_t(freq, dev),
                         allowed=_t(words(keep), dev), state=_t(state, dev), cfg=2.0)
    with np.errstate(invalid="ignore"):
        want, tol = plain(x, hist, length, rep=rep, freq=freq, keep=keep, state=state, cfg=2.0)
    check(out, want, tol)
    assert np.isneginf(want[[2, 4]]).all()


def test_unmasked_infinities_follow_the_formula(dev):
    from estudiocanciones_amd.kernels import process_logits
    x = np.float16([[np.inf, -np.inf, np.nan, 0.0, -0.0, 65504, -65504, 6e-8, 1]])
    hist = np.arange(9, dtype=np.int64)[None]
    out = process_logits(_t(x, dev), _t(hist, dev), repetition=_t(np.float32([2.0]), dev)).cpu().numpy()
    assert np.array_equal(out, np.float16([[np.inf, -np.inf, np.nan, 0, 0, 32752, -np.inf, 0, 0.5]]), equal_nan=True)


@pytest.mark.parametrize("T,V", [(6000, 8197), (20000, 50), (3, 100003)])
def test_frames_of_a_song_as_history(dev, T, V):
    """One codebook of frames [T, N, 8]: a history with strides along both; counts of one token past 16 bits."""
    import torch
    from estudiocanciones_amd.kernels import process_logits
    g = rng(T)
    N = 3
    frames = np.minimum((V * g.random((T, N, 8)) ** 4).astype(np.int64), V - 1)
    if V == 50:
        frames[:, 1] = 7
    x = randn16(2, N, V, std=3.0)
    ft = _t(frames, dev)
    freq, pres = np.float32([1e-4, 2e-4, 0.5]), np.float32([0.25])
    out = process_logits(_t(x, dev), ft[:, :, 5].t(), frequency=_t(freq, dev), presence=_t(pres, dev))
    check(out, *plain(x, frames[:, :, 5].T, freq=freq, pres=pres))
    assert torch.equal(ft, _t(frames, dev))


def test_long_history_of_one_token(dev):
    """70000 times the same token: counts have more than 16 bits."""
    from estudiocanciones_amd.kernels import process_logits
    x = randn16(1, 1, 100)
    hist = np.full((1, 70000), 42, np.int64)
    freq = np.float32([2.0 ** -10])
    check(process_logits(_t(x, dev), _t(hist, dev), frequency=_t(freq, dev)), *plain(x, hist, freq=freq))


@pytest.mark.parametrize("V", [100, 8197])
def test_strides_and_in_place(dev, V):
    """Logits, bias and out as parts of wider tensors at odd places; a result over its own logits, guided and not."""
    import torch
    from estudiocanciones_amd.kernels import process_logits
    g = rng(V)
    N = 3
    wide = _t(randn16(V, 2 * N, V + 11, std=3.0), dev)
    lg = wide[:, 5:5 + V]
    bw = _t(g.standard_normal((N, V + 7)).astype(np.float32), dev)
    hist = _t(g.integers(0, V, (N, 50)), dev)
    rep = _t(np.float32([1.1, 1.2, 1.3]), dev)
    for cfg in (None, 1.5):
        src = lg if cfg else lg[:N]
        kw = dict(hist=hist, repetition=rep, bias=bw[:, 3:3 + V], cfg=cfg)
        want = process_logits(src, **kw)
        check(want, *plain(src.cpu().numpy(), hist.cpu().numpy(), rep=rep.cpu().numpy(), bias=bw[:, 3:3 + V].cpu().numpy(), cfg=cfg))
        room = torch.full((N + 2, V + 9), 7.0, device=dev, dtype=torch.float16)
        process_logits(src, **kw, out=room[1:N + 1, 3:3 + V])
        assert torch.equal(room[1:N + 1, 3:3 + V], want)
        room[1:N + 1, 3:3 + V] = 7.0
        assert (room == 7.0).all()
        own = wide.clone()
        process_logits(own[:src.shape[0], 5:5 + V], **kw, out=own[:N, 5:5 + V])
        assert torch.equal(own[:N, 5:5 + V], want)
        own[:N, 5:5 + V] = lg[:N]
        assert torch.equal(own, wide)


def test_graph_replays_follow_the_device(dev):
    """A captured call reads the history's length, the penalties, states and masks anew at each replay."""
    import torch
    from estudiocanciones_amd.kernels import process_logits
    g = rng(9)
    N, V, T = 4, 8197, 128
    x = _t(randn16(9, 2 * N, V, std=3.0), dev)
    hist = _t(g.integers(0, V, (N, T)), dev)
    length = torch.zeros(N, device=dev, dtype=torch.int64)
    rep = torch.full((N,), 1.2, device=dev)
    keep = g.random((3, V)) < 0.9
    allowed = _t(words(keep), dev)
    state = torch.zeros(N, device=dev, dtype=torch.int32)
    call = lambda: process_logits(x, hist, length, repetition=rep, allowed=allowed, state=state, cfg=1.5)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call()
    for i in range(4):
        length.fill_(i * 40)
        rep.fill_(1.0 + i / 8)
        state.fill_(i - 1)
        hist.copy_(_t(g.integers(0, V, (N, T)), dev))
        gr.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        check(out, *plain(x.cpu().numpy(), hist.cpu().numpy(), length.cpu().numpy(), rep=rep.cpu().numpy(), keep=keep,
                          state=state.cpu().numpy(), cfg=1.5))


def test_sampled_tokens_are_allowed(dev):
    """A head's logits, processed, then sampled: no token that the mask forbids, and a heavy penalty moves the choice."""
    import torch
    from estudiocanciones_amd.kernels import process_logits, sample_topk
    g = rng(3)
    N, V = 4, 8197
    x = _t(randn16(3, N, V), dev)
    keep = g.random((1, V)) < 0.01
    out = process_logits(x, allowed=_t(words(keep), dev))
    tok = torch.empty(N, 1, device=dev, dtype=torch.int64)
    seed = torch.tensor([5], device=dev)
    for p in range(20):
        sample_topk(out, N, 1.0, 1.0, 200, tok[:, 0], seed=seed, pos=torch.tensor([p], device=dev))
        assert keep[0][tok[:, 0].cpu().numpy()].all()
    best = x.float().argmax(1)
    out = process_logits(x, best[:, None].contiguous(), presence=torch.full((1,), 100.0, device=dev))
    assert (out.float().argmax(1) != best).all()


def test_no_rows(dev):
    import torch
    from estudiocanciones_amd.kernels import process_logits
    assert process_logits(torch.empty(0, 10, device=dev, dtype=torch.float16)).shape == (0, 10)


def test_refusals(dev):
    import torch
    from estudiocanciones_amd.kernels import process_logits
    N, V = 4, 100
    x = torch.zeros(N, V, device=dev, dtype=torch.float16)
    hist = torch.zeros(N, 9, device=dev, dtype=torch.int64)
    one = torch.ones(1, device=dev)
    mask = torch.zeros(N, 4, device=dev, dtype=torch.int32)
    for err, call in [
        (TypeError, lambda: process_logits(x.float())),
        (RuntimeError, lambda: process_logits(x.cpu())),
        (ValueError, lambda: process_logits(x[0])),
        (ValueError, lambda: process_logits(x[:, ::2])),
        (ValueError, lambda: process_logits(x[:3], cfg=1.5)),                      # an odd number of rows
        (ValueError, lambda: process_logits(x, repetition=one)),                   # no history
        (ValueError, lambda: process_logits(x, length=torch.zeros(N, device=dev, dtype=torch.int64))),
        (ValueError, lambda: process_logits(x, window=5)),
        (ValueError, lambda: process_logits(x, hist.int(), repetition=one)),
        (ValueError, lambda: process_logits(x, hist[:3], repetition=one)),
        (ValueError, lambda: process_logits(x, hist.cpu(), repetition=one)),
        (ValueError, lambda: process_logits(x, hist, window=-1)),
        (TypeError, lambda: process_logits(x, hist, torch.zeros(N, device=dev, dtype=torch.int32), repetition=one)),
        (ValueError, lambda: process_logits(x, hist, repetition=torch.ones(2, device=dev))),
        (ValueError, lambda: process_logits(x, hist, presence=one.half())),
        (ValueError, lambda: process_logits(x, hist, frequency=one.cpu())),
        (ValueError, lambda: process_logits(x, bias=torch.zeros(99, device=dev))),
        (ValueError, lambda: process_logits(x, bias=torch.zeros(N, V, device=dev, dtype=torch.float16))),
        (ValueError, lambda: process_logits(x, bias=torch.zeros(V, N, device=dev).t())),
        (ValueError, lambda: process_logits(x, allowed=mask[:2])),                 # two masks for four rows, no state
        (ValueError, lambda: process_logits(x, allowed=mask[:, :3])),
        (TypeError, lambda: process_logits(x, allowed=mask.long())),
        (ValueError, lambda: process_logits(x, state=torch.zeros(N, device=dev, dtype=torch.int32))),
        (TypeError, lambda: process_logits(x, allowed=mask, state=torch.zeros(N, device=dev, dtype=torch.int64))),
        (ValueError, lambda: process_logits(x, out=torch.empty(N, V - 1, device=dev, dtype=torch.float16))),
        (ValueError, lambda: process_logits(x, out=torch.empty(N, V, device=dev))),
    ]:
        with pytest.raises(err):
            call()
