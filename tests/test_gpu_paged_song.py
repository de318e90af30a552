"""The paged cache in the engine: the prompt computed once, forked for the takes, decoded with shared attention, and the
prompt pass on int8 activations."""
import numpy as np
import pytest

from helpers import AUDIO_VOCAB, N_CB, assert_close16, model_weights_np, rng, tiny_cfgs, to_torch

pytestmark = pytest.mark.gpu


def _model(dev, seed=4):
    from estudiocanciones_amd.engine import HeartMuLaLite
    bb, dec = tiny_cfgs()
    wn = model_weights_np(bb, dec, seed=seed)
    return HeartMuLaLite(to_torch(wn, dev), device=dev, backbone=bb, decoder=dec), wn


def _frames(gm, dev, text, n, steps, paged, cfg=1.5):
    """Teacher-forced logits of the prompt's frame and of ``steps`` frames, by the calls that generate() makes."""
    import torch
    P = text.numel()
    gm.alloc(n, P + steps + 2, cfg, seed=1, paged=P if paged else None)
    g = rng(3)
    forced = torch.from_numpy(g.integers(0, AUDIO_VOCAB, (steps + 1, gm.B, N_CB)).astype(np.int64)).to(dev)
    if gm.B == 2 * n:
        forced[:, n:] = forced[:, :n]
    if paged:
        hb = gm._prompt_shared(text, 3)
    else:
        h = gm.text_emb(text.to(dev)).unsqueeze(0).repeat(gm.B, 1, 1)
        h[:n, 3] = gm.muq_b
        if gm.B == 2 * n:
            h[n:] = gm.uncond[0]
        hb = gm.backbone(h, torch.arange(P, device=dev).unsqueeze(0).expand(gm.B, P))[:, -1]
    out = []
    gm._frame_fast(hb.contiguous(), cfg, 50, 1.0, forced=forced[0], logits_out=out)
    for i in range(steps):
        pos = torch.full((gm.B, 1), P + i, dtype=torch.long, device=dev)
        gm._step(forced[i], pos, None, cfg, 50, 1.0, forced=forced[i + 1], logits_out=out)
    return [o.float().cpu().numpy() for o in out]


@pytest.mark.parametrize("n,cfg,P,steps", [(1, 1.0, 5, 3), (3, 1.5, 70, 61), (2, 1.5, 128, 3), (10, 1.5, 100, 4), (70, 1.5, 40, 2)])
def test_logits_of_shared_and_dense_caches(dev, n, cfg, P, steps):
    """Prompts within a page, that end in one and on a border; a step that takes a new page; more than 16 rows."""
    import torch
    gm, _ = _model(dev)
    text = torch.from_numpy(rng(9).integers(0, 64, P).astype(np.int64))
    want = _frames(gm, dev, text, n, steps, False, cfg)
    gm.release()
    got = _frames(gm, dev, text, n, steps, True, cfg)
    for i, (a, b) in enumerate(zip(got, want)):
        assert_close16(a, b, what=f"frame {i // N_CB} head {i % N_CB}")
    cache = gm.backbone.paged
    assert cache.error() == 0 and cache.length.tolist() == [P + steps] * gm.B
    page = cache.page
    ref, table = cache.ref.tolist(), cache.table.tolist()
    whole = P // page
    for b in range(gm.B):
        first = b - b % n
        assert table[b][:whole] == table[first][:whole] and all(ref[p] == n for p in table[b][:whole])
        own = table[b][whole:-(-(P + steps) // page)]
        assert all(ref[p] == 1 for p in own)
    assert sum(r > 0 for r in ref) == gm.B // n * whole + gm.B * (-(-(P + steps) // page) - whole)


def test_a_prompt_kept_and_compacted_goes_on_the_same(dev):
    """Takes freed and forked again from a kept prompt, and the cache moved to a smaller pool, give the same step."""
    import torch
    gm, _ = _model(dev)
    text = torch.from_numpy(rng(9).integers(0, 64, 70).astype(np.int64))
    gm.alloc(3, 200, 1.0, seed=1, paged=70)
    gm._prompt_shared(text, 3)
    cache = gm.backbone.paged
    tok = torch.from_numpy(rng(5).integers(0, AUDIO_VOCAB, (3, N_CB)).astype(np.int64)).to(dev)
    x = gm.audio_emb.sum_codebooks(tok, AUDIO_VOCAB)
    pos = torch.full((3,), 70, dtype=torch.long, device=dev)
    first = gm.backbone.decode_paged(x, pos).clone()
    for p in range(71, 131):
        gm.backbone.decode_paged(x, pos.new_full((3,), p))
    cache.free([1, 2])
    cache.free(torch.tensor([2, 1], dtype=torch.int32, device=dev))
    # sequence 0 went on: its prompt is no longer at its end, so the takes start again from a fork of a kept copy
    gm.backbone.free()
    gm.alloc(3, 200, 1.0, seed=1, paged=70)
    gm._prompt_shared(text, 3)
    cache = gm.backbone.paged
    gm.backbone.decode_paged(x, torch.tensor([-1, 70, 70], device=dev))
    cache.free([1, 2])
    cache.fork([0, 0], [2, 1])
    small = cache.compact(9)
    assert cache.error() == 0 and small.ref.sum() == cache.ref.sum()
    gm.backbone.paged = small
    again = gm.backbone.decode_paged(x, pos)
    assert small.error() == 0
    assert torch.equal(again, first)


def test_generate_shared_graph_equals_eager(dev):
    """Sampled songs over the paged cache: the captured loop and the eager one give the same tokens, twice."""
    import torch
    gm, _ = _model(dev)
    text = rng(9).integers(0, 64, 70)
    kw = dict(max_ms=80 * 70, seed=5, n=3, paged=True)
    a = gm.generate(text, 3, **kw)
    b = gm.generate(text, 3, use_graphs=False, **kw)
    c = gm.generate(text, 3, **kw)
    assert gm.backbone.paged is None  # released
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z) and x.shape[0] == N_CB
    one = gm.generate(text, 3, max_ms=800, seed=5, paged=True, cfg_scale=1.0)
    assert one.shape[0] == N_CB


@pytest.mark.parametrize("paged", [True, False])
def test_a_song_after_one_that_broke_off(dev, paged):
    """A callback that raises leaves a captured frame and caches behind: the next song does not run on them."""
    import torch
    gm, _ = _model(dev)
    text = rng(9).integers(0, 64, 40)
    forced = torch.from_numpy(rng(12).integers(0, 8193, (61, 4, N_CB)).astype(np.int64)).to(dev)
    kw = dict(max_ms=80 * 60, seed=5, n=2, paged=paged)
    want = gm.generate(text, 3, **kw)

    def stop(*_):
        raise KeyboardInterrupt

    with pytest.raises(KeyboardInterrupt):
        gm.generate(text, 3, progress=stop, forced=forced, **kw)
    kept = torch.zeros(64 << 20, dtype=torch.uint8, device=dev)  # what may lie where the old caches were
    for x, y in zip(gm.generate(text, 3, **kw), want):
        assert torch.equal(x, y)
    assert not kept.any()


def test_caches_of_the_two_kinds_replace_each_other(dev):
    """A model that is allocated anew, without release, runs on the new cache."""
    import torch
    gm, _ = _model(dev)
    text = torch.from_numpy(rng(9).integers(0, 64, 20).astype(np.int64))
    dense = _frames(gm, dev, text, 2, 2, False)
    assert gm.backbone.paged is None
    paged = _frames(gm, dev, text, 2, 2, True)
    assert gm.backbone.blocks[0].kc is None and gm.backbone.tail is None
    again = _frames(gm, dev, text, 2, 2, False)
    assert gm.backbone.paged is None
    for a, b, c in zip(dense, paged, again):
        assert np.array_equal(a, c)
        assert_close16(b, a, what="paged")


def test_int8_activations_need_packed_weights(dev):
    gm, _ = _model(dev)
    gm.backbone.blocks[1].w2.qp = None
    with pytest.raises(NotImplementedError, match="packed"):
        gm.generate([1, 2, 3], 1, max_ms=160, a8=True)
    with pytest.raises(NotImplementedError, match="packed"):
        gm.generate([1, 2, 3], 1, max_ms=160, paged=True)


def test_generate_stops_when_the_cache_refuses(dev):
    """A pool with too few pages: the song stops with RuntimeError, and the next one runs."""
    import torch
    gm, _ = _model(dev)
    text = rng(9).integers(0, 64, 70)
    alloc = type(gm.backbone).alloc_paged
    # 6 pages hold the two prompts and the takes' own parts; at slot 128 (frame 58) all four sequences need one more
    few = lambda seqs, pages, *a: alloc(gm.backbone, seqs, 8, *a)  # noqa: E731
    gm.backbone.alloc_paged = few
    forced = torch.from_numpy(rng(12).integers(0, 8193, (101, 4, N_CB)).astype(np.int64)).to(dev)  # no take ends
    with pytest.raises(RuntimeError, match="refused"):
        gm.generate(text, 3, max_ms=80 * 100, seed=5, n=2, paged=True, forced=forced)
    del gm.backbone.alloc_paged
    assert gm.backbone.paged is None
    assert len(gm.generate(text, 3, max_ms=800, seed=5, n=2, paged=True)) == 2


def _f16(w):
    """bf16 bit patterns as the fp16 values that the engine loads, in float64."""
    import torch
    return torch.from_numpy(w.astype(np.int16)).view(torch.bfloat16).to(torch.float16).double()


def _prompt_np(wn, x, S, heads, kv, eps=1e-5):
    """The prompt pass on int8 activations in float64, rounded to fp16 where the engine's tensors are."""
    import torch
    from oracle.rope import rope_cache
    r16 = lambda t: t.to(torch.float16).double()  # noqa: E731

    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w

    def lin(t, name):
        top = t.abs().amax(-1, keepdim=True)
        c = torch.round(t * 127 / top)
        return (c @ torch.from_numpy(wn[name + ".q8"]).double().T) * (top / 127) * _f16(wn[name + ".s8"])

    R, D = x.shape
    hd = D // heads
    rope = torch.from_numpy(np.asarray(rope_cache(hd, S), np.float64))
    for i in range(2):
        p = f"backbone.layers.{i}."
        y = norm(x, _f16(wn[p + "sa_norm.scale"]))
        q, k, v = (r16(lin(y, p + f"attn.{n}_proj.weight")).reshape(R // S, S, -1, hd) for n in "qkv")

        def turn(t):
            a, b = t[..., 0::2], t[..., 1::2]
            c, s = rope[None, :, None, :, 0], rope[None, :, None, :, 1]
            return r16(torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2))

        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(heads // kv, 2) for t in (k, v))
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / hd ** 0.5
        s = s.masked_fill(torch.ones(S, S, dtype=torch.bool).triu(1), float("-inf"))
        o = r16(torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).reshape(R, D))
        x = r16(lin(o, p + "attn.output_proj.weight") + x)
        y = norm(x, _f16(wn[p + "mlp_norm.scale"]))
        mm = r16(torch.nn.functional.silu(lin(y, p + "mlp.w1.weight")) * lin(y, p + "mlp.w3.weight"))
        x = r16(lin(mm, p + "mlp.w2.weight") + x)
    return norm(x, _f16(wn["backbone.norm.scale"]))


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("P", [9, 100])
def test_prompt_on_int8_activations(dev, paged, P):
    """Against float64 with the same quantisation.  What the two may differ by: values of the attention and of the norms off
    by one fp16 step or less (2^-11) move at most 127 2^-11 2 = 12% of the codes by one, of an rms of about 30: 1.2% of a
    product's norm at worst, in 8 products of which 6 feed a residual stream that is larger than they are: 5%."""
    import torch
    gm, wn = _model(dev)
    text = torch.from_numpy(rng(9).integers(0, 64, P).astype(np.int64))
    gm.alloc(2, P + 4, 1.5, seed=1, paged=P if paged else None)
    gm.backbone.prompt_a8 = True
    h = gm.text_emb(text.to(dev)).unsqueeze(0).repeat(gm.B, 1, 1)
    h[:2, 3] = gm.muq_b
    h[2:] = gm.uncond[0]
    if paged:
        got = gm._prompt_shared(text, 3)
    else:
        got = gm.backbone(h, torch.arange(P, device=dev).unsqueeze(0).expand(gm.B, P))[:, -1]
    want = _prompt_np(wn, h[[0, 2]].reshape(2 * P, -1).cpu().double(), P, 2, 1).reshape(2, P, -1)[:, -1]
    for b in range(4):
        d = got[b].cpu().double() - want[b // 2]
        assert d.norm() <= 0.05 * want[b // 2].norm(), (b, float(d.norm() / want[b // 2].norm()))


def test_generate_on_int8_activations(dev):
    import torch
    gm, _ = _model(dev)
    text = rng(9).integers(0, 64, 40)
    a = gm.generate(text, 3, max_ms=800, seed=5, n=2, paged=True, a8=True)
    assert not gm.backbone.prompt_a8
    b = gm.generate(text, 3, max_ms=800, seed=5, n=2, paged=True, a8=True)
    c = gm.generate(text, 3, max_ms=800, seed=5, n=2, a8=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and len(c) == 2


def test_the_parts_together(dev):
    """A layer by its kernels, as a host with a loop of its own would call them: int8 projection, the write into pages,
    forks, a step for every take, attention, freeing."""
    import torch
    from estudiocanciones_amd.kernels import (gemm_a8_packed, pack_i8, paged_attn, paged_attn_plan, paged_write, quant_a8)
    from estudiocanciones_amd.paged import PagedCache
    g = rng(8)
    D, Hq, Hk, HD, P, takes = 256, 6, 2, 64, 45, 5
    N = (Hq + 2 * Hk) * HD
    w = np.clip(np.rint(g.standard_normal((N, D)) * 40), -127, 127).astype(np.int8)
    s = (0.002 * (1 + g.random(N))).astype(np.float16)
    wp, sd = pack_i8(torch.from_numpy(w).to(dev)), torch.from_numpy(s).to(dev)
    x = torch.from_numpy(g.standard_normal((P + takes, D)).astype(np.float16)).to(dev)
    cache = PagedCache(1, takes, 12, Hk, HD, max_pages=8, page=16, device=dev)
    kp, vp = cache.layer(0)
    c, sx = quant_a8(x)
    qkv = gemm_a8_packed(c, sx, wp, sd, N, D)
    start = torch.full((takes,), -1, dtype=torch.long, device=dev)
    start[0] = P - 1
    cache.extend(start)
    paged_write(qkv[:P], kp, vp, cache.table[:1], torch.arange(P, device=dev), P, Hq, Hk)
    cache.fork([0] * (takes - 1), range(1, takes))
    pos = torch.full((takes,), P, dtype=torch.long, device=dev)
    cache.extend(pos)
    step = qkv[P:].contiguous()
    paged_write(step, kp, vp, cache.table, pos, 1, Hq, Hk)
    plan = paged_attn_plan([(takes, P)], Hq, Hk, HD, 128, dev)
    o = paged_attn(step[:, :Hq * HD], kp, vp, cache.table, pos, plan).cpu().double()
    assert cache.error() == 0
    # the same in float64, on the fp16 projections
    y = qkv.cpu().double().reshape(-1, Hq + 2 * Hk, HD)
    for t in range(takes):
        rows = list(range(P)) + [P + t]
        for h in range(Hq):
            k, v = y[rows, Hq + h // 3], y[rows, Hq + Hk + h // 3]
            want = (k @ y[P + t, h] / HD ** 0.5).softmax(0) @ v
            # probabilities to fp16, the scores' fp32 sums, one rounding: as in test_gpu_paged_attn.py
            ds = (HD + 8) * 2.0 ** -24 * float((k.abs() @ y[P + t, h].abs()).max()) / HD ** 0.5
            tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * ds + 2.0 ** -20) * v.abs().amax() + 2.0 ** -20
            assert ((o[t, h * HD:(h + 1) * HD] - want).abs() <= tol).all()
    cache.free(range(takes))
    assert cache.ref.sum() == 0 and (cache.table == -1).all()
