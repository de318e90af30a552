"""A backbone of 4-bit weights in the engine: the stack's paths against a float64 restatement, songs over dense and paged
caches, the converter's --int4; and generate()'s rules for logits (penalties, biases, masks, a shortest length)."""
import numpy as np
import pytest

from helpers import AUDIO_VOCAB, N_CB, assert_close16, model_weights_np, randn16, tiny_cfgs, to_torch

pytestmark = pytest.mark.gpu


def dequant(w, name, group):
    """float64 values of a 4-bit layer of an engine's weights."""
    q, s = w[name + ".q4"].cpu().numpy(), w[name + ".s4"].cpu().numpy().astype(np.float64)
    u = np.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1).astype(np.float64)
    z = np.repeat(w[name + ".z4"].cpu().numpy().astype(np.float64), group, 1)[:, :u.shape[1]] if name + ".z4" in w else 8.0
    return (u - z) * np.repeat(s, group, 1)[:, :u.shape[1]]


class Plain:
    """The stack's layers over growing caches in float64, row r a batch item."""

    def __init__(self, w, cfg, group, B):
        self.w = {k[:-3]: dequant(w, k[:-3], group) for k in w if k.startswith("backbone.") and k.endswith(".q4")}
        self.n = {k: v.float().half().cpu().numpy().astype(np.float64) for k, v in w.items() if k.startswith("backbone.") and k.endswith(".scale")}
        self.cfg, self.B = cfg, B
        self.k = [[[] for _ in range(B)] for _ in range(cfg["layers"])]
        self.v = [[[] for _ in range(B)] for _ in range(cfg["layers"])]

    def rms(self, x, n):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * self.n[n]

    def step(self, x, pos, rope):
        D, Hq, Hk = self.cfg["dim"], self.cfg["heads"], self.cfg["kv_heads"]
        hd = D // Hq
        c, s = rope[pos, :, 0], rope[pos, :, 1]

        def turn(t):
            a, b = t[..., 0::2], t[..., 1::2]
            return np.stack([a * c - b * s, b * c + a * s], -1).reshape(t.shape)

        for i in range(self.cfg["layers"]):
            p = f"backbone.layers.{i}."
            y = self.rms(x, p + "sa_norm.scale")
            q, k, v = (y @ self.w[p + f"attn.{n}_proj.weight"].T for n in "qkv")
            o = np.zeros((self.B, Hq * hd))
            for b in range(self.B):
                self.k[i][b].append(turn(k[b].reshape(Hk, hd)))
                self.v[i][b].append(v[b].reshape(Hk, hd))
                K, V = np.stack(self.k[i][b]), np.stack(self.v[i][b])
                qb = turn(q[b].reshape(Hq, hd))
                for h in range(Hq):
                    kh = h // (Hq // Hk)
                    sc = K[:, kh] @ qb[h] / np.sqrt(hd)
                    e = np.exp(sc - sc.max())
                    o[b, h * hd:(h + 1) * hd] = e / e.sum() @ V[:, kh]
            x = x + o @ self.w[p + "attn.output_proj.weight"].T
            y = self.rms(x, p + "mlp_norm.scale")
            a, g = y @ self.w[p + "mlp.w1.weight"].T, y @ self.w[p + "mlp.w3.weight"].T
            x = x + (a / (1 + np.exp(-a)) * g) @ self.w[p + "mlp.w2.weight"].T
        return self.rms(x, "backbone.norm.scale")


def model(dev, group=64, zeros=False, stacks=("backbone",), seed=0):
    from estudiocanciones_amd.engine import HeartMuLaLite
    from estudiocanciones_amd.quant import to_q4
    bb, dec = tiny_cfgs()
    w = to_torch(model_weights_np(bb, dec, seed=seed), dev)
    for st in stacks:
        w = to_q4(w, group, zeros, dev, st)
    return w, bb, HeartMuLaLite(w, device=dev, backbone=bb, decoder=dec)


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_stack_against_float64(dev, group, zeros):
    """Steps over dense and over paged caches, and the same rows as one prompt (few and many), against float64."""
    import torch
    w, bb, m = model(dev, group, zeros)
    st = m.backbone
    assert st.four() and st.packed() and not st.eight()
    B, S = 2, 40
    D = bb["dim"]
    x = randn16(1, S, B, D)
    st.alloc(B, 160, dev, torch.float16)
    rope = st.rope.double().cpu().numpy()
    plain = Plain(w, bb, group, B)
    want = np.stack([plain.step(x[t].astype(np.float64), t, rope) for t in range(S)])
    xt = torch.from_numpy(x).to(dev)
    at = lambda t: torch.full((B,), t, dtype=torch.int64, device=dev)  # noqa: E731
    for t in range(S):
        assert_close16(st.decode(xt[t], at(t), 1).cpu().numpy(), want[t], what=f"step {t}")
    for n in (20, S):  # 40 rows through the decode path, 80 through the prompt's
        st.alloc(B, 160, dev, torch.float16)
        pos = torch.arange(n, device=dev).expand(B, n)
        h = st(xt[:n].transpose(0, 1).contiguous(), pos)
        assert_close16(h.transpose(0, 1).cpu().numpy(), want[:n], what=f"prompt of {n}")
        y = st.decode(xt[n - 1], at(n - 1), 1, final_norm=False)  # its last slot again
        assert_close16(torch.nn.functional.rms_norm(y.float(), (D,), st.norm.float(), 1e-5).cpu().numpy(), want[n - 1])
    with pytest.raises(NotImplementedError):
        st.decode(xt[0], at(0), 1, o0=y)
    with pytest.raises(NotImplementedError):
        st.decode_reference(xt[0], at(0), 1)
    st.alloc_paged(B, 8, 4, dev, [(B, 0)])
    h = st.prompt_paged(xt[:30].transpose(0, 1).contiguous(), torch.arange(B, device=dev))
    assert_close16(h.cpu().numpy(), want[29], what="paged prompt")
    for t in range(30, S):
        assert_close16(st.decode_paged(xt[t], at(t)).cpu().numpy(), want[t], what=f"paged step {t}")
    assert int(st.paged.err.item()) == 0


@pytest.mark.parametrize("stacks", [("backbone",), ("decoder",), ("backbone", "decoder")])
@pytest.mark.parametrize("paged", [False, True])
def test_songs(dev, stacks, paged):
    """A song on 4-bit weights: graph replays and eager steps choose the same codes; both stacks may be in 4 bits."""
    import torch
    _, _, m = model(dev, 128, True, stacks)
    text = torch.arange(1, 13)
    kw = dict(max_ms=1600, seed=5, n=2, paged=paged, cfg_scale=1.5, topk=20)
    a = m.generate(text, 3, **kw)
    b = m.generate(text, 3, **kw, use_graphs=False)
    for x, y in zip(a, b):
        assert x.shape[0] == N_CB and torch.equal(x, y)
        assert ((x >= 0) & (x < AUDIO_VOCAB)).all()
    with pytest.raises(NotImplementedError):
        if "backbone" in stacks:
            m.generate(text, 3, a8=True, **kw)
        else:
            raise NotImplementedError


def test_converted_checkpoint(dev, tmp_path):
    """--int4 stores the backbone's linear layers as q4_rows of the fp32 weights; the engine loads the file."""
    import json

    import torch
    from safetensors import safe_open
    from safetensors.torch import save_file
    from estudiocanciones_amd.convert import convert_file
    from estudiocanciones_amd.engine import HeartMuLaLite
    from estudiocanciones_amd.quant import q4_rows, weight_shapes
    bb, dec = tiny_cfgs()
    lin, dense = weight_shapes(bb, dec, 64)
    g = torch.Generator().manual_seed(4)
    ck = {k: torch.randn(*s, generator=g) * 0.02 for k, s in lin.items() if not k.startswith("audio_head.")}
    ck["audio_head"] = torch.randn(N_CB - 1, dec["dim"], AUDIO_VOCAB, generator=g) * 0.02
    ck.update({k: torch.ones(s) if k.endswith(".scale") else torch.randn(*s, generator=g) for k, s in dense.items()})
    save_file(ck, str(tmp_path / "a.safetensors"))
    convert_file(tmp_path / "a.safetensors", tmp_path / "b.safetensors", group=64, zeros=True)
    with safe_open(str(tmp_path / "b.safetensors"), "pt") as f:
        assert json.loads(f.metadata()["lite"]) == {"mode": "int4"}
        four = sorted(k[:-3] for k in f.keys() if k.endswith(".q4"))
        assert four == sorted(k for k in lin if k.startswith("backbone.layers."))
        for k in four:
            q, s, z = q4_rows(ck[k].to(dev), 64, True)
            assert torch.equal(f.get_tensor(k + ".q4"), q.cpu()) and torch.equal(f.get_tensor(k + ".z4"), z.cpu())
            assert torch.equal(f.get_tensor(k + ".s4"), s.cpu())
        assert "decoder.layers.0.mlp.w1.weight.q8" in f.keys() and "codebook0_head.weight.q8" in f.keys()
    m = HeartMuLaLite(str(tmp_path / "b.safetensors"), device=dev, backbone=bb, decoder=dec)
    assert m.backbone.four() and m.decoder.eight()
    assert m.generate(torch.arange(1, 9), 2, max_ms=800, seed=1, topk=10).shape[0] == N_CB


def test_layers_that_do_not_fit_together(dev):
    import torch
    from estudiocanciones_amd.engine import Linear, fuse
    from estudiocanciones_amd.quant import q4_rows, q8_rows
    t = torch.randn(32, 128, device=dev)
    q8, s8 = q8_rows(t)
    a = Linear(q8=q8, s8=s8.half())
    b, c, d = (Linear(q4=q, s4=s, z4=z) for q, s, z in (q4_rows(t, 64), q4_rows(t, 32), q4_rows(t, 64, True)))
    for parts in ([a, b], [b, c], [b, d]):
        with pytest.raises(ValueError):
            fuse(parts)
    f = fuse([b, b])
    x = torch.randn(3, 128, device=dev).half()
    assert f.N == 64 and torch.equal(f(x), torch.cat([b(x), b(x)], 1))
    with pytest.raises(NotImplementedError):
        Linear()


# ---------------------------------------------------------------- rules for logits
@pytest.fixture(scope="module")
def song(dev):
    import torch
    _, _, m = model(dev)
    text = torch.arange(1, 13)

    def sing(**kw):
        d = dict(max_ms=2400, seed=7, n=2, topk=60, temperature=1.5)
        d.update(kw)
        out = m.generate(text, 3, **d)
        return [t.cpu().numpy() for t in (out if isinstance(out, list) else [out])]

    return sing


@pytest.mark.parametrize("cfg_scale", [1.0, 1.5])
@pytest.mark.parametrize("window", [0, 4])
def test_presence_keeps_codes_from_coming_again(dev, song, cfg_scale, window):
    """A heavy penalty: no codebook repeats a code within the window; without it some do (few codes are allowed)."""
    import torch
    some = torch.zeros(N_CB, AUDIO_VOCAB, dtype=torch.bool)
    some[:, 100:150] = True

    def repeats(codes):
        n = 0
        for row in codes:
            for t in range(len(row)):
                n += row[t] in row[max(0, t - window) if window else 0:t]
        return n

    kw = dict(cfg_scale=cfg_scale, allowed=some, max_ms=2400)
    free, held = song(**kw), song(**kw, presence=3e4, window=window)
    assert all(((c >= 100) & (c < 150)).all() for c in free + held)
    assert sum(map(repeats, free)) > 0 and sum(map(repeats, held)) == 0


def test_rules_in_graphs_and_eager(dev, song):
    import torch
    g = torch.Generator().manual_seed(1)
    kw = dict(repetition=1.3, presence=0.5, frequency=0.2, window=10, bias=torch.randn(N_CB, AUDIO_VOCAB, generator=g),
              allowed=torch.rand(N_CB, AUDIO_VOCAB, generator=g) < 0.8, min_ms=1000)
    a, b = song(**kw), song(**kw, use_graphs=False)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    assert not all(np.array_equal(x, y) for x, y in zip(a, song()))
    c = song(**kw, paged=True)
    assert all(kw["allowed"].numpy()[i][row].all() for t in c for i, row in enumerate(t))


@pytest.mark.parametrize("min_ms", [0, 80, 1000])
def test_shortest_length(dev, song, min_ms):
    """A bias that ends the song at once: it ends in the first frame that may."""
    import torch
    bias = torch.zeros(N_CB, AUDIO_VOCAB)
    bias[:, 8193:] = 200.0
    out = song(bias=bias, min_ms=min_ms)
    frames = max(1, -(-min_ms // 80))  # (the frame of the prompt pass is never scanned for an end)
    assert all(t.shape == (N_CB, frames) for t in out)
    assert all((t[:, 1:] < 8193).all() for t in out)


def test_neutral_rules_change_nothing(dev, song):
    a = song()
    b = song(repetition=1.0, presence=0.0, frequency=0.0, window=5, min_ms=0)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))


def test_rules_refused_before_the_caches_go(dev):
    import torch
    _, _, m = model(dev)
    m.alloc(1, 64)
    kc = m.backbone.blocks[0].kc
    text = torch.arange(1, 5)
    for kw in (dict(repetition=0.0), dict(repetition=float("nan")), dict(presence=float("inf")), dict(frequency=float("nan")),
               dict(window=-1), dict(bias=torch.zeros(AUDIO_VOCAB)), dict(bias=torch.zeros(N_CB, AUDIO_VOCAB, dtype=torch.float64)),
               dict(allowed=torch.ones(N_CB, AUDIO_VOCAB)), dict(allowed=torch.ones(N_CB, 5, dtype=torch.bool))):
        with pytest.raises(ValueError):
            m.generate(text, 1, max_ms=160, **kw)
    assert m.backbone.blocks[0].kc is kc


def test_layer_of_any_input(dev):
    """A single 4-bit layer takes what an 8-bit one takes: leading dimensions, strides, rows that start anywhere."""
    import torch
    from estudiocanciones_amd.engine import Linear
    from estudiocanciones_amd.quant import q4_rows
    N, K = 40, 128
    g = torch.Generator(device=dev).manual_seed(1)
    q, s, z = q4_rows(torch.randn(N, K, generator=g, device=dev), 64, True)
    lin = Linear(q4=q, s4=s, z4=z)
    x = torch.randn(3, 2, K, generator=g, device=dev).half()
    res = torch.randn(3, 2, N, generator=g, device=dev).half()
    want = lin(x.reshape(6, K), res.reshape(6, N))
    assert torch.equal(lin(x, res).reshape(6, N), want)
    wide = torch.zeros(6, K + 5, device=dev, dtype=torch.float16)
    wide[:, 3:K + 3] = x.reshape(6, K)
    assert torch.equal(lin(wide[:, 3:K + 3], res.reshape(6, N)), want)
    assert torch.equal(lin(x.reshape(6, K).t().contiguous().t(), res.reshape(6, N)), want)
    assert torch.equal(lin(x[0, 0]), lin(x.reshape(6, K))[0]) and lin(x[:0]).shape == (0, 2, N)
    q, s, _ = q4_rows(torch.randn(N, K, generator=g, device=dev), 128)
    assert Linear(q4=q, s4=s)(x).shape == (3, 2, N)


def test_a_codebook_with_nothing_to_draw_ends_the_take(dev, song):
    """Penalties that take every allowed logit to -inf: the take ends at that frame, and nothing else happens."""
    import torch
    allowed = torch.zeros(N_CB, AUDIO_VOCAB, dtype=torch.bool)
    allowed[:, 10:13] = True
    for kw in (dict(), dict(use_graphs=False), dict(cfg_scale=1.0)):
        got = song(presence=1e9, allowed=allowed, **kw)
        assert all(1 <= t.shape[1] <= 3 and all(len(set(row.tolist())) == row.size for row in t) for t in got)
        assert all(((t >= 10) & (t < 13)).all() for t in got)

