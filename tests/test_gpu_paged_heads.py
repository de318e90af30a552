"""The paged cache and the int8 prompt in the engine over other heads than one prompt kernel takes: head_dim 64 and 256, and
more than four query heads per kv head (whose prompt attention runs a row per workgroup)."""
import numpy as np
import pytest

from helpers import assert_close16, model_weights_np, rng, tiny_cfgs, to_torch
from test_gpu_paged_song import N_CB, _frames, _prompt_np

pytestmark = pytest.mark.gpu

HEADS = [(4, 2, 256), (4, 1, 256), (6, 1, 384), (8, 1, 512),   # head_dim 64
         (6, 1, 768), (8, 1, 1024),                            # 128
         (1, 1, 256), (2, 1, 512), (4, 1, 1024), (6, 1, 1536)]  # 256


def _model(dev, heads, kv, dim):
    from estudiocanciones_amd.engine import HeartMuLaLite
    bb, dec = tiny_cfgs()
    bb.update(heads=heads, kv_heads=kv, dim=dim)
    wn = model_weights_np(bb, dec, seed=4)
    return HeartMuLaLite(to_torch(wn, dev), device=dev, backbone=bb, decoder=dec), wn


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("n,P", [(3, 70), (1, 9)])
def test_logits_of_shared_and_dense_caches(dev, heads, kv, dim, n, P):
    """(Caches of at most 128 slots: dense attention of head_dim 64 is for those.)"""
    import torch
    gm, _ = _model(dev, heads, kv, dim)
    text = torch.from_numpy(rng(9).integers(0, 64, P).astype(np.int64))
    want = _frames(gm, dev, text, n, 3, False)
    got = _frames(gm, dev, text, n, 3, True)
    assert gm.backbone.paged.error() == 0
    for i, (a, b) in enumerate(zip(got, want)):
        assert_close16(a, b, what=f"frame {i // N_CB} head {i % N_CB}")


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("paged", [False, True])
def test_prompt_on_int8_activations(dev, heads, kv, dim, paged):
    """Against float64 with the same quantisation; the bound is derived beside the test of the same name of two heads on one,
    from the codes that a step of fp16 moves, whatever the widths."""
    import torch
    P = 70
    gm, wn = _model(dev, heads, kv, dim)
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
    want = _prompt_np(wn, h[[0, 2]].reshape(2 * P, -1).cpu().double(), P, heads, kv).reshape(2, P, -1)[:, -1]
    for b in range(4):
        d = got[b].cpu().double() - want[b // 2]
        assert d.norm() <= 0.05 * want[b // 2].norm(), (b, float(d.norm() / want[b // 2].norm()))


def test_prompt_attention_by_rows_in_several_launches(dev):
    """70000 rows: 700 sequences of 100 rows, and one of 70000 at the positions of a short cache, against float64."""
    import torch
    gm, _ = _model(dev, 6, 1, 768)
    b = gm.backbone.blocks[0]
    g = torch.Generator(device=dev).manual_seed(3)
    for B, S, L in ((700, 100, 100), (1, 70000, 96)):
        q = torch.randn(B * S, 768, generator=g, device=dev, dtype=torch.float16)
        kc, vc = (torch.randn(B, 1, L, 128, generator=g, device=dev, dtype=torch.float16) for _ in range(2))
        pos = (torch.arange(B * S, device=dev) * 7 % L).contiguous()
        got = gm.backbone._prompt_attn(b, q, kc, vc, pos, S)
        pick = torch.tensor(sorted({0, 1, 65534, 65535, 65536, 65499, 65500, 65599, 69999, 40321}), device=dev)
        seq = pick // S
        k, v = kc[seq, 0].double(), vc[seq, 0].double()
        s = (q[pick].double().view(-1, 6, 128) @ k.mT.contiguous()) / 128 ** 0.5
        s = s.masked_fill((torch.arange(L, device=dev) > pos[pick, None])[:, None], float("-inf"))
        want = (s.softmax(-1) @ v).reshape(len(pick), -1)
        # one fp16 rounding of the weights and one of the result, 2^-11 of the values' size (at most 5.5) each
        assert ((got[pick].double() - want).abs() <= 2 * 2.0 ** -11 * float(v.abs().max())).all()
        assert torch.isfinite(got).all()
