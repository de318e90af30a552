"""Songs under rules for their logits at the ends of the range: biases that force a code or leave none, from the first frame on."""
import numpy as np
import pytest

from helpers import AUDIO_VOCAB, N_CB
from test_gpu_q4_model import model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def song(dev):
    import torch
    _, _, m = model(dev)
    text = torch.arange(1, 13)

    def sing(**kw):
        d = dict(max_ms=1600, seed=7, n=2, topk=60, temperature=1.5)
        d.update(kw)
        out = m.generate(text, 3, **d)
        return [t.cpu().numpy() for t in (out if isinstance(out, list) else [out])]

    return sing


WAYS = [dict(), dict(use_graphs=False), dict(cfg_scale=1.0), dict(paged=True), dict(n=1)]


@pytest.mark.parametrize("way", range(len(WAYS)))
def test_a_bias_past_the_range_forces_its_code(dev, song, way):
    """+1e5 on one code of every codebook: that code in every frame, and no end before the last."""
    import torch
    bias = torch.zeros(N_CB, AUDIO_VOCAB)
    codes = np.arange(N_CB) * 1000 + 17
    bias[torch.arange(N_CB), torch.from_numpy(codes)] = 1e5
    for t in song(bias=bias, min_ms=400, **WAYS[way]):
        assert t.shape == (N_CB, 1600 // 80 + 1) and (t == codes[:, None]).all()


@pytest.mark.parametrize("way", range(len(WAYS)))
def test_a_first_frame_with_nothing_to_draw_is_a_song_of_no_frames(dev, song, way):
    """A bias that takes every code of a codebook out of fp16's range below: no frame, and no number that is not a code."""
    import torch
    for row in (0, 3, 7):
        bias = torch.zeros(N_CB, AUDIO_VOCAB)
        bias[row] = -1e30
        for t in song(bias=bias, **WAYS[way]):
            assert t.shape == (N_CB, 0)


@pytest.mark.parametrize("use_graphs", [True, False])
def test_a_song_that_may_only_end_later_does_not_start_with_nothing(dev, song, use_graphs):
    """Codes out of the range below but for the end codes, which a shortest length forbids at first: no frames again."""
    import torch
    bias = torch.full((N_CB, AUDIO_VOCAB), -1e30)
    bias[:, 8193:] = 0
    for t in song(bias=bias, min_ms=400, use_graphs=use_graphs):
        assert t.shape == (N_CB, 0)


def test_int8_activations_need_eight_bits_in_the_backbone_alone(dev):
    """A 4-bit decoder beside an int8 backbone sings with int8 activations; a 4-bit backbone refuses them."""
    import torch
    text = torch.arange(1, 13)
    _, _, m = model(dev, 128, True, ("decoder",))
    assert m.backbone.eight() and m.decoder.four()
    for paged in (False, True):
        for t in m.generate(text, 3, max_ms=800, seed=5, n=2, topk=20, a8=True, paged=paged):
            assert t.shape[0] == N_CB and t.shape[1] >= 1 and ((t >= 0) & (t < AUDIO_VOCAB)).all()
    _, _, m = model(dev, 128, True, ("backbone",))
    with pytest.raises(NotImplementedError, match="int8 activations"):
        m.generate(text, 3, max_ms=800, a8=True)


@pytest.mark.parametrize("min_ms,frames", [(80, 1), (80.5, 2), (159.9, 2), (160.25, 3)])
def test_a_shortest_length_between_frames(dev, song, min_ms, frames):
    """A bias towards the end codes: the song ends in the first frame at or past the shortest length."""
    import torch
    bias = torch.zeros(N_CB, AUDIO_VOCAB)
    bias[:, 8193:] = 200.0
    for t in song(bias=bias, min_ms=min_ms):
        assert t.shape == (N_CB, frames) and (t < 8193).all()
