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
