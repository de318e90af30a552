"""Rules for logits that generate() refuses: host logic."""
import pytest
import torch


@pytest.mark.parametrize("kw", [dict(repetition=1e-50), dict(repetition=1e50), dict(repetition=1e-38), dict(presence=1e39),
                                dict(presence=-1e38), dict(frequency=1e50), dict(bias=3e38), dict(bias=-3e38)])
def test_rules_that_would_leave_32_bits_are_refused(kw):
    """Factors and terms up to 2^100 either way, whose sums over any history stay in fp32's range."""
    from estudiocanciones_amd.engine import AUDIO_VOCAB, N_CB, HeartMuLaLite
    d = dict(repetition=1.0, presence=0.0, frequency=0.0, window=0, bias=None, allowed=None)
    for v in (2.0 ** 100, 2.0 ** -100):
        HeartMuLaLite._check_rules(**{**d, "repetition": v, "presence": v, "frequency": -v, "bias": torch.full((N_CB, AUDIO_VOCAB), -v)})
    if "bias" in kw:
        kw = {"bias": torch.zeros(N_CB, AUDIO_VOCAB).index_fill_(1, torch.tensor([9]), kw["bias"])}
    with pytest.raises(ValueError):
        HeartMuLaLite._check_rules(**{**d, **kw})
