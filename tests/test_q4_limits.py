"""Sizes, layouts and states in which 4-bit calls are taken or refused: host logic."""
import pytest
import torch


def test_blocks_of_few_rows_are_chosen_for_as_many_as_a_launch_takes():
    """The few-row kernel's launch counts 65535 blocks of 16 rows: of more, a product goes by the tiles."""
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    most = 16 * 65535
    few = False
    for N, K in [(8, 1024), (16, 1024), (16, 8192), (48, 192), (250, 64), (1001, 192)]:
        for choice in (lambda M: L.ecd_mm_q4_choice(M, N, K), lambda M: L.ecd_mm_q4_norm_choice(M, N, K, 0),
                       lambda M: L.ecd_mm_q4_norm_choice(M, N, K, 1)):
            few |= bool(choice(most) & 16)
            for M in (most + 1, 1_100_000, 3_000_000):
                p = choice(M)
                assert p > 0 and not p & 16, (M, N, K, p)
    assert few  # (the rule above is what decides)


def linear(N, K, bits):
    from estudiocanciones_amd.engine import Linear
    if bits == 8:
        return Linear(q8=torch.zeros(N, K, dtype=torch.int8), s8=torch.ones(N, dtype=torch.float16))
    return Linear(q4=torch.full((N, K // 2), 0x88, dtype=torch.uint8), s4=torch.ones(N, -(-K // 128), dtype=torch.float16))


def test_a_layer_is_not_laid_out_inside_a_capture(monkeypatch):
    """The layout would run at the replays only, over weights that are gone by then."""
    lin = linear(32, 64, 4)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lin.pack, lambda: lin(torch.zeros(1, 64, dtype=torch.float16))):
        with pytest.raises(RuntimeError, match="captur"):
            call()
    assert lin.q4 is not None and lin.w4 is None


@pytest.mark.parametrize("where", ["layers.1.", "attn.output_proj", "mlp.w2", "mlp.w1", "attn.", None])
def test_a_stack_is_of_4_bits_throughout_or_not_at_all(where):
    from estudiocanciones_amd.engine import Stack
    cfg = dict(layers=2, heads=2, kv_heads=1, max_seq=64, dim=64)

    def p(name, norm=False):
        if norm:
            return torch.ones(64, dtype=torch.float16)
        return linear(64, 64, 8 if where is None or where not in name else 4)

    if where is None:
        assert len(Stack(p, "backbone", cfg).blocks) == 2
    else:
        with pytest.raises(ValueError, match="4-bit"):
            Stack(p, "backbone", cfg)


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
