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


def test_whether_matrices_meet():
    """Against the sets of their elements: columns of rows of one stride are told apart, others that reach across each other are not."""
    import random
    from estudiocanciones_amd.kernels import _meet
    r = random.Random(1)
    flat = torch.zeros(4000, dtype=torch.float16)
    told = 0
    for _ in range(3000):
        M, ld = r.randint(1, 6), r.randint(4, 60)
        lds = [ld, ld if r.random() < 0.7 else r.randint(4, 60)]
        w = [r.randint(1, d) for d in lds]
        at = [r.randint(0, 200) for _ in range(2)]
        rows = [M, r.choice([M, 2 * M])]
        t, u = (flat.as_strided((n, k), (d, 1), o) for n, k, d, o in zip(rows, w, lds, at))
        share = bool({o + i * d + j for n, k, d, o in [(rows[0], w[0], lds[0], at[0])] for i in range(n) for j in range(k)} &
                     {o + i * d + j for n, k, d, o in [(rows[1], w[1], lds[1], at[1])] for i in range(n) for j in range(k)})
        got = _meet(t, lds[0], u, lds[1])
        assert got or not share
        if lds[0] == lds[1] and at[0] + rows[0] * ld >= at[1] and not share and rows[0] > 1 and rows[1] > 1:
            told += not got
    assert told > 100


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
