"""What the entries of 4-bit weights and of logits refuse, and what the calls refuse without a GPU: host logic."""
import pytest
import torch

I, N = -22, -95


def mm(**kw):
    d = dict(x=16, ldx=64, nw=None, eps=1e-5, codes=16, scales=16, zeros=0, group=64, res=None, ldr=0, y=16, ldy=32, M=1, N=32,
             K=64, silu=0, plan=0, ws=None)
    d.update(kw)
    return lambda L: L.ecd_mm_q4(*d.values(), None)


def lg(**kw):
    d = dict(logits=8, ld=100, guided=0, cfg=1.0, hist=None, hrow=0, htok=0, T=0, length=None, window=0, rep=None, pres=None,
             freq=None, per_row=0, bias=None, ldb=0, allowed=None, lda=0, A=0, state=None, out=8, ldo=100, N=4, V=100)
    d.update(kw)
    return lambda L: L.ecd_process_logits(*d.values(), None)


@pytest.mark.parametrize("want,call", [
    (I, lambda L: L.ecd_quantize_rows_q4(None, 0, 16, 16, None, 1, 64, 64, None)),
    (I, lambda L: L.ecd_quantize_rows_q4(16, 3, 16, 16, None, 1, 64, 64, None)),        # no such type
    (I, lambda L: L.ecd_quantize_rows_q4(16, 0, 16, 16, None, 1, 96, 32, None)),        # K % 64
    (I, lambda L: L.ecd_quantize_rows_q4(16, 0, 16, 16, None, 1, 64, 16, None)),        # group
    (I, lambda L: L.ecd_quantize_rows_q4(24, 0, 16, 16, None, 1, 64, 64, None)),        # alignment
    (I, lambda L: L.ecd_quantize_rows_q4(16, 0, 16, 16, None, 0, 64, 64, None)),
    (N, lambda L: L.ecd_quantize_rows_q4(16, 0, 16, 16, None, 0x7FFFFFFF, 1 << 20, 64, None)),
    (I, lambda L: L.ecd_pack_q4(16, None, None, 32, 64, 64, 0, 16, 16, None)),
    (I, lambda L: L.ecd_pack_q4(16, 16, None, 31, 64, 64, 1, 16, 16, None)),            # odd rows to interleave
    (I, lambda L: L.ecd_pack_q4(16, 16, None, 32, 64, 48, 0, 16, 16, None)),
    (I, lambda L: L.ecd_pack_q4(16, 16, None, 32, 64, 64, 0, 24, 16, None)),
    (N, lambda L: L.ecd_pack_q4(16, 16, None, 0x7FFFFFF0, 64, 64, 0, 16, 16, None)),
    (I, mm(x=None)), (I, mm(codes=None)), (I, mm(scales=None)), (I, mm(y=None)), (I, mm(M=0)), (I, mm(N=0)), (I, mm(K=0)),
    (I, mm(K=96, ldx=96)), (I, mm(ldx=56)), (I, mm(ldx=68)), (I, mm(x=24)), (I, mm(nw=24)), (I, mm(codes=24)),
    (I, mm(scales=24)), (I, mm(group=256)), (I, mm(ldy=31)), (I, mm(res=16, ldr=31)), (I, mm(silu=1, N=31)),
    (I, mm(silu=1, res=16, ldr=32)), (I, mm(nw=16, eps=-1.0)), (I, mm(nw=16, eps=float("nan"))),
    (I, mm(M=17)), (I, mm(plan=7 + 256)), (I, mm(plan=1)), (I, mm(plan=1 + 512)), (I, mm(plan=-1)),  # plans: K / 64 ways at most
    (I, mm(plan=1 + 512, K=128, ldx=128)), (I, mm(plan=1 + 512, K=128, ldx=128, ws=24)), (I, mm(plan=1 + 256, nw=16)),  # no workspace
    (N, mm(ldx=1 << 27)), (N, mm(plan=1 + 256, ldx=1 << 27, M=99)), (N, mm(plan=1 + 256, K=1 << 24, ldx=1 << 24)),
    (I, lg(logits=None)), (I, lg(out=None)), (I, lg(N=0)), (I, lg(V=0)), (I, lg(ld=99)), (I, lg(ldo=99)), (I, lg(window=-1)),
    (I, lg(T=-1)), (I, lg(rep=8)), (I, lg(pres=8)), (I, lg(freq=8)), (I, lg(hist=8, hrow=-1)), (I, lg(bias=8, ldb=99)),
    (I, lg(allowed=8, lda=3, A=1)), (I, lg(allowed=8, lda=4, A=0)), (I, lg(allowed=8, lda=4, A=3)),
    (N, lg(N=65536)), (N, lg(hist=8, hrow=0, htok=0, T=(1 << 30) + 1)), (N, lg(V=0x7FFFFFFF, ld=0x7FFFFFFF, ldo=0x7FFFFFFF)),
])
def test_entries_refuse_on_the_host(want, call):
    from estudiocanciones_amd import _ffi
    assert call(_ffi.lib()) == want


def test_packed_bytes():
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    assert [L.ecd_packed_bytes_q4(n, k) for n, k in ((1, 64), (32, 64), (33, 64), (8197, 3072), (1, 65), (0, 64))] == \
        [1024, 1024, 2048, 257 * 48 * 1024, 0, 0]
    assert L.ecd_packed_bytes_q4(1 << 20, 1 << 16) == 1 << 35  # (past 32 bits)


def test_plans():
    """Few rows run without a plan of tiles; every plan names a tile and a split that the product takes; the workspace holds the
    parts and the normed rows."""
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    for M, N, K in [(1, 1, 64), (8, 16384, 3072), (16, 1024, 4096), (16, 1024, 8192), (17, 33, 64), (48, 3072, 3072),
                    (187, 3072, 8192), (2048, 16384, 3072), (100000, 8197, 1024), (30, 2000000, 128)]:
        p = L.ecd_mm_q4_plan(M, N, K)
        if M <= 8:
            assert p == 0
        if M > 16:
            assert p > 0
        if p:
            tile, ks = p & 255, p >> 8
            assert 1 <= tile <= 6 and 1 <= ks <= K // 64
            part = ks * M * (-(-N // 8) * 8) * 4 if ks > 1 else 0
            assert L.ecd_mm_q4_ws_bytes(M, N, K, p, 0) == part and L.ecd_mm_q4_ws_bytes(M, N, K, p, 1) == part + 2 * M * K
    assert L.ecd_mm_q4_ws_bytes(8, 64, 64, 0, 1) == 0
    assert [L.ecd_mm_q4_plan(*a) for a in ((0, 1, 64), (1, 0, 64), (1, 1, 65), (1, 1, 0))] == [-22] * 4


def test_calls_refuse_tensors_that_are_not_on_a_gpu():
    from estudiocanciones_amd import kernels as K
    from estudiocanciones_amd.quant import q4_rows
    x = torch.zeros(4, 64, dtype=torch.float16)
    for call in (lambda: q4_rows(x), lambda: K.pack_q4(torch.zeros(4, 32, dtype=torch.uint8), x[:, :1]),
                 lambda: K.process_logits(x)):
        with pytest.raises(RuntimeError):
            call()


def test_choices():
    """Up to 16 rows no plan; more run by a tile or by the few-row kernel over blocks of rows, whose workspace is the normed rows'."""
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    seen = set()
    for M, N, K in [(1, 1, 64), (16, 1024, 8192), (17, 33, 64), (48, 3072, 3072), (20, 5120, 3072), (187, 3072, 8192),
                    (2048, 16384, 3072), (1 << 24, 64, 64), (30, 2000000, 128)]:
        p = L.ecd_mm_q4_choice(M, N, K)
        seen.add(p & 255)
        assert (p == 0) == (M <= 16)
        if p:
            tile, ks = p & 255, p >> 8
            assert 1 <= ks <= K // 64 and (1 <= tile <= 6 or (17 <= tile <= 19 and ks == 1 and M <= 16 * 65535))
            if tile > 6:
                assert L.ecd_mm_q4_ws_bytes(M, N, K, p, 0) == 0 and L.ecd_mm_q4_ws_bytes(M, N, K, p, 1) == 2 * M * K
    assert seen & {17, 18, 19} and seen & set(range(1, 7))
    assert [L.ecd_mm_q4_choice(*a) for a in ((0, 1, 64), (1, 0, 64), (1, 1, 65), (1, 1, 0))] == [-22] * 4


@pytest.mark.parametrize("code,call", [
    (I, mm(plan=16 + 256)), (I, mm(plan=17)), (I, mm(plan=17 + 512)), (I, mm(plan=20 + 256)), (I, mm(plan=18 + 256, nw=16)),
    (N, mm(plan=17 + 256, ldx=1 << 27)), (N, mm(plan=19 + 256, M=16 * 65535 + 1)),
    (N, mm(plan=19 + 256, M=16 * 65535 + 1, nw=16, ws=16))])
def test_refused_few_row_plans(code, call):
    from estudiocanciones_amd import _ffi
    assert call(_ffi.lib()) == code


def test_choices_with_two_parts():
    """A norm in two parts: 32 more than a plan, and for the tiles twice the normed rows in the workspace; none without a norm."""
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    seen = set()
    for M, N, K in [(1, 2, 64), (16, 1024, 8192), (17, 34, 64), (48, 3072, 3072), (2048, 16384, 3072), (1 << 24, 64, 64)]:
        p = L.ecd_mm_q4_norm_choice(M, N, K, 1)
        assert (p == 0) == (M <= 16)
        if p:
            tile, ks = (p & 255) - 32, p >> 8
            seen.add(tile)
            assert 1 <= ks <= K // 64 and (1 <= tile <= 6 or (17 <= tile <= 19 and ks == 1))
            part = ks * M * (-(-N // 8) * 8) * 4 if ks > 1 else 0
            assert L.ecd_mm_q4_ws_bytes(M, N, K, p, 1) == (part + 4 * M * K if tile <= 6 else 0)
            assert mm(plan=p, M=M, N=N, K=K, ldx=K, ldy=N)(L) == I
    assert seen & {17, 18, 19} and seen & set(range(1, 7))
    # without a SiLU the tiles take rows rounded once
    for M in (17, 48, 300, 2048):
        p = L.ecd_mm_q4_norm_choice(M, 16384, 3072, 0)
        assert (p & 32) == (32 if p & 16 else 0) and L.ecd_mm_q4_ws_bytes(M, 16384, 3072, p, 1) == (0 if p & 16 else 2 * M * 3072) + \
            ((p >> 8) * M * 16384 * 4 if p >> 8 > 1 else 0)
    assert mm(plan=32 + 1 + 256, nw=16)(L) == I and mm(plan=32 + 1 + 256, nw=16, ws=24)(L) == I  # no workspace for it
    assert mm(plan=32, nw=16, ws=16)(L) == I and mm(plan=32 + 16 + 256, nw=16, ws=16)(L) == I
    assert mm(plan=64 + 1 + 256, nw=16, ws=16)(L) == I
    assert [L.ecd_mm_q4_norm_choice(*a) for a in ((0, 1, 64, 0), (1, 0, 64, 1), (1, 1, 65, 0), (1, 1, 0, 1))] == [-22] * 4


def test_rules_that_leave_nothing_are_refused():
    """A codebook without a code, or before the shortest length with none but end codes; biases that are not finite."""
    from estudiocanciones_amd.engine import AUDIO_EOS, AUDIO_VOCAB, N_CB, HeartMuLaLite
    check = HeartMuLaLite._check_rules
    some = torch.zeros(N_CB, AUDIO_VOCAB, dtype=torch.bool)
    some[:, 5] = True
    check(1.0, 0.0, 0.0, 0, None, some, 10)
    none = some.clone()
    none[3] = False
    ends = none.clone()
    ends[3, AUDIO_EOS] = True
    check(1.0, 0.0, 0.0, 0, None, ends)
    check(1.0, 0.0, 0.0, 0, torch.full((N_CB, AUDIO_VOCAB), -1e30), ends, 0)
    for allowed, first in ((none, 0), (none, 4), (ends, 1)):
        with pytest.raises(ValueError, match="allowed"):
            check(1.0, 0.0, 0.0, 0, None, allowed, first)
    for v in (float("nan"), float("inf"), float("-inf")):
        bias = torch.zeros(N_CB, AUDIO_VOCAB)
        bias[7, -1] = v
        with pytest.raises(ValueError, match="bias"):
            check(1.0, 0.0, 0.0, 0, bias, None)

