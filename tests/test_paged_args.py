"""What the paged cache and the int8-activation entries refuse, and how a batch is cut into parts: host logic, no GPU."""
import pytest
import torch

I, N = -22, -95


@pytest.mark.parametrize("want,call", [
    (I, lambda L: L.ecd_page_free(None, 4, 8, 4, 8, 2, 16, 8, 1, 8, None)),
    (I, lambda L: L.ecd_page_free(8, 4, 8, 4, 8, 2, 0, 8, 1, 8, None)),                 # page of 0 slots
    (I, lambda L: L.ecd_page_free(8, 4, 8, 4, 8, 2, 16, 8, 0, 8, None)),                # no sequences
    (I, lambda L: L.ecd_page_fork(None, 8, 4, 8, 4, 8, 2, 8, 8, 1, 16, 8, 2, 1, 16, 64, None)),
    (I, lambda L: L.ecd_page_fork(16, 8, 4, 8, 4, 8, 2, 8, 8, 1025, 16, 8, 2, 1, 16, 64, None)),  # too many at once
    (I, lambda L: L.ecd_page_fork(24, 8, 4, 8, 4, 8, 2, 8, 8, 1, 16, 8, 2, 1, 16, 64, None)),     # kv not 16-byte aligned
    (I, lambda L: L.ecd_page_fork(16, 8, 4, 8, 4, 8, 2, 8, 8, 1, 24, 8, 2, 1, 16, 64, None)),     # plan not aligned
    (I, lambda L: L.ecd_page_fork(16, 8, 4, 8, 4, 8, 2, 8, 8, 1, 16, 8, 2, 1, 16, 60, None)),     # HD % 8
    (I, lambda L: L.ecd_page_extend(8, 4, 8, 4, 8, 1025, 16, 8, 8, None)),
    (I, lambda L: L.ecd_page_extend(8, 4, 8, 4, 8, 2, 16, None, 8, None)),
    (N, lambda L: L.ecd_page_extend(8, 4, 8, 1 << 30, 8, 4, 16, 8, 8, None)),           # 2^32 pages of a table
    (N, lambda L: L.ecd_page_free(8, 4, 8, 4, 8, 2, 16, 8, 1 << 24, 8, None)),          # 2^32 threads
    (N, lambda L: L.ecd_page_fork(16, 8, 4, 8, 4, 8, 2, 8, 8, 1, 16, 8, 1 << 20, 16, 16, 64, None)),
    (N, lambda L: L.ecd_paged_write(16, 512, None, 0, 8, None, 16, 16, 8, 4, 4, 4, 1 << 28, 1, 4, 2, 16, 64, None)),
    (N, lambda L: L.ecd_quant_a8(16, 64, None, 0.0, 16, 128, 16, 1 << 24, 64, None)),
    (I, lambda L: L.ecd_page_compact(16, 8, 4, 8, 8, 16, 8, 4, 8, 8, 2, 4, 8, 8, 2, 1, 16, 64, None)),  # kv2 is kv
    (I, lambda L: L.ecd_page_compact(16, 8, 4, 8, 8, 32, 8, 0, 8, 8, 2, 4, 8, 8, 2, 1, 16, 64, None)),  # empty pool
    (I, lambda L: L.ecd_paged_write(16, 512, None, 0, 8, None, 16, 16, 8, 4, 4, 4, 1, 1, 4, 2, 16, 60, None)),   # HD % 8
    (I, lambda L: L.ecd_paged_write(16, 504, None, 0, 8, None, 16, 16, 8, 4, 4, 4, 1, 1, 4, 2, 16, 64, None)),   # ld short
    (I, lambda L: L.ecd_paged_write(16, 512, 16, 9, 8, None, 16, 16, 8, 4, 4, 4, 1, 1, 4, 2, 16, 64, None)),     # rope, no q
    (I, lambda L: L.ecd_paged_write(16, 512, None, 0, 8, None, 16, 16, 8, 3, 4, 4, 1, 1, 4, 2, 16, 64, None)),   # table rows
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, None, 8, 1, 1, 2, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, 0.1, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, None, 8, 8, 0, 2, 2, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, 0.1, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 2, 1, 4, 9, 4, 2, 24, 128, 0.1, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 2, 1, 4, 9, 4, 2, 8, 128, 0.1, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 2, 1, 4, 9, 4, 3, 16, 128, 0.1, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, 0.0, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 1 << 27, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 2, 1, 1 << 27, 9, 4, 2, 16, 128, 0.1, None)),
    (I, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 1 << 22, 1, 4, 9, 4, 2, 16, 128, 0.1, None)),
    (N, lambda L: L.ecd_paged_attn(16, 768, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 1, 4, 2, 1, 4, 9, 4, 2, 16, 192, 0.1, None)),
    (N, lambda L: L.ecd_paged_attn(16, 1024, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 1, 1, 2, 4, 2, 1, 4, 9, 4, 2, 16, 256, 0.1, None)),
    (N, lambda L: L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, 16, 8, 8, 0, 513, 513, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, 0.1, None)),
    (I, lambda L: L.ecd_quant_a8(16, 96, None, 0.0, 16, 128, 16, 1, 96, None)),         # K % 64
    (I, lambda L: L.ecd_quant_a8(16, 64, None, 0.0, 16, 64, 16, 1, 64, None)),          # ldc % 128
    (I, lambda L: L.ecd_quant_a8(16, 64, None, -1.0, 16, 128, 16, 1, 64, None)),        # eps
    (I, lambda L: L.ecd_quant_a8(16, 1 << 18, None, 0.0, 16, 1 << 18, 16, 1, 1 << 18, None)),  # K > 2^17
    (I, lambda L: L.ecd_gemm_a8(16, 128, 16, 16, 16, None, 0, 16, 16, 0, 16, 64, None)),  # no rows
    (I, lambda L: L.ecd_gemm_a8(16, 128, 16, 16, 16, None, 0, 16, 15, 1, 16, 64, None)),  # ldy < N
    (I, lambda L: L.ecd_gemm_a8(16, 128, 16, 16, 16, 16, 15, 16, 16, 1, 16, 64, None)),   # ldr < N
    (I, lambda L: L.ecd_gemm_a8(16, 1 << 24, 16, 16, 16, None, 0, 16, 16, 1, 16, 64, None)),  # rows 16 MB apart
    (I, lambda L: L.ecd_gemm_a8_tuned(16, 128, 16, 16, 16, None, 0, 16, 16, 1, 16, 64, 9, None)),
    (I, lambda L: L.ecd_gemm_a8_silu(16, 128, 16, 16, 16, 16, 7, 1, 8, 64, None)),        # ldm < F
    (I, lambda L: L.ecd_gemm_a8_silu(16, 128, 16, 16, 16, 16, 8, 1, 0, 64, None)),
])
def test_entries_refuse_on_the_host(want, call):
    from estudiocanciones_amd import _ffi
    assert call(_ffi.lib()) == want


def test_calls_refuse_tensors_that_are_not_on_a_gpu():
    from estudiocanciones_amd import kernels as K
    from estudiocanciones_amd.paged import PagedCache
    ref, table = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    length, err = torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        K.page_free(ref, table, length, ref, 16, err)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        K.quant_a8(x)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        K.paged_attn_plan([(1, 0)], 4, 2, 64, 64, "cpu")
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        PagedCache(1, 1, 1, 1, 64, device="cpu")


@pytest.mark.parametrize("kw", [dict(groups=[]), dict(groups=[(0, 4)]), dict(max_len=-1), dict(groups=[(2, -1)]),
                                dict(Hq=5), dict(Hq=34), dict(HD=96), dict(HD=384)])
def test_plan_refuses(kw):
    from estudiocanciones_amd.kernels import paged_attn_plan
    a = dict(groups=[(2, 4)], Hq=4, Hk=2, HD=64, max_len=64, device="cuda")
    with pytest.raises(ValueError):
        paged_attn_plan(**{**a, **kw})


@pytest.mark.parametrize("kw", [dict(layers=0), dict(page=8), dict(page=48), dict(head_dim=20), dict(seqs=1025), dict(pages=0),
                                dict(max_pages=0)])
def test_cache_refuses(kw):
    from estudiocanciones_amd.paged import PagedCache
    a = dict(layers=1, seqs=1, pages=1, kv_heads=1, head_dim=64)
    with pytest.raises(ValueError):
        PagedCache(**{**a, **kw}, device="cuda")


@pytest.mark.parametrize("groups", [[(1, 0)], [(1, 50)], [(4, 256), (4, 256)], [(3, 1), (9, 277), (2, 0), (21, 6000)],
                                    [(64, 7000), (1, 8000)], [(1000, 130)]])
@pytest.mark.parametrize("Hq,Hk,HD", [(24, 8, 128), (5, 5, 64), (16, 1, 128), (8, 2, 256), (32, 2, 64)])
def test_parts_of_a_plan(groups, Hq, Hk, HD):
    """Every shared slot of every row and kv head lies in exactly one part, and no two parts of a row have one number."""
    from estudiocanciones_amd.kernels import _make_plan
    G = Hq // Hk
    plan = _make_plan(groups, Hq, Hk, HD, 8192, torch.device("cpu"), share=True)
    rows = plan.flat[:2 * plan.R].view(-1, 2).tolist()
    items = plan.flat[2 * plan.R:].view(-1, 6).tolist()
    assert plan.R == sum(n for n, _ in groups) and len(items) == plan.nitems
    seen = {}
    for row0, n, lo, hi, part, kh in items:
        assert 1 <= n and n * G <= 16 * plan.ctiles and 0 <= lo < hi and 0 <= kh < Hk and lo % 32 == 0
        for r in range(row0, row0 + n):
            seen.setdefault((r, kh), []).append((lo, hi, part))
    r = 0
    for n, p in groups:
        for _ in range(n):
            shared, parts = rows[r]
            assert shared == (p if n > 1 else 0) and parts + plan.nown <= plan.parts <= 512
            for kh in range(Hk):
                got = sorted(seen.get((r, kh), []))
                assert len(got) == parts and [g[2] for g in got] == list(range(parts))
                ends = [0] + [g[1] for g in got]
                assert [g[0] for g in got] == ends[:-1] and ends[-1] == shared
            r += 1
    heads = plan.R * Hq
    assert plan.ws == (0 if plan.parts == 1 else 2 * (-(-heads * plan.parts // 4) * 4) + heads * plan.parts * HD)


@pytest.mark.parametrize("share", [None, True, False])
def test_a_prefix_that_no_row_can_hold_is_not_shared(share):
    from estudiocanciones_amd.kernels import _make_plan
    a = _make_plan([(3, 100), (2, 65), (4, 64)], 4, 2, 64, 64, torch.device("cpu"), share=share)
    b = _make_plan([(3, 0), (2, 0), (4, 64)], 4, 2, 64, 64, torch.device("cpu"), share=share)
    assert (a.nitems, a.nown, a.parts, a.ws) == (b.nitems, b.nown, b.parts, b.ws) and torch.equal(a.flat, b.flat)
    assert _make_plan([(1, 5)], 4, 2, 64, 0, torch.device("cpu"), share=share).parts == 1


def test_plans_by_the_rule():
    """Little to share: a workgroup per row and kv head and nothing to join; much to share, or too few pairs for long rows: parts."""
    from estudiocanciones_amd.kernels import _make_plan
    cpu = torch.device("cpu")
    solo = _make_plan([(4, 100), (4, 100)], 24, 8, 128, 512, cpu)
    assert (solo.nitems, solo.parts, solo.ws, solo.waves) == (0, 1, 0, 8)
    assert _make_plan([(2, 100)], 8, 2, 64, 1024, cpu).parts == 1
    assert _make_plan([(2, 100)], 8, 2, 64, 1025, cpu).parts > 1
    assert _make_plan([(32, 100)], 24, 8, 128, 8192, cpu).waves == 8
    assert _make_plan([(16, 4096)], 24, 8, 128, 8192, cpu).nitems > 0
    assert _make_plan([(16, 4096)], 24, 8, 128, 8192, cpu, share=False).nitems == 0
