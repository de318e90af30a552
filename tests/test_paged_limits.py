"""What the paged cache and the int8-activation entries refuse on the host: calls that would reach past their buffers or whose
sizes pass what the kernels count in."""
import pytest

I, N = -22, -95


def _attn(L, nitems, nown, parts, ws):
    return L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, ws, 16, 8, nitems, nown, parts, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, 0.1, None)


@pytest.mark.parametrize("nitems,nown,parts,ws", [(1, 1, 1, None), (1, 1, 1, 16), (3, 4, 4, 16), (1, 2, 2, 16)])
def test_shared_parts_need_places_of_their_own(nitems, nown, parts, ws):
    """Shared parts with as many parts as a row's own slots have: they would be written to the own parts' places, or to a
    workspace that is not there."""
    from estudiocanciones_amd import _ffi
    assert _attn(_ffi.lib(), nitems, nown, parts, ws) == I


BIG = 2 ** 31 - 1


def _a8(L, M, N, cfg=0):
    return L.ecd_gemm_a8_tuned(16, 128, 16, 16, 16, None, 0, 16, N, M, N, 64, cfg, None)


@pytest.mark.parametrize("call", [
    # 2^32 threads of a launch: 16 features of 512 threads, tiles of 256 and 512 threads
    lambda L: L.ecd_gemm_a8(16, 128, 16, 16, 16, None, 0, 16, 1 << 27, 1, 1 << 27, 64, None),
    lambda L: L.ecd_gemm_a8_silu(16, 128, 16, 16, 16, 16, 1 << 26, 1, 1 << 26, 64, None),
    lambda L: _a8(L, 1 << 30, 32, 2), lambda L: _a8(L, 1 << 29, 64, 3), lambda L: _a8(L, 64, 1 << 30, 4),
    lambda L: _a8(L, 1 << 29, 256, 5), lambda L: _a8(L, 1 << 28, 1024, 6), lambda L: _a8(L, 1 << 28, 4096, 7),
    lambda L: _a8(L, 1 << 28, 2048, 8), lambda L: _a8(L, 1, 1 << 27, 1),
    # row and feature numbers that pass 32 bits within a tile
    lambda L: _a8(L, BIG, 256, 8), lambda L: _a8(L, 256, BIG, 8), lambda L: _a8(L, 1, BIG, 1), lambda L: _a8(L, BIG, 16),
    # page numbers and table columns that are counted in 32 bits, a workgroup's step at a time
    lambda L: L.ecd_page_free(8, BIG, 8, 4, 8, 2, 16, 8, 1, 8, None),
    lambda L: L.ecd_page_free(8, 4, 8, BIG, 8, 2, 16, 8, 1, 8, None),
    lambda L: L.ecd_page_extend(8, BIG, 8, 4, 8, 2, 16, 8, 8, None),
    lambda L: L.ecd_page_extend(8, 4, 8, BIG, 8, 1, 16, 8, 8, None),
    lambda L: L.ecd_page_fork(16, 8, BIG, 8, 4, 8, 2, 8, 8, 1, 16, 8, 2, 1, 16, 64, None),
    lambda L: L.ecd_page_fork(16, 8, 4, 8, BIG, 8, 2, 8, 8, 1, 16, 8, 2, 1, 16, 64, None),
    lambda L: L.ecd_page_compact(16, 8, BIG, 8, 8, 32, 8, 9, 8, 8, 2, 4, 8, 8, 2, 1, 16, 64, None),
    lambda L: L.ecd_page_compact(16, 8, 4, 8, 8, 32, 8, BIG, 8, 8, 2, 4, 8, 8, 2, 1, 16, 64, None),
    lambda L: L.ecd_page_compact(16, 8, 4, 8, 8, 32, 8, 9, 8, 8, 2, BIG, 8, 8, 2, 1, 16, 64, None),
    # pages of 2^34 values: their pieces pass 32 bits
    lambda L: L.ecd_page_fork(16, 8, 4, 8, 4, 8, 2, 8, 8, 1, 16, 8, 2, 1, 1 << 28, 64, None),
    # products of sizes that pass 64 bits
    lambda L: L.ecd_page_fork(16, 8, 4, 8, 4, 8, 2, 8, 8, 1, 16, 8, 1 << 30, 1 << 30, 16, 2048, None),
])
def test_sizes_that_the_kernels_do_not_count(call):
    from estudiocanciones_amd import _ffi
    assert call(_ffi.lib()) == N


@pytest.mark.parametrize("call", [
    # 2^30 + 2 2^30 heads are not -2^30
    lambda L: L.ecd_paged_write(16, 512, None, 0, 8, None, 16, 16, 8, 4, 4, 4, 1, 1, 1 << 30, 1 << 30, 16, 64, None),
    # 2^31 pages of 2^30 slots and 8 heads are not 0 rows of the pool
    lambda L: L.ecd_paged_attn(16, 2048, 16, 16, 8, 1, 8, 8, None, 8, 8, 0, 1, 1, 1, 4, 1, 1, 1, 1 << 30, 16, 16, 1 << 30, 128, 0.1, None),
])
def test_sizes_whose_products_pass_64_bits(call):
    from estudiocanciones_amd import _ffi
    assert call(_ffi.lib()) in (I, N)


@pytest.mark.parametrize("scale", [float("inf"), 3e38, 1e300])
def test_a_scale_that_no_number_of_32_bits_holds_times_log2_e(scale):
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    assert L.ecd_paged_attn(16, 512, 16, 16, 8, 4, 8, 8, None, 8, 8, 0, 1, 1, 1, 4, 2, 1, 4, 9, 4, 2, 16, 128, scale, None) == I


class _Made:
    """A tensor as the calls' checks look at it, of sizes that need no memory."""

    def __init__(self, dtype, *shape):
        import torch
        self.dtype, self.shape, self.device, self.is_cuda = dtype, torch.Size(shape), torch.device("cuda", 0), True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i=None):
        s = [1]
        for n in reversed(self.shape[1:]):
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("far", [2 ** 32 + 1, 2 ** 31, 2 ** 33 + 16, 2 ** 40])
def test_counts_that_would_wrap_in_the_entry(monkeypatch, far):
    """Rows per sequence and slots per page go to the library as 32-bit numbers: 2^32 + 1 rows would be 1 there, and each row
    would have a row of the table of its own, also where the table has not."""
    import ctypes
    import torch
    from types import SimpleNamespace
    from estudiocanciones_amd import kernels as K
    assert ctypes.c_int(2 ** 32 + 1).value == 1
    monkeypatch.setattr(K, "_call_on", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(K.torch, "empty", lambda *a, **k: _Made(torch.float16, 3, 256))
    h, i32, i64 = torch.float16, torch.int32, torch.int64
    kp, table, pos = _Made(h, 9, 2, 16, 64), _Made(i32, 1, 4), _Made(i64, 3)
    plan = SimpleNamespace(R=3, Hq=4, Hk=2, HD=64, dev=kp.device, ws=0, items_ptr=0, rows_ptr=0, nitems=0, nown=1, parts=1,
                           ctiles=1, waves=4)
    with pytest.raises(ValueError):
        K.paged_attn(_Made(h, 3, 256), kp, kp, table, pos, plan, S=far)
    with pytest.raises(ValueError):
        K.paged_write(_Made(h, 3, 512), kp, kp, table, pos, far, 4, 2)
    state = (_Made(i32, 9), _Made(i32, 2, 4), _Made(i64, 2))
    with pytest.raises(ValueError):
        K.page_free(*state, _Made(i32, 1), far, _Made(i32, 1))
    with pytest.raises(ValueError):
        K.page_extend(*state, _Made(i64, 2), far, _Made(i32, 1))
