"""What the engine's paged and int8-activation paths refuse before they touch a cache: host logic, no GPU."""
from types import SimpleNamespace

import pytest
import torch

from estudiocanciones_amd import engine


def _stack(heads=2, kv=1, dim=256, packed=True):
    """A stack of one layer whose weights are names only."""
    lin = lambda: SimpleNamespace(qp=object() if packed else None)  # noqa: E731
    st = object.__new__(engine.Stack)
    b = SimpleNamespace(qkv=lin(), o=lin(), w13=lin(), w2=lin(), h=heads, kvh=kv, hd=dim // heads, kc=None, vc=None)
    st.blocks, st.dim, st.hd, st.rope, st.prompt_a8 = [b], dim, dim // heads, None, False
    st.tail = st.tail2 = st.att_ws = st.att_cnt = st.paged = st.paged_plan = None
    return st


def _no_gpu(monkeypatch):
    def call(name, *_):
        raise AssertionError(f"{name} was launched")
    monkeypatch.setattr(engine._ffi, "call", call)


@pytest.mark.parametrize("call", ["__call__", "decode", "decode_reference"])
@pytest.mark.parametrize("packed", [True, False])
def test_a_stack_in_pages_refuses_the_dense_calls(monkeypatch, call, packed):
    _no_gpu(monkeypatch)
    st = _stack(packed=packed)
    st.paged = SimpleNamespace()
    x, pos = torch.zeros(1, 3, 256, dtype=torch.float16), torch.arange(3)[None]
    with pytest.raises(RuntimeError, match="in pages"):
        st(x, pos) if call == "__call__" else getattr(st, call)(x[0], pos[0], 3)


def test_a_stack_without_pages_refuses_the_paged_calls(monkeypatch):
    _no_gpu(monkeypatch)
    st = _stack()
    with pytest.raises(RuntimeError, match="alloc_paged"):
        st.decode_paged(torch.zeros(3, 256, dtype=torch.float16), torch.arange(3))
    with pytest.raises(RuntimeError, match="alloc_paged"):
        st.prompt_paged(torch.zeros(1, 3, 256, dtype=torch.float16), torch.tensor([0]))


def test_a_prompt_longer_than_the_table_is_refused_before_it_takes_pages(monkeypatch):
    _no_gpu(monkeypatch)
    st = _stack()
    st.paged = SimpleNamespace(table=torch.zeros(2, 3, dtype=torch.int32), page=16, length=torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="48 slots"):
        st.prompt_paged(torch.zeros(1, 49, 256, dtype=torch.float16), torch.tensor([0]))


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 1536),    # head_dim 384: no paged attention
                                          (4, 2, 384),     # 96
                                          (5, 1, 640),     # five query heads on one: no prompt attention
                                          (16, 1, 2048)])
def test_heads_that_the_paged_path_does_not_run(monkeypatch, heads, kv, dim):
    """Refused before the old caches go."""
    _no_gpu(monkeypatch)
    st = _stack(heads, kv, dim)
    st.blocks[0].kc = st.blocks[0].vc = kept = object()
    with pytest.raises(NotImplementedError, match="head"):
        st.alloc_paged(2, 9, 4, torch.device("cuda"), [(2, 16)], 16)
    assert st.paged is None and st.paged_plan is None and st.blocks[0].kc is kept


def _model(**kw):
    gm = object.__new__(engine.HeartMuLaLite)
    gm.backbone, gm.graphs = _stack(**kw), {}
    return gm


@pytest.mark.parametrize("paged", [-1, 11, 200])
def test_a_prompt_longer_than_the_capacity_is_refused(monkeypatch, paged):
    _no_gpu(monkeypatch)
    with pytest.raises(ValueError, match="capacity"):
        _model().alloc(2, 10, 1.5, seed=1, paged=paged)


@pytest.mark.parametrize("kw", [dict(a8=True), dict(paged=True), dict(a8=True, paged=True)])
def test_generate_refuses_heads_without_a_prompt_attention(monkeypatch, kw):
    _no_gpu(monkeypatch)
    gm = _model(heads=5, kv=1, dim=640)
    gm.alloc = lambda *a, **k: gm.backbone.alloc_paged(2, 9, 4, torch.device("cuda"), [(2, 16)], 16) if k.get("paged") else \
        pytest.fail("allocated")
    with pytest.raises(NotImplementedError, match="head"):
        gm.generate([1, 2, 3], 1, max_ms=160, **kw)


@pytest.mark.parametrize("B,S", [(3, 7), (66000, 1), (700, 100), (2, 40000), (1, 70000), (65535, 1), (65536, 1), (3, 65536)])
def test_prompt_attention_by_rows_stays_within_a_launch(monkeypatch, B, S):
    """Head shapes without a prompt kernel take a row per workgroup along the third grid dimension, which ends at 65536:
    every row exactly once, with its own sequence's cache."""
    Hq, Hk, HD, L = 6, 1, 128, 4
    rows, seen = B * S, torch.zeros(B * S, dtype=torch.long)
    st, calls = _stack(6, 1, 768), []

    class At:  # (its pointers are fictions: only offsets are looked at)
        def __init__(self, base, step, shape, i0=0):
            self.base, self.step, self.shape, self.i0, self.device, self.dtype = base, step, shape, i0, "cpu", torch.float16

        def data_ptr(self):
            return self.base + self.step * self.i0

        def __getitem__(self, s):
            a, b, _ = s.indices(self.shape[0])
            return At(self.base, self.step, (b - a,) + tuple(self.shape[1:]), self.i0 + a)

    monkeypatch.setattr(engine._ffi, "call", lambda name, *a: calls.append((name, a)))
    monkeypatch.setattr(engine, "stream_ptr", lambda d: 0)
    out = At(3 << 40, Hq * HD * 2, (rows, Hq * HD))
    monkeypatch.setattr(engine.torch, "empty_like", lambda t: out)
    q, pos = At(1 << 40, Hq * HD * 2, (rows, Hq * HD)), At(2 << 40, 8, (rows,))
    kc, vc = At(4 << 40, Hk * L * HD * 2, (B, Hk, L, HD)), At(5 << 40, Hk * L * HD * 2, (B, Hk, L, HD))
    assert st._prompt_attn(st.blocks[0], q, kc, vc, pos, S) is out
    for name, a in calls:
        assert name == "ecd_decode_attn"
        qp, kp, vp, pp, op, _, _, _, R, s, hq, hk, l, hd, ns, scale, _ = a
        assert 0 < R <= 65535 and (hq, hk, l, hd, ns) == (Hq, Hk, L, HD, 1) and scale == pytest.approx(HD ** -0.5)
        r0, b0 = (qp - (1 << 40)) // (Hq * HD * 2), (kp - (4 << 40)) // (Hk * L * HD * 2)
        assert (pp - (2 << 40)) // 8 == r0 == (op - (3 << 40)) // (Hq * HD * 2) and (vp - (5 << 40)) // (Hk * L * HD * 2) == b0
        for r in (0, R // 2, R - 1):  # (the kernel's own sequence number of a row)
            assert b0 + r // s == (r0 + r) // S
        seen[r0:r0 + R] += 1
    assert (seen == 1).all()


@pytest.mark.parametrize("groups", [[(1, 16)], [(3, 0)], [(2, 16), (1, 0)], []])
def test_groups_that_are_not_the_sequences(monkeypatch, groups):
    """A row per sequence: rows that the plan does not know would come out as whatever lay in the memory."""
    _no_gpu(monkeypatch)
    st = _stack()
    st.blocks[0].kc = kept = object()
    with pytest.raises(ValueError, match="2 sequences"):
        st.alloc_paged(2, 9, 4, torch.device("cuda"), groups, 16)
    assert st.paged is None and st.blocks[0].kc is kept
