"""Paged operators on plans and states that hold something out of range: skipped or reported, the rest as it would be."""
import numpy as np
import pytest

from test_gpu_paged_attn import Batch

pytestmark = pytest.mark.gpu


def test_shared_parts_out_of_range_are_skipped(dev):
    """Items of a part number that no row has, or that one of its rows has not (the places of a row's own slots), of rows and
    heads that are not there and of too many rows: the results are those without them, bit for bit."""
    import torch
    from estudiocanciones_amd.kernels import PagedAttnPlan, paged_attn, paged_attn_plan
    Hq, Hk, HD = 6, 2, 128
    b = Batch([(4, 700), (3, 150), (1, 0)], [701, 830, 900, 700, 151, 400, 150, 620], Hq, Hk, HD, 32, seed=4)
    plan = paged_attn_plan(b.groups, Hq, Hk, HD, 1024, dev, share=True)
    R = plan.R
    rows = [tuple(x) for x in plan.flat[:2 * R].view(-1, 2).tolist()]
    items = [tuple(x) for x in plan.flat[2 * R:].view(-1, 6).tolist()]
    few, most, big = rows[4][1], plan.parts - plan.nown, 2 ** 31 - 1
    assert 0 < few < most and plan.nown > 1 and rows[7][1] == 0
    bad = [(4, 3, 0, 128, part, h) for part in range(few, most) for h in range(Hk)]  # rows with fewer shared parts
    bad += [(7, 1, 0, 128, 0, 0), (0, 4, 0, 128, most, 0), (0, 4, 0, 128, plan.parts, 1), (0, 4, 0, 128, -1, 0),
            (0, 4, 0, 128, big, 0), (-1, 2, 0, 128, 0, 0), (R - 1, 2, 0, 128, 0, 0), (R, 1, 0, 128, 0, 0), (big, 1, 0, 128, 0, 0),
            (0, 0, 0, 128, 0, 0), (0, -3, 0, 128, 0, 0), (0, 6, 0, 128, 0, 0), (0, big, 0, 128, 0, 0), (0, 4, 0, 128, 0, Hk),
            (0, 4, 0, 128, 0, -1)]
    # part 4 of row 3 (formed twice, the same bits) beside row 4, which has no part 4
    assert (0, 4, 512, 640, 4, 0) in items
    bad += [(3, 2, 512, 640, 4, h) for h in range(Hk)]
    more = PagedAttnPlan(items + bad, rows, plan.nown, plan.parts, plan.ctiles, plan.waves, Hq, Hk, HD, dev)
    kv, table, q = (torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in (b.pool, b.table, b.q))
    pos = torch.tensor(b.lens, device=dev) - 1
    want = paged_attn(q, kv[0], kv[1], table, pos, plan)
    for _ in range(3):
        assert torch.equal(paged_attn(q, kv[0], kv[1], table, pos, more), want)


def _pool(dev, pages=9, B=6, MP=4, P=16):
    from test_gpu_pages import Model, State
    st = State(dev, 2, pages, 1, P, 8, B, MP)
    m = Model(st.np.view(np.uint16), B, MP)
    pos = [40, 31] + [-1] * (B - 2)  # three pages, the last one partial; two whole pages
    m.extend(pos)
    st.extend(pos)
    return st, m


@pytest.mark.parametrize("bad", [-1, -7, 9, 2 ** 31 - 1])
@pytest.mark.parametrize("seq,col", [(0, 0), (0, 1), (0, 2), (1, 0), (1, 1)])
def test_fork_reports_a_page_number_out_of_range(dev, bad, seq, col):
    """Among the whole pages as well as the partial one: bit 1, and nothing else changes, for the good source's child neither."""
    st, m = _pool(dev)
    st.table[seq, col] = bad
    m.table[seq][col] = bad
    st.fork([1 - seq, seq], [2, 3])
    st.same(m, "two sources", 1)
    st.err.zero_()
    st.fork([seq] * 3, [4, 2, 5])
    st.same(m, "one source", 1)
    st.err.zero_()
    st.fork([1 - seq], [3])  # the other one is as good as before
    m.fork([1 - seq], [3])
    st.same(m, "the good one")


def test_fork_looks_at_all_pages_of_many_children(dev):
    """A bad page behind 200 good ones, of the last of 1000 children, whose sources do not repeat in a row."""
    st, m = _pool(dev, pages=1600, B=1024, MP=260, P=16)
    pos = [-1, -1] + [16 * 203 - 1] * 3 + [-1] * 1019  # whole pages only
    m.extend(pos)
    st.extend(pos)
    src, dst = [2 + i % 2 for i in range(1000)], list(range(24, 1024))
    src[-1] = 4
    st.table[4, 202] = 1600
    m.table[4][202] = 1600
    st.fork(src, dst)
    st.same(m, "bad", 1)
    st.err.zero_()
    src[-1] = 3
    m.fork(src, dst)
    st.fork(src, dst)
    st.same(m, "good")


def test_fork_without_enough_pages_changes_nothing(dev):
    """Four pages are free: five children with a partial page each get bit 4 alone, four of them are made."""
    st, m = _pool(dev, B=8)
    st.fork([0, 1, 0, 0, 0, 0], [2, 3, 4, 5, 6, 7])
    st.same(m, "five partial pages", 4)
    st.err.zero_()
    m.fork([0, 1, 0, 0, 0], [2, 3, 4, 5, 6])
    st.fork([0, 1, 0, 0, 0], [2, 3, 4, 5, 6])
    st.same(m, "four partial pages")
    st.fork([0], [7])
    st.same(m, "none is left", 4)


@pytest.mark.parametrize("far", [2 ** 63 - 1, 2 ** 62, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5])
def test_positions_behind_the_table_attend_all_of_it(dev, far):
    """A position past the table's last slot counts as that slot, whatever its size; one far below 0 as none."""
    import torch
    from estudiocanciones_amd.kernels import page_extend, paged_attn, paged_attn_plan, paged_write
    b = Batch([(2, 64), (1, 0), (1, 0)], [127, 128, 128, 1], 6, 2, 64, 32, seed=2)
    MP = 4
    table = b.table[:, :MP]
    assert (table[:3] >= 0).all()
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    kv, q, tab = T(b.pool), T(b.q), T(table)
    for share in (True, False):
        plan = paged_attn_plan(b.groups, 6, 2, 64, 4096, dev, share)
        want = paged_attn(q, kv[0], kv[1], tab, torch.tensor([126, 127, 127, -1], device=dev), plan)
        got = paged_attn(q, kv[0], kv[1], tab, torch.tensor([126, far, far, -far], device=dev), plan)
        assert torch.equal(got, want) and (got[3] == 0).all() and got[2].any()
    before = kv.clone()
    paged_write(torch.ones(4, 10 * 64, dtype=torch.float16, device=dev), kv[0], kv[1], tab, torch.full((4,), far, device=dev), 1, 6, 2)
    assert torch.equal(kv, before)
    st, m = _pool(dev)
    page_extend(st.ref, st.table, st.length, torch.tensor([-1, far, -far, -1, -1, -1], device=dev), 16, st.err)
    st.same(m, "extend", 8)


def test_the_workspace_is_held_until_the_launch(dev, monkeypatch):
    """What another thread allocates while a call is on its way to its launch does not lie in the call's workspace."""
    import torch
    from estudiocanciones_amd import kernels as K
    b = Batch([(4, 700), (2, 0)], [701, 830, 900, 700, 151, 400], 6, 2, 128, 32, seed=4)
    kv, table, q = (torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in (b.pool, b.table, b.q))
    pos = torch.tensor(b.lens, device=dev) - 1
    plan = K.paged_attn_plan(b.groups, 6, 2, 128, 1024, dev, share=True)
    assert plan.ws
    want = K.paged_attn(q, kv[0], kv[1], table, pos, plan)
    launch, met = K._call_on, []

    def later(d, name, *args):
        other = torch.empty(plan.ws, device=d, dtype=torch.float32)  # on the same stream, as another thread's would be
        met.append(other.data_ptr() in args)
        launch(d, name, *args)
    monkeypatch.setattr(K, "_call_on", later)
    for _ in range(3):
        assert torch.equal(K.paged_attn(q, kv[0], kv[1], table, pos, plan), want)
    assert met == [False] * 3
