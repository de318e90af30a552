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
