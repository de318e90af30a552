"""Decode attention over pages with shared prefixes against float64 attention of each row over the slots it attends."""
import math

import numpy as np
import pytest

from helpers import randn16, rng

pytestmark = pytest.mark.gpu


class Batch:
    """Rows in groups (rows, prefix) over pages in any order; lens[r] slots of row r.  Where a row holds the whole prefix
    it shares the group's pages (the partial one copied), else it has pages of its own."""

    def __init__(self, groups, lens, Hq, Hk, HD, P, seed=0, S=1, poison=None):
        g = rng(seed)
        self.groups, self.lens, self.H = groups, lens, (Hq, Hk, HD, P)
        R = sum(n for n, _ in groups)
        assert R == len(lens)
        B = -(-R // S)
        MP = max(1, -(-max(lens) // P)) + 1
        seqs, n, tails, r = [], 0, [], 0
        for rows, pre in groups:
            first = None
            for k in range(rows):
                m = max(lens[r - r % S:r - r % S + S])  # what the sequence holds
                if r % S == 0:
                    full = pre // P if m >= pre and first is not None else 0
                    own = -(-max(lens[r:r + S]) // P) - full
                    pages = (first[:full] if full else []) + list(range(n, n + own))
                    n += own
                    if m >= pre and pre:
                        if first is None:
                            first = pages
                        elif pre % P:
                            tails.append((first[pre // P], pages[pre // P], pre % P))
                    seqs.append(pages)
                r += 1
        order = g.permutation(n + 2)
        self.pool = randn16(seed + 1, 2, n + 2, Hk, P, HD)
        for a, b, k in tails:
            self.pool[:, order[b], :, :k] = self.pool[:, order[a], :, :k]
        self.table = np.full((B, MP), -1, np.int32)
        for b, pages in enumerate(seqs):
            self.table[b, :len(pages)] = order[pages]
        if poison is not None:  # slots that nobody attends
            used = np.zeros((n + 2, P), bool)
            for r, m in enumerate(lens):
                t = np.arange(m)
                used[self.table[r // S, t // P], t % P] = True
            self.pool[:, ~used.all(1)] = np.where(used[~used.all(1)][None, :, None, :, None], self.pool[:, ~used.all(1)], poison)
        self.q = randn16(seed + 2, R, Hq * HD)
        self.S, self.R = S, R

    def want(self, scale):
        """(o, bound) in float64, the bound of each value derived below."""
        Hq, Hk, HD, P = self.H
        G = Hq // Hk
        o, tol = np.zeros((self.R, Hq * HD)), np.zeros((self.R, Hq * HD))
        for r, m in enumerate(self.lens):
            if not m:
                continue
            t = np.arange(m)
            k, v = (self.pool[i][self.table[r // self.S, t // P], :, t % P].astype(np.float64) for i in (0, 1))
            for h in range(Hq):
                q = self.q[r, h * HD:(h + 1) * HD].astype(np.float64)
                s = k[:, h // G] @ q * scale
                p = np.exp(s - s.max())
                l = p.sum()
                out = p @ v[:, h // G] / l
                # scores: HD products and sums in fp32, two more roundings in the exponent's argument; the exponential
                # 2^-22; probabilities to fp16 (2^-11, or 2^-25 below the normal range); fp32 sums over the slots and the
                # parts; one rounding to fp16
                ds = (HD + 8) * 2.0 ** -24 * (np.abs(k[:, h // G]) @ np.abs(q)).max() * scale + 2.0 ** -24 * 4 * np.abs(s).max()
                rel = 2.0 ** -11 + 2 * ds + 2.0 ** -20
                avg = p @ np.abs(v[:, h // G]) / l
                at = slice(h * HD, (h + 1) * HD)
                o[r, at] = out
                tol[r, at] = 2.0 ** -11 * np.abs(out) + rel * avg + 2.0 ** -25 * (1 + m * np.abs(v[:, h // G]).max() / l)
        return o, tol

    def run(self, dev, max_len=None, scale=None, plan=None, out=None, share=True):
        import torch
        from estudiocanciones_amd.kernels import paged_attn, paged_attn_plan
        Hq, Hk, HD, P = self.H
        T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        kv = T(self.pool)
        plan = plan or paged_attn_plan(self.groups, Hq, Hk, HD, max_len or self.table.shape[1] * P, dev, share)
        pos = T(np.array(self.lens, np.int64) - 1)
        return paged_attn(T(self.q), kv[0], kv[1], T(self.table), pos, plan, S=self.S, scale=scale, out=out)

    def check(self, dev, **kw):
        """With shared parts, without them (split and joined, or a workgroup per row), and as the rule has it."""
        want, tol = self.want(kw.get("scale") or 1 / math.sqrt(self.H[2]))
        for share in (True, False, None):
            got = self.run(dev, share=share, **kw).float().cpu().numpy()
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (share, int(bad.sum()), np.abs(got - want).max(), np.argwhere(bad)[:4])
            for r, m in enumerate(self.lens):
                if not m:
                    assert (got[r] == 0).all()


HEADS = [(24, 8, 128), (8, 2, 128), (12, 2, 64), (5, 5, 64), (16, 1, 128), (8, 2, 256), (32, 2, 64), (6, 2, 256)]


@pytest.mark.parametrize("Hq,Hk,HD", HEADS)
@pytest.mark.parametrize("P", [16, 64])
def test_groups_of_every_shape(dev, Hq, Hk, HD, P):
    # one row alone, a pair, nine rows with a prefix that ends inside a page, rows with nothing in common; an idle row in
    # front of its group, a row shorter than the prefix, lengths of one and around the borders of tiles and pages
    groups = [(1, 0), (2, 31), (9, 277), (3, 0), (1, 50)]
    lens = [1, 32, 31 + 64, 0, 277, 278, 300, 277 + 130, 276, 277 + 31, 1, 511, 16, 17, 129, 55]
    Batch(groups, lens, Hq, Hk, HD, P, seed=Hq + P).check(dev)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2049])
def test_one_row_of_any_length(dev, n):
    Batch([(1, 0)], [n], 6, 2, 128, 32, seed=n).check(dev)
    Batch([(2, n)], [n, n + 1], 6, 2, 128, 16, seed=n).check(dev)


@pytest.mark.parametrize("rows", [2, 5, 6, 10, 11, 21, 22, 43, 64])
def test_groups_of_any_size(dev, rows):
    """3 query heads per kv head: one, two and four tiles of columns, and several shared parts side by side."""
    lens = [700 + (37 * r) % 90 for r in range(rows)]
    Batch([(rows, 700)], lens, 3, 1, 128, 64, seed=rows).check(dev)


def test_many_parts_and_a_long_table(dev):
    b = Batch([(3, 5000), (4, 33)], [5001, 9000, 5130, 34, 8190, 33, 0], 6, 2, 128, 128, seed=5)
    b.check(dev, max_len=9216)
    b.check(dev, max_len=9216, scale=0.5)


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_what_is_not_attended_does_not_matter(dev, poison):
    groups, lens = [(4, 100), (2, 0)], [101, 0, 100, 150, 7, 33]
    Batch(groups, lens, 12, 4, 128, 64, seed=9, poison=poison).check(dev)


@pytest.mark.parametrize("long", [False, True])
def test_split_rows_without_sharing(dev, long):
    """Rows too few or too long for a workgroup each: split over their slots and joined."""
    lens = [4100, 1, 3000, 0] if long else [900, 700, 31, 32]
    Batch([(2, 500), (2, 0)] if not long else [(4, 0)], lens, 6, 2, 128, 64, seed=3).check(dev, max_len=16384)


def test_a_short_row_does_not_see_its_groups_slots(dev):
    """A row that does not hold the whole prefix takes nothing from the shared parts: a NaN in them stays out of it."""
    b = Batch([(3, 96)], [97, 40, 120], 6, 2, 64, 32, seed=4)
    b.pool[1, b.table[0, 2]] = np.nan  # slots 64 .. 95 of the pages that rows 0 and 2 share
    want, tol = b.want(1 / 8)
    got = b.run(dev).float().cpu().numpy()
    assert np.isnan(got[[0, 2]]).all() and (np.abs(got[1] - want[1]) <= tol[1]).all()


def test_a_query_that_is_no_number_gives_none(dev):
    b = Batch([(3, 600)], [601, 700, 650], 6, 2, 128, 32, seed=4)
    b.q[1, 3 * 128 + 5] = np.nan
    want, tol = b.want(1 / math.sqrt(128))
    got = b.run(dev).float().cpu().numpy()
    bad = np.zeros(got.shape, bool)
    bad[1, 3 * 128:4 * 128] = True
    assert np.isnan(got[bad]).all() and (np.abs(got - want) <= tol)[~bad].all()


def test_rows_of_one_sequence(dev):
    """S = 3 rows per sequence at consecutive slots."""
    lens = [201, 202, 203, 64, 65, 66, 1, 2, 3]
    Batch([(6, 0), (3, 0)], lens, 6, 2, 128, 32, seed=11, S=3).check(dev)


def test_large_scores(dev):
    b = Batch([(5, 300)], [301, 310, 333, 400, 300], 6, 2, 128, 64, seed=6)
    b.q *= np.float16(30)
    b.check(dev)


def test_rows_behind_the_plan_and_strides(dev):
    import torch
    from estudiocanciones_amd.kernels import paged_attn, paged_attn_plan
    b = Batch([(3, 64)], [70, 80, 64], 6, 2, 64, 16, seed=2)
    want, tol = b.want(1 / 8)
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    kv = T(b.pool)
    plan = paged_attn_plan(b.groups, 6, 2, 64, 200, dev)
    wide = torch.full((5, 10 * 64), float("nan"), dtype=torch.float16, device=dev)
    wide[:3, :384] = T(b.q)
    tab = torch.full((5, b.table.shape[1] + 3), 10 ** 6, dtype=torch.int32, device=dev)
    tab[:3, :b.table.shape[1]] = T(b.table)
    pos = torch.tensor([69, 79, 63, 10 ** 9, -5], device=dev)
    out = torch.full((5, 384), 3.0, dtype=torch.float16, device=dev)
    got = paged_attn(wide[:, :384], kv[0], kv[1], tab[:, :b.table.shape[1]], pos, plan, out=out)
    assert got is out and (out[3:] == 3).all()
    assert (np.abs(out[:3].float().cpu().numpy() - want) <= tol).all()


def test_the_same_bits_each_time_and_in_graphs(dev):
    """Two graphs of one plan, replayed in turn with eager calls between them."""
    import torch
    from estudiocanciones_amd.kernels import paged_attn, paged_attn_plan
    b = Batch([(6, 900)], [1000, 901, 900, 1400, 0, 950], 24, 8, 128, 64, seed=8)
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    kv, table, q = T(b.pool), T(b.table), T(b.q)
    pos = T(np.array(b.lens, np.int64) - 1)
    plan = paged_attn_plan(b.groups, 24, 8, 128, 1536, dev, share=True)
    first = paged_attn(q, kv[0], kv[1], table, pos, plan).clone()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(paged_attn(q, kv[0], kv[1], table, pos, plan))
        graphs.append(gr)
    for k in range(4):
        outs[k % 2].zero_()
        graphs[k % 2].replay()
        assert torch.equal(outs[k % 2], first)
        assert torch.equal(paged_attn(q, kv[0], kv[1], table, pos, plan), first)
    # a replay reads the positions as they are then
    pos.sub_(1)
    want = paged_attn(q, kv[0], kv[1], table, pos, plan)
    graphs[0].replay()
    assert torch.equal(outs[0], want) and not torch.equal(want, first)


def test_on_another_stream(dev):
    import torch
    b = Batch([(4, 500)], [501, 700, 650, 520], 24, 8, 128, 64, seed=8)
    first = b.run(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = b.run(dev)
    s.synchronize()
    assert torch.equal(first, other)


def test_two_calls_at_once(dev):
    """One plan on two streams, each with queries of its own."""
    import torch
    from estudiocanciones_amd.kernels import paged_attn, paged_attn_plan
    b = Batch([(8, 2000), (4, 300)], [2000 + 40 * r for r in range(8)] + [300, 301, 420, 777], 24, 8, 128, 64, seed=8)
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    kv, table, pos = T(b.pool), T(b.table), T(np.array(b.lens, np.int64) - 1)
    qs = [T(b.q), T(b.q[::-1])]
    plan = paged_attn_plan(b.groups, 24, 8, 128, 4096, dev, share=True)
    want = [paged_attn(q, kv[0], kv[1], table, pos, plan) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attn(qs[i], kv[0], kv[1], table, pos, plan))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])


def test_refusals(dev):
    import torch
    from estudiocanciones_amd.kernels import paged_attn, paged_attn_plan, paged_write
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    plan = paged_attn_plan([(2, 16)], 4, 2, 64, 64, dev)
    good = dict(q=h(2, 256), kp=h(9, 2, 16, 64), vp=h(9, 2, 16, 64), table=torch.zeros(2, 4, dtype=torch.int32, device=dev),
                pos=torch.zeros(2, dtype=torch.long, device=dev), plan=plan)
    assert paged_attn(**good).shape == (2, 256)
    for bad in (dict(q=h(1, 256)), dict(q=h(2, 192)), dict(q=h(2, 512)[:, ::2]), dict(q=h(3, 264)[1:, 4:260]),
                dict(kp=h(9, 2, 24, 64), vp=h(9, 2, 24, 64)), dict(kp=h(9, 1, 16, 64), vp=h(9, 1, 16, 64)),
                dict(vp=h(8, 2, 16, 64)), dict(kp=h(9, 2, 64, 16).transpose(2, 3)), dict(table=good["table"][:1]),
                dict(table=good["table"].t()), dict(table=good["table"].cpu()), dict(pos=good["pos"][:1]), dict(scale=0.0),
                dict(scale=float("nan")), dict(out=h(2, 128)), dict(S=0)):
        with pytest.raises(ValueError):
            paged_attn(**{**good, **bad})
    for bad in (dict(q=h(2, 256).float()), dict(pos=good["pos"].int()), dict(kp=h(9, 2, 16, 64).bfloat16())):
        with pytest.raises(TypeError):
            paged_attn(**{**good, **bad})
    w = dict(qkv=h(2, 512), kp=good["kp"], vp=good["vp"], table=good["table"], pos=good["pos"], S=1, Hq=4, Hk=2)
    for bad in (dict(S=0), dict(Hk=1), dict(qkv=h(3, 512)), dict(rope=torch.zeros(64, 30, 2, device=dev)), dict(table=good["table"][:1])):
        with pytest.raises(ValueError):
            paged_write(**{**w, **bad})


def test_rows_of_one_sequence_share_a_prefix(dev):
    """S = 2: a group of three sequences with two rows each, one of them behind the prefix's end and one before it."""
    Batch([(6, 100)], [130, 131, 101, 102, 99, 100], 6, 2, 128, 32, seed=12, S=2).check(dev)


def test_pool_offsets_past_32_bits(dev):
    """Pages at the end of a pool of more than 2^32 values a plane: the write, the attention and a fork reach them."""
    import torch
    from estudiocanciones_amd.kernels import page_fork, paged_attn, paged_attn_plan, paged_write
    NP, P, HD, n = 263000, 128, 128, 300
    kv = torch.empty(1, 2, NP, 1, P, HD, dtype=torch.float16, device=dev)
    assert kv[0, 0].numel() > 1 << 32
    ref = torch.ones(NP, dtype=torch.int32, device=dev)
    ref[[NP - 9, NP - 5]] = 0
    table = torch.full((3, 3), -1, dtype=torch.int32, device=dev)
    table[0] = torch.tensor([NP - 1, 7, NP - 2], device=dev)
    length = torch.tensor([n, 0, 0], device=dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.from_numpy(randn16(1, n, 5 * HD)).to(dev)
    paged_write(x, kv[0, 0], kv[0, 1], table[:1], torch.arange(n, device=dev), n, 3, 1)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    page_fork(kv, ref, table, length, i32(0, 0), i32(1, 2), err)
    assert err.item() == 0 and table[1:, 2].tolist() == [NP - 9, NP - 5]
    q = torch.from_numpy(randn16(2, 3, 3 * HD)).to(dev)
    plan = paged_attn_plan([(3, n)], 3, 1, HD, 3 * P, dev, share=True)
    o = paged_attn(q, kv[0, 0], kv[0, 1], table, torch.full((3,), n - 1, device=dev), plan).cpu().double().reshape(3, 3, HD)
    k, v = (x[:, i * HD:(i + 1) * HD].cpu().double() for i in (3, 4))
    s = q.cpu().double().reshape(3, 3, HD) @ k.T / HD ** 0.5
    want = s.softmax(-1) @ v
    ds = (HD + 8) * 2.0 ** -24 * float((q.cpu().double().abs().reshape(9, HD) @ k.abs().T).max()) / HD ** 0.5 + 2.0 ** -20
    tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * ds) * (s.softmax(-1) @ v.abs()) + 2.0 ** -20
    assert ((o - want).abs() <= tol).all()


def test_prefixes_and_rows_past_the_plans_length(dev):
    """A prefix longer than any row can hold (nobody attends all of it), rows that hold more than the plan was made for."""
    Batch([(1, 500), (3, 400)], [0, 20, 0, 33], 6, 2, 128, 16, seed=21).check(dev)
    Batch([(2, 50), (2, 0)], [61, 300, 1000, 52], 6, 2, 64, 32, seed=22).check(dev, max_len=60)
