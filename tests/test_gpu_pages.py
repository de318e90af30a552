"""Pages of a KV cache on the device (page_free, page_fork, page_extend, page_compact, paged_write) against the same
operations on Python lists: page numbers, counts and copied bits are equal or wrong."""
import numpy as np
import pytest

from helpers import randn16, rng

pytestmark = pytest.mark.gpu


class Model:
    """The page state as the operations define it."""

    def __init__(self, kv, B, MP):
        self.kv = kv.copy()  # uint16 [layers, 2, NP, Hk, P, HD]
        self.P = kv.shape[4]
        self.ref = [0] * kv.shape[2]
        self.table = [[-1] * MP for _ in range(B)]
        self.length = [0] * B

    def pages(self, n):
        return -(-n // self.P)

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.length):
                for j in range(self.pages(self.length[s])):
                    self.ref[self.table[s][j]] -= 1
                    self.table[s][j] = -1
                self.length[s] = 0

    def extend(self, pos):
        for b, p in enumerate(pos):
            if p >= self.length[b]:
                for j in range(self.pages(self.length[b]), self.pages(p + 1)):
                    k = self.ref.index(0)
                    self.ref[k], self.table[b][j] = 1, k
                self.length[b] = p + 1

    def fork(self, src, dst):
        n = [self.length[s] for s in src]
        for s, d, m in zip(src, dst, n):
            full, tail = divmod(m, self.P)
            if tail:
                k = self.ref.index(0)
                self.ref[k], self.table[d][full] = 1, k
                self.kv[:, :, k, :, :tail] = self.kv[:, :, self.table[s][full], :, :tail]
            for j in range(full):
                self.table[d][j] = self.table[s][j]
                self.ref[self.table[s][j]] += 1
            self.length[d] = m


class State:
    def __init__(self, dev, layers, pages, Hk, P, HD, B, MP, seed=0):
        import torch
        self.np = randn16(seed, layers, 2, pages, Hk, P, HD)
        self.kv = torch.from_numpy(self.np).to(dev)
        self.ref = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.table = torch.full((B, MP), -1, dtype=torch.int32, device=dev)
        self.length = torch.zeros(B, dtype=torch.int64, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self.dev, self.P = dev, P

    def i32(self, v):
        import torch
        return torch.tensor(v, dtype=torch.int32, device=self.dev)

    def i64(self, v):
        import torch
        return torch.tensor(v, dtype=torch.int64, device=self.dev)

    def extend(self, pos):
        from estudiocanciones_amd.kernels import page_extend
        page_extend(self.ref, self.table, self.length, self.i64(pos), self.P, self.err)

    def fork(self, src, dst):
        from estudiocanciones_amd.kernels import page_fork
        page_fork(self.kv, self.ref, self.table, self.length, self.i32(src), self.i32(dst), self.err)

    def free(self, seqs):
        from estudiocanciones_amd.kernels import page_free
        page_free(self.ref, self.table, self.length, self.i32(seqs), self.P, self.err)

    def same(self, m, what, err=0):
        assert self.err.item() == err, (what, self.err.item())
        assert self.ref.tolist() == m.ref, what
        assert self.table.tolist() == m.table, what
        assert self.length.tolist() == m.length, what
        assert np.array_equal(self.kv.cpu().numpy().view(np.uint16), m.kv), what


SHAPES = [  # layers, pages, Hk, P, HD, sequences, pages of a sequence
    (1, 9, 1, 1, 8, 3, 4), (2, 40, 2, 16, 64, 6, 7), (3, 1500, 1, 5, 24, 7, 300), (2, 2100, 1, 16, 8, 40, 60),
    (1, 30, 3, 128, 128, 4, 5)]


@pytest.mark.parametrize("shape", SHAPES)
def test_operations_in_turn(dev, shape):
    layers, pages, Hk, P, HD, B, MP = shape
    st = State(dev, *shape)
    m = Model(st.np.view(np.uint16), B, MP)
    g = rng(3)
    for step in range(40):
        op = ["extend", "fork", "free", "extend"][step % 4]
        if op == "extend":
            pos = [int(min(MP * P - 1, m.length[b] + g.integers(-2, 2 * P + 1))) for b in range(B)]
            need = sum(max(0, m.pages(max(p + 1, n)) - m.pages(n)) for p, n in zip(pos, m.length))
            if need > m.ref.count(0):
                pos = [-1] * B
            m.extend(pos)
            st.extend(pos)
            st.extend(pos)  # the same again changes nothing
        elif op == "fork":
            empty = [b for b in range(B) if m.length[b] == 0]
            held = [b for b in range(B) if m.length[b]]
            n = min(len(empty), m.ref.count(0), 5)
            if not held or not n:
                continue
            dst = [int(d) for d in g.permutation(empty)[:n]]
            src = [int(held[g.integers(len(held))]) for _ in range(n)]
            m.fork(src, dst)
            st.fork(src, dst)
        else:
            seqs = [int(s) for s in g.integers(0, B, 2)]  # the same sequence twice at times
            m.free(seqs)
            st.free(seqs)
        st.same(m, (step, op))


def test_fork_of_many_and_of_nothing(dev):
    st = State(dev, 2, 1300, 1, 16, 16, 700, 3)
    m = Model(st.np.view(np.uint16), 700, 3)
    for pos in ([20, 31] + [-1] * 698,):
        m.extend(pos)
        st.extend(pos)
    src, dst = [i % 3 for i in range(690)], list(range(3, 693))  # sequence 2 holds nothing; 1 has no partial page
    m.fork(src, dst)
    st.fork(src, dst)
    st.same(m, "fork")
    m.free(dst)
    st.free(dst)
    st.same(m, "free")
    assert sum(r > 0 for r in m.ref) == 4


@pytest.mark.parametrize("what", ["index", "target", "twice", "full", "table", "extend-full", "free-index"])
def test_what_cannot_be_done_changes_nothing(dev, what):
    st = State(dev, 1, 8, 1, 16, 8, 5, 4)
    m = Model(st.np.view(np.uint16), 5, 4)
    pos = [40, 16, -1, -1, -1]  # 3 + 2 pages, both with a partial one
    m.extend(pos)
    st.extend(pos)
    if what == "index":
        st.fork([0, 5], [2, 3])
        st.same(m, what, 1)
    elif what == "target":
        st.fork([0, 0], [2, 1])
        st.same(m, what, 2)
    elif what == "twice":
        st.fork([0, 1], [2, 2])
        st.same(m, what, 2)
    elif what == "full":
        st.fork([0, 0, 1, 1], [2, 3, 4, 4])
        st.same(m, what, 2 | 4)
    elif what == "table":
        st.extend([64, -1, -1, -1, -1])
        st.same(m, what, 8)
    elif what == "extend-full":
        st.extend([-1, -1, 33, 15, -1])
        st.same(m, what, 4)
    else:
        st.free([-1, 1, 5])  # the others are freed
        m.free([1])
        st.same(m, what, 1)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("room", [0, 5, -1])
def test_compact(dev, shape, room):
    import torch
    from estudiocanciones_amd.kernels import page_compact
    layers, pages, Hk, P, HD, B, MP = shape
    st = State(dev, *shape)
    m = Model(st.np.view(np.uint16), B, MP)
    m_pos = [P + 1] * (B // 2) + [-1] * (B - B // 2)
    for op, v in (("extend", m_pos), ("free", [0]), ("fork", ([B // 2 - 1], [B - 1])), ("extend", [2 * P] + [-1] * (B - 1))):
        if op == "fork" and B // 2 - 1 == 0:
            continue
        getattr(m, op)(*(v if op == "fork" else (v,)))
        getattr(st, op)(*(v if op == "fork" else (v,)))
    st.same(m, "before")
    used = [p for p in range(pages) if m.ref[p]]
    n2 = max(1, len(used) + room)
    kv2 = torch.full((layers, 2, n2, Hk, P, HD), 7.0, dtype=torch.float16, device=dev)
    ref2 = torch.full((n2,), 9, dtype=torch.int32, device=dev)
    table2, length2 = torch.full_like(st.table, 5), torch.full_like(st.length, 5)
    page_compact(st.kv, st.ref, st.table, st.length, kv2, ref2, table2, length2, st.err)
    if len(used) > n2:
        st.same(m, "refused", 16)
        assert (kv2 == 7).all() and (ref2 == 9).all() and (table2 == 5).all() and (length2 == 5).all()
        return
    st.same(m, "after")
    want = np.full((layers, 2, n2, Hk, P, HD), 7.0, np.float16).view(np.uint16)
    want[:, :, :len(used)] = m.kv[:, :, used]
    assert np.array_equal(kv2.cpu().numpy().view(np.uint16), want)
    assert ref2.tolist() == [m.ref[p] for p in used] + [0] * (n2 - len(used))
    new = {p: k for k, p in enumerate(used)}
    assert table2.tolist() == [[new.get(p, -1) for p in t] for t in m.table]
    assert length2.tolist() == m.length


def test_captured_and_replayed(dev):
    """free, fork, extend and compact in a graph, replayed with eager work between the replays."""
    import torch
    from estudiocanciones_amd.kernels import page_compact, page_extend, page_fork, page_free
    st = State(dev, 2, 30, 2, 16, 64, 6, 5)
    m = Model(st.np.view(np.uint16), 6, 5)
    st.extend([35, -1, -1, -1, -1, -1])
    m.extend([35, -1, -1, -1, -1, -1])
    src, dst = st.i32([0, 0, 0]), st.i32([1, 3, 4])
    pos = st.i64([-1, 48, -1, 36, 60, -1])
    out = [torch.zeros(2, 2, 20, 2, 16, 64, dtype=torch.float16, device=dev), torch.zeros(20, dtype=torch.int32, device=dev),
           torch.zeros_like(st.table), torch.zeros_like(st.length)]

    def step():
        page_free(st.ref, st.table, st.length, dst, 16, st.err)
        page_fork(st.kv, st.ref, st.table, st.length, src, dst, st.err)
        page_extend(st.ref, st.table, st.length, pos, 16, st.err)
        page_compact(st.kv, st.ref, st.table, st.length, *out, st.err)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    m.fork([0, 0, 0], [1, 3, 4])
    m.extend([-1, 48, -1, 36, 60, -1])
    st.same(m, "eager")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        # other sequences come and go between the replays
        st.extend([-1, -1, 20 + k, -1, -1, 3])
        m.extend([-1, -1, 20 + k, -1, -1, 3])
        graph.replay()
        m.free([1, 3, 4])
        m.fork([0, 0, 0], [1, 3, 4])
        m.extend([-1, 48, -1, 36, 60, -1])
        st.same(m, k)
        assert out[1].sum().item() == sum(m.ref) and out[3].tolist() == m.length
        st.free([2, 5])
        m.free([2, 5])


# ---------------------------------------------------------------- the write of rows into pages
def _rope_np(x, t):
    """x [M, H, HD] fp16, t [M, HD/2, 2] fp32 -> float64 rotation of the interleaved pairs."""
    a, b = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    c, s = t[:, None, :, 0].astype(np.float64), t[:, None, :, 1].astype(np.float64)
    out = np.empty(x.shape)
    out[..., 0::2], out[..., 1::2] = a * c - b * s, b * c + a * s
    return out


@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("S,B,Hq,Hk,HD,P,MP,pad", [(1, 1, 1, 1, 8, 16, 1, 0), (1, 8, 24, 8, 128, 64, 3, 0),
                                                   (7, 3, 6, 2, 64, 16, 4, 24), (130, 2, 5, 5, 256, 32, 9, 8),
                                                   (3, 5, 4, 4, 24, 5, 7, 0)])
def test_paged_write(dev, rope, S, B, Hq, Hk, HD, P, MP, pad):
    import torch
    from estudiocanciones_amd.kernels import paged_write
    M, NP, W, L = S * B, B * MP + 3, (Hq + 2 * Hk) * HD, MP * P
    g = rng(S + HD)
    wide = randn16(1, M, W + pad)
    pool = randn16(2, 2, NP, Hk, P, HD)
    table = g.permutation(NP)[:B * MP].reshape(B, MP).astype(np.int32)
    pos = np.concatenate([np.sort(g.permutation(L)[:S]) for _ in range(B)]).astype(np.int64) if S <= L else None
    ang = g.standard_normal((L, HD // 2)) * 10
    rt = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    dead = []
    if M > 2:  # a slot outside the table, none, and one whose page is not there
        pos[M - 1], pos[M // 2] = L, -1
        table[0, pos[0] // P] = -1
        dead = [m for m in range(M) if not 0 <= pos[m] < L or table[m // S, pos[m] // P] < 0]
        assert dead
    T = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    qkv, kv = T(wide)[:, :W], T(pool)
    q = paged_write(qkv, kv[0], kv[1], T(table), T(pos), S, Hq, Hk, rope=T(rt) if rope else None)
    x = wide[:, :W].reshape(M, Hq + 2 * Hk, HD)
    want, exactly = pool.astype(np.float64), np.ones(pool.shape, bool)
    turned = _rope_np(x[:, :Hq + Hk], rt[np.clip(pos, 0, L - 1)])
    for m in range(M):
        if m not in dead:
            at = (table[m // S, pos[m] // P], slice(None), pos[m] % P)
            want[(0, *at)] = turned[m, Hq:] if rope else x[m, Hq:Hq + Hk]
            want[(1, *at)] = x[m, Hq + Hk:]
            exactly[(0, *at)] = not rope
    got = kv.cpu().numpy().astype(np.float64)
    assert np.array_equal(got[exactly], want[exactly])
    # a rotated value: two fp32 products and their sum (each within 2^-24 of |x| sqrt 2 at most), one fp16 rounding
    big = 2.0 ** -22 * np.abs(x.astype(np.float64)).max()
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + big + 2.0 ** -25).all()
    if rope:
        qw = turned[:, :Hq].reshape(M, -1)
        assert (np.abs(q.cpu().numpy() - qw) <= 2.0 ** -11 * np.abs(qw) + big + 2.0 ** -25).all()
    else:
        assert q is None
