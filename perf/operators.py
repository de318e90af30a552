"""The operators of one prompt shared by many takes, as cases that can be timed and checked.

Four operators that serve together: pages of a KV cache (forked, extended, freed, compacted), RoPE with the
write of keys and values into pages, decode attention that reads a group's shared prefix once, and the
product of int8 activations (one scale per row) with int8 weights (one scale per output channel).

``own`` chooses between the framework's calls and their plain forms: elementary torch operations in 32 bits,
rounded once.  Sizes are those of the model's configurations (the 3B backbone's 28 layers of 24 query heads
on 8 kv heads of 128, the 1024-wide depth decoder's 8 on 2) and generic ones.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # two takes of the depth decoder's shape start from a short prompt: small pages, the latency of the calls
        {"name": "restart_2takes", "kind": "restart", "layers": 4, "hk": 2, "hd": 128, "page": 16, "groups": 1,
         "takes": 2, "prompt": 77, "others": 3},
        # 16 takes with guidance start again from prompts of 1000 tokens: 32 tails of 40 slots copied in 28 layers
        {"name": "restart_16takes_guided", "kind": "restart", "layers": 28, "hk": 8, "hd": 128, "page": 64,
         "groups": 2, "takes": 16, "prompt": 1000, "others": 2},
        # a server that closed songs moves the live pages of 28 layers into a smaller pool
        {"name": "compact_28layers", "kind": "compact", "layers": 28, "hk": 8, "hd": 128, "page": 64, "seqs": 12,
         "slots": 800, "pages": 256, "shared": 4},
        # keys and values of one frame of 4 takes with guidance
        {"name": "write_step_8rows", "kind": "write", "seqs": 8, "rows": 1, "start": 750, "hq": 24, "hk": 8,
         "hd": 128, "page": 64, "rope": False},
        # a long prompt and its unconditional twin: RoPE and the write of 2 x 4000 rows, from the middle of a page
        {"name": "write_prompt_2x4000", "kind": "write", "seqs": 2, "rows": 4000, "start": 40, "hq": 24, "hk": 8,
         "hd": 128, "page": 64, "rope": True},
        # one frame of 4 takes with guidance, one minute into a song (the two prompts of 256 slots shared)
        {"name": "attn_8rows_kv750", "kind": "attn", "groups": 2, "takes": 4, "hq": 24, "hk": 8, "hd": 128,
         "page": 64, "prefix": 256, "own": 494, "ragged": False, "idle": 0},
        # 16 continuations, with guidance, of a song of 4096 slots: most of what each row attends is shared
        {"name": "attn_32rows_prefix4096", "kind": "attn", "groups": 2, "takes": 16, "hq": 24, "hk": 8, "hd": 128,
         "page": 64, "prefix": 4096, "own": 1024, "ragged": True, "idle": 0},
        # 32 takes with guidance near the end of the backbone's 8192 slots (the largest attention)
        {"name": "attn_64rows_prefix7000", "kind": "attn", "groups": 2, "takes": 32, "hq": 24, "hk": 8, "hd": 128,
         "page": 64, "prefix": 7000, "own": 600, "ragged": True, "idle": 3},
        # other heads, small pages, prefixes that end inside a page, a finished take whose row attends nothing
        {"name": "attn_9rows_odd", "kind": "attn", "groups": 3, "takes": 3, "hq": 12, "hk": 2, "hd": 64,
         "page": 16, "prefix": 277, "own": 300, "ragged": True, "idle": 1},
        # the gate and up projections of one frame of 4 takes with guidance (norm, product, SiLU)
        {"name": "a8_8rows_silu", "kind": "a8", "rows": 8, "n": 16384, "k": 3072, "norm": True, "silu": True, "res": False},
        # the same for a prompt of 2048 rows (the largest product)
        {"name": "a8_2048rows_silu", "kind": "a8", "rows": 2048, "n": 16384, "k": 3072, "norm": True, "silu": True, "res": False},
        # a short prompt's down projection with its residual, ragged rows
        {"name": "a8_187rows_res", "kind": "a8", "rows": 187, "n": 3072, "k": 8192, "norm": False, "silu": False, "res": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["restart", "compact", "write", "attn", "attn", "attn", "a8", "a8", "a8"])
    if kind in ("restart", "compact"):
        layers, hk, hd = rng.choice([(4, 2, 128), (28, 8, 128), (6, 3, 64), (8, 4, 256)])
        page = rng.choice([16, 32, 64, 128]) if layers < 28 else rng.choice([16, 32, 64])
        if kind == "restart":
            return {"kind": kind, "layers": layers, "hk": hk, "hd": hd, "page": page, "groups": rng.randint(1, 3),
                    "takes": _log_int(rng, 1, 12), "prompt": _log_int(rng, 1, 1000), "others": rng.randint(0, 4)}
        seqs, slots = rng.randint(1, 12), _log_int(rng, 5, 700)
        shared = rng.randint(0, 4)
        need = shared + seqs * -(-slots // page)
        return {"kind": kind, "layers": layers, "hk": hk, "hd": hd, "page": page, "seqs": seqs, "slots": slots,
                "pages": need + rng.randint(1, 60), "shared": shared}
    heads = [(24, 8, 128), (24, 8, 128), (8, 2, 128), (12, 2, 64), (5, 5, 64), (16, 1, 128), (8, 2, 256)]
    if kind == "write":
        hq, hk, hd = rng.choice(heads)
        return {"kind": kind, "seqs": rng.randint(1, 8), "rows": _log_int(rng, 1, 900), "start": _log_int(rng, 1, 1000),
                "hq": hq, "hk": hk, "hd": hd, "page": rng.choice([16, 32, 64, 128]), "rope": rng.random() < 0.6}
    if kind == "attn":
        hq, hk, hd = rng.choice(heads)
        return {"kind": kind, "groups": rng.randint(1, 3), "takes": _log_int(rng, 1, 20), "hq": hq, "hk": hk, "hd": hd,
                "page": rng.choice([16, 32, 64, 128]), "prefix": _log_int(rng, 1, 6000), "own": _log_int(rng, 1, 1000),
                "ragged": rng.random() < 0.7, "idle": rng.randint(0, 1)}
    n, k = rng.choice([(5120, 3072), (3072, 3072), (3072, 8192), (8197, 1024), (1024, 8192), (1001, 192), (4608, 1536)])
    silu = rng.random() < 0.3
    return {"kind": kind, "rows": _log_int(rng, 1, 3000), "n": 2 * (n // 2) if silu else n, "k": k,
            "norm": rng.random() < 0.5, "silu": silu, "res": not silu and rng.random() < 0.5}


# ---------------------------------------------------------------- sizes of a case
def _cdiv(a, b):
    return -(-a // b)


def _prefix(case, g):
    """Shared slots of group g: the later groups' prompts are shorter where rows are ragged."""
    p = case["prefix"]
    return p - p * g // (2 * case["groups"]) if case["ragged"] else p


def _lengths(case):
    """Slots that each row of an attention case attends."""
    out = []
    rows = case["groups"] * case["takes"]
    for r in range(rows):
        n = case["own"]
        if case["ragged"]:
            n = 1 + int((n - 1) * math.fmod(0.618034 * (r + 1), 1.0))
        out.append(0 if r >= rows - case["idle"] else _prefix(case, r // case["takes"]) + n)
    return out


def _compact_lengths(case):
    """Slots of each sequence behind the shared pages: from a third of ``slots`` up to all of them."""
    return [max(1, case["slots"] - case["slots"] * 2 * i // (3 * case["seqs"])) for i in range(case["seqs"])]


# ---------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + salt)


def _rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16).mul_(scale)


def _perm(seed, salt, n):
    return torch.randperm(n, generator=torch.Generator().manual_seed(1000003 * (seed + 1) + salt)).tolist()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _i64(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def _prepare_pages(case, seed):
    """A pool of pages in use by prompts (or shared pages), by the takes and by other sequences, in any order."""
    P = case["page"]
    lens, tabs = [], []
    if case["kind"] == "restart":
        per, seqs = _cdiv(case["prompt"], P), case["groups"] * (1 + case["takes"]) + case["others"]
        order = _perm(seed, 2, case["groups"] * (per + 2 * case["takes"]) + case["others"] * 3 + 5)
        for s in range(seqs):
            n = case["prompt"] if s < case["groups"] else 0 if s < seqs - case["others"] else 2 * P + 1
            lens.append(n)
            tabs.append([order.pop() for _ in range(_cdiv(n, P))])
        width, pages = per + 2, case["groups"] * (per + 2 * case["takes"]) + case["others"] * 3 + 5
        width = max(width, 3)
    else:
        order = _perm(seed, 2, case["pages"])
        common = [order.pop() for _ in range(case["shared"])]
        for n in _compact_lengths(case):
            lens.append(case["shared"] * P + n)
            tabs.append(common + [order.pop() for _ in range(_cdiv(n, P))])
        width, pages = case["shared"] + _cdiv(case["slots"], P) + 1, case["pages"]
    ref = [0] * pages
    for t in tabs:
        for p in t:
            ref[p] += 1
    kv = _rand(_gen(seed, 1), case["layers"], 2, pages, case["hk"], P, case["hd"])
    st = {"kv": kv, "ref": _i32(ref), "table": _i32([t + [-1] * (width - len(t)) for t in tabs]), "length": _i64(lens),
          "err": torch.zeros(1, dtype=torch.int32, device=DEV)}
    if case["kind"] == "restart":
        G, T = case["groups"], case["takes"]
        st["src"] = _i32([t // T for t in range(G * T)])
        st["dst"] = _i32([G + t for t in range(G * T)])
        pos = [-1] * len(lens)
        pos[G:G + G * T] = [case["prompt"]] * (G * T)
        st["pos"] = _i64(pos)
    else:
        used = sum(1 for r in ref if r)
        st["out"] = {"kv": torch.zeros(case["layers"], 2, used + 2, case["hk"], P, case["hd"], dtype=torch.float16, device=DEV),
                     "ref": torch.zeros(used + 2, dtype=torch.int32, device=DEV),
                     "table": torch.full_like(st["table"], -1), "length": torch.zeros_like(st["length"])}
    return st


def _prepare_write(case, seed):
    P, hk, hd = case["page"], case["hk"], case["hd"]
    per = _cdiv(case["start"] + case["rows"], P) + 1
    order = _perm(seed, 2, case["seqs"] * per + 3)
    g = _gen(seed, 1)
    slots = case["start"] + case["rows"]
    angle = torch.arange(slots, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return {"qkv": _rand(g, case["seqs"] * case["rows"], (case["hq"] + 2 * hk) * hd),
            "kv": _rand(g, 2, len(order), hk, P, hd),
            "table": _i32([[order.pop() for _ in range(per)] for _ in range(case["seqs"])]),
            "pos": _i64([case["start"] + i for _ in range(case["seqs"]) for i in range(case["rows"])]),
            "rope": torch.stack([angle.cos(), angle.sin()], -1).float().to(DEV) if case["rope"] else None}


def _prepare_attn(case, seed):
    P, hk, hd, T = case["page"], case["hk"], case["hd"], case["takes"]
    rows = case["groups"] * T
    lens = _lengths(case)
    width = max(_cdiv(max(lens), P), 1) + 1
    tabs, tails, n = [], [], 0
    for r in range(rows):
        pre = _prefix(case, r // T)
        full = pre // P
        if r % T == 0:
            first = list(range(n, n + full))
            n += full
        mine = max(0, _cdiv(lens[r], P) - full) if lens[r] else 1
        tabs.append(first + list(range(n, n + mine)))
        n += mine
        if pre % P and r % T:
            tails.append((tabs[r - r % T][full], tabs[r][full], pre % P))
    order = _perm(seed, 2, n)
    g = _gen(seed, 1)
    kv = _rand(g, 2, n, hk, P, hd)
    for a, b, k in tails:  # a fork copied the shared slots of a page that was not full
        kv[:, order[b], :, :k] = kv[:, order[a], :, :k]
    qkv = _rand(g, rows, (case["hq"] + 2 * hk) * hd)
    st = {"q": qkv[:, :case["hq"] * hd], "kv": kv, "table": _i32([[order[p] for p in t] + [-1] * (width - len(t)) for t in tabs]),
          "pos": _i64([k - 1 for k in lens])}
    if own:  # how rows share prefixes: set up once for all layers and frames of a song
        from estudiocanciones_amd import kernels
        st["plan"] = kernels.paged_attn_plan([(T, _prefix(case, i)) for i in range(case["groups"])], case["hq"], hk, hd,
                                             width * P, DEV)
    return st


def _prepare_a8(case, seed):
    g = _gen(seed, 1)
    M, N, K = case["rows"], case["n"], case["k"]
    x = _rand(g, M, K)
    x *= torch.rand(1, K, generator=g, device=DEV).mul_(3.0).exp_().half()  # channels of unequal size
    w = torch.randn(N, K, generator=g, device=DEV).mul_(30.5).round_().clamp_(-127, 127).to(torch.int8)
    s = (0.02 / 30.5 * (1 + 0.1 * torch.rand(N, generator=g, device=DEV))).half()
    st = {"x": x, "nw": (1 + 0.02 * torch.randn(K, generator=g, device=DEV)).half() if case["norm"] else None,
          "res": _rand(g, M, N) if case["res"] else None, "w": w, "s": s}
    if own:  # weights are laid out once, when a model is loaded
        from estudiocanciones_amd import kernels
        st["wp"] = kernels.pack_i8(w, interleave=case["silu"])
        st["sp"] = torch.stack([s[:N // 2], s[N // 2:]], 1).reshape(-1).contiguous() if case["silu"] else s
    return st


def prepare(case, seed):
    f = {"restart": _prepare_pages, "compact": _prepare_pages, "write": _prepare_write, "attn": _prepare_attn,
         "a8": _prepare_a8}[case["kind"]]
    return {"case": dict(case), **f(case, seed)}


# ---------------------------------------------------------------- plain forms
def _free(ref, table, length, seqs):
    rows = table[seqs]
    ref.index_add_(0, rows.clamp(min=0).reshape(-1), (rows < 0).int().sub_(1).reshape(-1))
    table[seqs] = -1
    length[seqs] = 0


def _take(ref, k):
    """The pages of the k-th free entries (0-based), lowest-numbered page first."""
    return torch.searchsorted((ref == 0).cumsum(0).int(), (k + 1).int()).int()


def _plain_restart(st):
    kv, ref, table, length = st["kv"], st["ref"], st["table"], st["length"]
    src, dst, pos, P = st["src"].long(), st["dst"].long(), st["pos"], st["kv"].shape[4]
    _free(ref, table, length, dst)
    # fork: whole pages shared, the slots of a last page that is not full copied into a page of the child's own
    n = length[src]
    full, tail = n // P, n % P
    need = tail > 0
    page = torch.where(need, _take(ref, need.cumsum(0) - need.int()), 0)
    col = torch.arange(table.shape[1], device=DEV)
    shared = col < full[:, None]
    rows = torch.where(shared, table[src], torch.where((col == full[:, None]) & need[:, None], page[:, None], -1)).int()
    old = table[src, full.clamp(max=table.shape[1] - 1)].clamp(min=0).long()
    to = torch.where(need, page, old).long()
    slot = torch.arange(P, device=DEV)[None, None, None, None, :, None]
    kv[:, :, to] = torch.where(slot < tail[None, None, :, None, None, None], kv[:, :, old], kv[:, :, to])
    ref.index_add_(0, rows.clamp(min=0).reshape(-1), (rows >= 0).int().reshape(-1))
    table[dst] = rows
    length[dst] = n
    # extend: every sequence holds slot pos afterwards
    more = torch.maximum(length, pos + 1)
    add = (col >= ((length + P - 1) // P)[:, None]) & (col < ((more + P - 1) // P)[:, None])
    page = _take(ref, (add.reshape(-1).cumsum(0) - 1).clamp(min=0)).reshape(add.shape)
    table.copy_(torch.where(add, page, table))
    ref.index_add_(0, torch.where(add, page, 0).reshape(-1), add.int().reshape(-1))
    length.copy_(more)
    return {"kv": kv.view(torch.int16), "ref": ref, "table": table, "length": length}


def _plain_compact(st):
    out, ref = st["out"], st["ref"]
    used = ref > 0
    n = out["ref"].shape[0]
    new = torch.where(used, used.cumsum(0) - 1, n).long()  # unused pages go to a place that is cut off
    src = torch.zeros(n + 1, dtype=torch.int64, device=DEV).scatter_(0, new, torch.arange(ref.shape[0], device=DEV))[:n]
    live = torch.arange(n, device=DEV) < used.sum()
    out["kv"].copy_(torch.where(live[None, None, :, None, None, None], st["kv"][:, :, src], out["kv"]))
    out["ref"].copy_(torch.where(live, ref[src], 0))
    out["table"].copy_(torch.where(st["table"] < 0, -1, new[st["table"].clamp(min=0).long()]))
    out["length"].copy_(st["length"])
    return {k: v.view(torch.int16) if k == "kv" else v for k, v in out.items()}


def _rope(x, rope, pos):
    """Rotates the interleaved pairs of x [M, H, HD] by the table's (cos, sin) at pos."""
    t = rope[pos][:, None]
    a, b = x.float().unflatten(-1, (-1, 2)).unbind(-1)
    return torch.stack([a * t[..., 0] - b * t[..., 1], b * t[..., 0] + a * t[..., 1]], -1).flatten(-2)


def _plain_write(st):
    case, pos, kv = st["case"], st["pos"], st["kv"]
    hq, hk, hd, P = case["hq"], case["hk"], case["hd"], case["page"]
    q, k, v = st["qkv"].unflatten(1, (-1, hd)).split([hq, hk, hk], 1)
    if st["rope"] is not None:
        q, k = _rope(q, st["rope"], pos).half(), _rope(k, st["rope"], pos).half()
    page = st["table"][torch.arange(case["seqs"], device=DEV).repeat_interleave(case["rows"]), pos // P].long()
    kv[0][page, :, pos % P] = k
    kv[1][page, :, pos % P] = v
    return {"kv": kv} if st["rope"] is None else {"kv": kv, "q": q.flatten(1)}


def _plain_attn(st):
    case, P = st["case"], st["case"]["page"]
    rows, hk, hd = st["q"].shape[0], case["hk"], case["hd"]
    slots = st["table"].shape[1] * P
    k, v = (st["kv"][i][st["table"].clamp(min=0).long()].transpose(1, 2).reshape(rows, hk, slots, hd).float() for i in (0, 1))
    s = st["q"].float().view(rows, hk, -1, hd) @ k.transpose(2, 3).contiguous() * (1.0 / math.sqrt(hd))
    s = s.masked_fill((torch.arange(slots, device=DEV) > st["pos"][:, None])[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    return (p @ v / p.sum(-1, keepdim=True).clamp(min=1e-30)).reshape(rows, -1).half()


def _plain_a8(st):
    case = st["case"]
    x = st["x"].float()
    if case["norm"]:
        x = x * (x.square().mean(1, keepdim=True) + EPS).rsqrt() * st["nw"].float()
    top = x.abs().amax(1, keepdim=True)
    codes = torch.where(top > 0, (x * 127 / top).round(), 0)
    y = (codes @ st["w"].float().t()) * (top / 127) * st["s"].float()
    if case["silu"]:
        a, b = y.chunk(2, 1)
        y = a / (1 + (-a).exp()) * b
    return (y if st["res"] is None else y + st["res"].float()).half()


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from estudiocanciones_amd import kernels as K
        if kind == "restart":
            K.page_free(st["ref"], st["table"], st["length"], st["dst"], case["page"], st["err"])
            K.page_fork(st["kv"], st["ref"], st["table"], st["length"], st["src"], st["dst"], st["err"])
            K.page_extend(st["ref"], st["table"], st["length"], st["pos"], case["page"], st["err"])
            return {"kv": st["kv"].view(torch.int16), "ref": st["ref"], "table": st["table"], "length": st["length"]}
        if kind == "compact":
            o = st["out"]
            K.page_compact(st["kv"], st["ref"], st["table"], st["length"], o["kv"], o["ref"], o["table"], o["length"], st["err"])
            return {k: v.view(torch.int16) if k == "kv" else v for k, v in o.items()}
        if kind == "write":
            q = K.paged_write(st["qkv"], st["kv"][0], st["kv"][1], st["table"], st["pos"], case["rows"], case["hq"],
                              case["hk"], rope=st["rope"])
            return {"kv": st["kv"]} if q is None else {"kv": st["kv"], "q": q}
        if kind == "attn":
            return K.paged_attn(st["q"], st["kv"][0], st["kv"][1], st["table"], st["pos"], st["plan"])
        codes, scale = K.quant_a8(st["x"], st["nw"], EPS)
        if case["silu"]:
            return K.gemm_a8_silu_packed(codes, scale, st["wp"], st["sp"], case["n"] // 2, case["k"])
        return K.gemm_a8_packed(codes, scale, st["wp"], st["sp"], case["n"], case["k"], st["res"])
    return {"restart": _plain_restart, "compact": _plain_compact, "write": _plain_write, "attn": _plain_attn,
            "a8": _plain_a8}[kind](st)


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind in ("restart", "compact"):
        return None  # page numbers, counts and copied bits: equal or wrong
    st = prepare(case, seed)
    if kind == "write":  # the rotation as a complex product, the slots of a sequence by flat numbers
        hq, hk, hd, P = case["hq"], case["hk"], case["hd"], case["page"]
        M = case["seqs"] * case["rows"]
        z = torch.view_as_complex(st["qkv"].double().reshape(M, hq + 2 * hk, hd // 2, 2))
        if st["rope"] is not None:
            turn = torch.view_as_complex(st["rope"].double())[st["pos"]]
            z = torch.cat([z[:, :hq + hk] * turn[:, None], z[:, hq + hk:]], 1)
        y = torch.view_as_real(z).reshape(M, hq + 2 * hk, hd)
        kv = st["kv"].double()
        for s in range(case["seqs"]):
            at = slice(s * case["rows"], (s + 1) * case["rows"])
            slot = st["pos"][at]
            flat = st["table"][s].long()[slot // P] * P + slot % P
            for i in (0, 1):
                pool = kv[i].transpose(1, 2).reshape(-1, hk, hd)
                pool[flat] = y[at, hq + i * hk:hq + (i + 1) * hk]
                kv[i] = pool.reshape(-1, P, hk, hd).transpose(1, 2)
        return {"kv": kv} if st["rope"] is None else {"kv": kv, "q": y[:, :hq].reshape(M, -1)}
    if kind == "attn":  # row by row over the slots that it attends
        hq, hk, hd, P = case["hq"], case["hk"], case["hd"], case["page"]
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
        for r, n in enumerate(_lengths(case)):
            if not n:
                continue
            pages = st["table"][r, :_cdiv(n, P)].long()
            k, v = (st["kv"][i][pages].double().permute(1, 0, 2, 3).reshape(hk, -1, hd)[:, :n] for i in (0, 1))
            q = st["q"][r].double().reshape(hk, hq // hk, hd)
            out[r] = (torch.softmax(q @ k.mT.contiguous() / math.sqrt(hd), -1) @ v).reshape(-1)
        return out
    M, N = case["rows"], case["n"]
    y = torch.empty(M, N // 2 if case["silu"] else N, dtype=torch.float64, device=DEV)
    w = st["w"].double() * st["s"].double()[:, None]
    for m in range(0, M, 512):
        x = st["x"][m:m + 512].double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(1, keepdim=True) / case["k"] + EPS) * st["nw"].double()
        top = x.abs().amax(1, keepdim=True).clamp(min=1e-300)
        z = (torch.round(x * 127 / top) * (top / 127)) @ w.t()
        if case["silu"]:
            z = torch.nn.functional.silu(z[:, :N // 2]) * z[:, N // 2:]
        y[m:m + 512] = z if st["res"] is None else z + st["res"][m:m + 512].double()
    return y


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "restart":
        n, P = case["groups"] * case["takes"], case["page"]
        slot = case["layers"] * 2 * case["hk"] * case["hd"] * 2
        pages = _cdiv(case["prompt"] + 1, P)
        return {"bytes": (case["groups"] + n) * (case["prompt"] % P) * slot + n * pages * 12, "flops": 0}
    if kind == "compact":
        pages = case["shared"] + sum(_cdiv(n, case["page"]) for n in _compact_lengths(case))
        return {"bytes": 2 * pages * case["layers"] * 2 * case["hk"] * case["page"] * case["hd"] * 2 + case["pages"] * 4, "flops": 0}
    if kind == "write":
        M, wide = case["seqs"] * case["rows"], (case["hq"] + 2 * case["hk"]) * case["hd"]
        return {"bytes": M * (wide * 4 + 8) + (case["rows"] * case["hd"] * 4 if case["rope"] else 0),
                "flops": 3 * M * (case["hq"] + case["hk"]) * case["hd"] if case["rope"] else 0}
    if kind == "attn":
        lens = _lengths(case)
        T = case["takes"]
        slots = 0
        for g in range(case["groups"]):
            mine = [n for n in lens[g * T:(g + 1) * T] if n]
            slots += sum(n - _prefix(case, g) for n in mine) + (_prefix(case, g) if mine else 0)
        return {"bytes": slots * case["hk"] * case["hd"] * 4 + len(lens) * case["hq"] * case["hd"] * 4,
                "flops": 4 * sum(lens) * case["hq"] * case["hd"]}
    M, N, K = case["rows"], case["n"], case["k"]
    return {"bytes": M * K * 2 + N * K + 2 * N + (M * N if case["silu"] else 2 * M * N) + (2 * M * N if case["res"] else 0)
            + (2 * K if case["norm"] else 0), "flops": 2 * M * N * K}
