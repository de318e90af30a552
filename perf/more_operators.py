"""Products with 4-bit weights and the processing of logits before the sampler, as cases that can be timed and checked.

Two operators of a decoding step: ``mm_q4``, the product of fp16 rows with weights of 4 bits and a scale for each
group of 32, 64 or 128 of them (with the RMS norm before it, a residual or SiLU(a) * b behind it), from one row to a
prompt's; and ``process_logits``, which takes the logits of a vocabulary to those a sampler draws from: guidance,
penalties for the tokens of a history, biases and masks of allowed tokens.

``own`` chooses between the framework's calls and their plain forms: elementary torch operations in 32 bits,
rounded once.  Sizes are those of the model's configurations (the 3B backbone's 3072 channels and 8192 of its MLP, the
depth decoder's 1024, the 8197 tokens of a codebook) and generic ones.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the head of the first codebook for a single take without guidance (latency counts)
        {"name": "q4_1row_head", "kind": "q4", "rows": 1, "n": 8197, "k": 3072, "group": 128, "zeros": False,
         "norm": True, "silu": False, "res": False},
        # a frame of 4 takes with guidance: norm and query, key and value projections of a backbone layer
        {"name": "q4_8rows_qkv", "kind": "q4", "rows": 8, "n": 5120, "k": 3072, "group": 128, "zeros": False,
         "norm": True, "silu": False, "res": False},
        # the same frame: norm, gate and up projections, SiLU
        {"name": "q4_8rows_silu", "kind": "q4", "rows": 8, "n": 16384, "k": 3072, "group": 128, "zeros": False,
         "norm": True, "silu": True, "res": False},
        # the same frame: down projection and residual
        {"name": "q4_8rows_res", "kind": "q4", "rows": 8, "n": 3072, "k": 8192, "group": 128, "zeros": False,
         "norm": False, "silu": False, "res": True},
        # the narrow depth decoder's down projection for 8 takes with guidance: few outputs over a long sum, the finest
        # groups, with zero points
        {"name": "q4_16rows_narrow", "kind": "q4", "rows": 16, "n": 1024, "k": 8192, "group": 32, "zeros": True,
         "norm": False, "silu": False, "res": True},
        # 24 takes with guidance: the output projection of attention
        {"name": "q4_48rows_res", "kind": "q4", "rows": 48, "n": 3072, "k": 3072, "group": 64, "zeros": False,
         "norm": False, "silu": False, "res": True},
        # a short prompt's down projection with its residual, ragged rows, zero points
        {"name": "q4_187rows_res", "kind": "q4", "rows": 187, "n": 3072, "k": 8192, "group": 128, "zeros": True,
         "norm": False, "silu": False, "res": True},
        # the gate and up projections of a prompt of 2048 rows (the largest product)
        {"name": "q4_2048rows_silu", "kind": "q4", "rows": 2048, "n": 16384, "k": 3072, "group": 128, "zeros": False,
         "norm": False, "silu": True, "res": False},
        # one take, one codebook, a penalty for the tokens of the last 64 frames (latency counts)
        {"name": "logits_1take", "kind": "logits", "takes": 1, "vocab": 8197, "guided": False, "history": 750,
         "window": 64, "frames": True, "ragged": False, "penalties": 1, "bias": 0, "masks": 0},
        # 4 takes with guidance, late in a song of 4 minutes: penalties over all of it, a bias, end tokens not allowed
        {"name": "logits_4takes_song", "kind": "logits", "takes": 4, "vocab": 8197, "guided": True, "history": 3000,
         "window": 0, "frames": True, "ragged": False, "penalties": 3, "bias": 1, "masks": 1},
        # a batch of 128 takes with guidance
        {"name": "logits_128takes", "kind": "logits", "takes": 128, "vocab": 8197, "guided": True, "history": 750,
         "window": 0, "frames": True, "ragged": False, "penalties": 3, "bias": 1, "masks": 1},
        # a text vocabulary: 32 rows of ragged histories, each row with its own bias and its grammar state's mask
        {"name": "logits_32rows_text", "kind": "logits", "takes": 32, "vocab": 100003, "guided": False, "history": 4096,
         "window": 0, "frames": False, "ragged": True, "penalties": 3, "bias": 2, "masks": 20},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.65:
        n, k = rng.choice([(5120, 3072), (3072, 3072), (3072, 8192), (8197, 3072), (8197, 1024), (1024, 8192), (1536, 1024),
                           (1001, 192), (4608, 1536), (250, 64), (16384, 1024)])
        silu = rng.random() < 0.3
        return {"kind": "q4", "rows": _log_int(rng, 1, 2500), "n": 2 * (n // 2) if silu else n, "k": k,
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.4, "norm": rng.random() < 0.5, "silu": silu,
                "res": not silu and rng.random() < 0.5}
    vocab = rng.choice([8197, 8197, _log_int(rng, 40, 120000)])
    frames = rng.random() < 0.5
    return {"kind": "logits", "takes": _log_int(rng, 1, 200 if vocab < 10000 else 32), "vocab": vocab,
            "guided": rng.random() < 0.5, "history": _log_int(rng, 1, 6000), "window": rng.choice([0, 0, _log_int(rng, 1, 500)]),
            "frames": frames, "ragged": not frames and rng.random() < 0.7, "penalties": rng.randint(0, 3),
            "bias": rng.randint(0, 2), "masks": rng.choice([0, 1, rng.randint(2, 30)])}


# ---------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + salt)


def _rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16).mul_(scale)


def _groups(case):
    return -(-case["k"] // case["group"])


def _prepare_q4(case, seed):
    g = _gen(seed, 1)
    M, N, K = case["rows"], case["n"], case["k"]
    x = _rand(g, M, K)
    x *= torch.rand(1, K, generator=g, device=DEV).mul_(2.0).exp_().half()  # channels of unequal size
    u = torch.randn(N, K, generator=g, device=DEV).mul_(2.6).round_().add_(8).clamp_(0, 15).to(torch.uint8)
    q = u[:, 0::2] | (u[:, 1::2] << 4)  # element 2 i in the low half of byte i
    s = (0.02 / 2.6 * (1 + 0.3 * torch.rand(N, _groups(case), generator=g, device=DEV))).half()
    z = torch.randint(5, 12, (N, _groups(case)), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
    st = {"x": x, "nw": (1 + 0.02 * torch.randn(K, generator=g, device=DEV)).half() if case["norm"] else None,
          "res": _rand(g, M, N) if case["res"] else None, "q": q, "s": s, "z": z}
    if own:  # weights are laid out once, when a model is loaded
        from estudiocanciones_amd import kernels
        st["w"] = kernels.pack_q4(q, s, z, interleave=case["silu"])
    return st


def _lengths(case):
    """Tokens that each row's history holds."""
    return [int(case["history"] * math.fmod(0.618034 * (r + 1), 1.0)) if case["ragged"] else case["history"]
            for r in range(case["takes"])]


def _prepare_logits(case, seed):
    g = _gen(seed, 1)
    N, V, T = case["takes"], case["vocab"], case["history"]
    rows = 2 * N if case["guided"] else N
    wide = -(-V // 64) * 64  # rows start aligned, as the engine lays logits out
    logits = _rand(g, rows, wide, scale=4.0)[:, :V]
    often = (V * torch.rand(N, T, 8, generator=g, device=DEV) ** 3).long().clamp_(max=V - 1)  # some tokens come often
    if case["frames"]:  # the song's frames [T, N, codebooks], of which one codebook is the history
        hist = often.transpose(0, 1).contiguous()[:, :, 3].t()
    else:
        hist = often[:, :, 3].contiguous()
    st = {"logits": logits, "hist": hist, "length": torch.tensor(_lengths(case), dtype=torch.int64, device=DEV),
          "cfg": 1.5 if case["guided"] else None, "repetition": None, "presence": None, "frequency": None,
          "bias": None, "allowed": None, "state": None}
    row = torch.rand(3, N, generator=g, device=DEV)
    if case["penalties"] >= 1:
        st["repetition"] = 1 + 0.3 * row[0]
    if case["penalties"] >= 2:
        st["presence"] = 0.5 * row[1]
    if case["penalties"] >= 3:
        st["frequency"] = 0.1 * row[2]
    if case["bias"]:
        some = torch.rand(N if case["bias"] == 2 else 1, V, generator=g, device=DEV)
        st["bias"] = torch.where(some < 0.05, 40 * some - 1, 0.0)
        if case["bias"] == 1:
            st["bias"] = st["bias"][0]
    if case["masks"]:  # one mask for all rows (end tokens), or a grammar's states, of which each row is in one
        A = case["masks"]
        keep = torch.rand(A, -(-V // 32) * 32, generator=g, device=DEV) < (0.2 if A > 1 else 0.999)
        if A > 2:
            keep[2] = False  # a state that nothing leaves
        word = keep.view(A, -1, 32).long() << torch.arange(32, device=DEV)
        st["allowed"] = word.sum(2).to(torch.int32)  # (the low 32 bits)
        if A > 1:
            st["state"] = torch.randint(-1, A, (N,), generator=g, device=DEV, dtype=torch.int32)  # -1: no mask
        else:
            logits[:, V - V // 50:] = math.inf  # what may not be drawn holds anything
            st["allowed"][:, (V - V // 50) // 32:] = 0
    return st


def prepare(case, seed):
    return {"case": dict(case), **(_prepare_q4 if case["kind"] == "q4" else _prepare_logits)(case, seed)}


# ---------------------------------------------------------------- plain forms
def _plain_q4(st):
    case, G = st["case"], st["case"]["group"]
    x = st["x"].float()
    if case["norm"]:
        x = x * (x.square().mean(1, keepdim=True) + EPS).rsqrt() * st["nw"].float()
    u = torch.stack([st["q"] & 15, st["q"] >> 4], -1).flatten(1).float()
    z = 8.0 if st["z"] is None else st["z"].float().repeat_interleave(G, 1)[:, :case["k"]]
    w = (u - z) * st["s"].float().repeat_interleave(G, 1)[:, :case["k"]]
    y = x @ w.t()
    if case["silu"]:
        a, b = y.chunk(2, 1)
        y = a / (1 + (-a).exp()) * b
    return (y if st["res"] is None else y + st["res"].float()).half()


def _plain_logits(st):
    case = st["case"]
    N, V = case["takes"], case["vocab"]
    l = st["logits"].float()
    if st["cfg"] is not None:
        l = l[N:] + (l[:N] - l[N:]) * st["cfg"]
    if case["penalties"]:
        T = st["hist"].shape[1]
        at, n = torch.arange(T, device=DEV), st["length"][:, None]
        live = (at < n) & (at >= n - case["window"]) if case["window"] else at < n
        c = torch.zeros(N, V, device=DEV).scatter_add_(1, st["hist"], live.float())
        rep = st["repetition"][:, None]
        l = torch.where(c > 0, torch.where(l > 0, l / rep, l * rep), l)
        if st["presence"] is not None:
            l = torch.where(c > 0, l - st["presence"][:, None], l)
        if st["frequency"] is not None:
            l = l - st["frequency"][:, None] * c
    if st["bias"] is not None:
        l = l + st["bias"]
    if st["allowed"] is not None:
        bit = (st["allowed"][:, :, None] >> torch.arange(32, device=DEV)) & 1
        keep = bit.flatten(1)[:, :V] > 0
        if st["state"] is not None:
            s = st["state"].long()
            keep = keep[s.clamp(min=0)] | (s < 0)[:, None]
        l = torch.where(keep, l, -math.inf)
    return l.half()


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    if not own:
        return _plain_q4(st) if case["kind"] == "q4" else _plain_logits(st)
    from estudiocanciones_amd import kernels as K
    if case["kind"] == "q4":
        if case["silu"]:
            return K.mm_q4_silu(st["x"], st["w"], nw=st["nw"], eps=EPS)
        return K.mm_q4(st["x"], st["w"], res=st["res"], nw=st["nw"], eps=EPS)
    return K.process_logits(st["logits"], st["hist"], st["length"], window=case["window"], repetition=st["repetition"],
                            presence=st["presence"], frequency=st["frequency"], bias=st["bias"], allowed=st["allowed"],
                            state=st["state"], cfg=st["cfg"])


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "q4":  # group by group: s * (sum of x u - z * sum of x)
        M, N, K, G = case["rows"], case["n"], case["k"], case["group"]
        y = torch.zeros(M, N, dtype=torch.float64, device=DEV)
        x = st["x"].double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(1, keepdim=True) / K + EPS) * st["nw"].double()
        for g in range(_groups(case)):
            part = x[:, g * G:(g + 1) * G].contiguous()
            code = st["q"][:, g * G // 2:(g + 1) * G // 2]
            u = torch.empty(N, part.shape[1], dtype=torch.float64, device=DEV)
            u[:, 0::2], u[:, 1::2] = code % 16, code // 16
            z = torch.full((N,), 8.0, dtype=torch.float64, device=DEV) if st["z"] is None else st["z"][:, g].double()
            y += (part @ u.t().contiguous() - part.sum(1, keepdim=True) * z) * st["s"][:, g].double()
        if case["silu"]:
            y = torch.nn.functional.silu(y[:, :N // 2]) * y[:, N // 2:]
        return y if st["res"] is None else y + st["res"].double()
    N, V, W = case["takes"], case["vocab"], case["window"]
    out = torch.empty(N, V, dtype=torch.float64, device=DEV)
    lens = _lengths(case)
    for r in range(N):  # row by row, the history's tokens counted one row at a time
        l = st["logits"][r].double()
        if st["cfg"] is not None:
            w = st["logits"][N + r].double()
            l = st["cfg"] * l + (1 - st["cfg"]) * w
            same = torch.isinf(st["logits"][r]) | torch.isinf(st["logits"][N + r])
            l[same] = math.nan  # (masked below)
        seen = st["hist"][r, max(0, lens[r] - W) if W else 0:lens[r]]
        c = torch.bincount(seen, minlength=V).double()
        t = c > 0
        if st["repetition"] is not None:
            f = st["repetition"][r].double()
            l[t] = torch.minimum(l[t] * f, l[t] / f)  # (f >= 1)
        if st["presence"] is not None:
            l[t] -= st["presence"][r].double()
        if st["frequency"] is not None:
            l -= c * st["frequency"][r].double()
        if st["bias"] is not None:
            l += (st["bias"][r] if case["bias"] == 2 else st["bias"]).double()
        a = None if st["allowed"] is None else 0 if st["state"] is None else int(st["state"][r])
        if a is not None and a >= 0:
            byte = st["allowed"][a].contiguous().view(torch.uint8)
            bits = torch.stack([byte >> i & 1 for i in range(8)], -1).reshape(-1)[:V]
            l[bits == 0] = -math.inf
        out[r] = l
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "q4":
        M, N, K, ng = case["rows"], case["n"], case["k"], _groups(case)
        return {"bytes": M * K * 2 + N * K // 2 + N * ng * 2 + (N * ng // 2 if case["zeros"] else 0)
                + (M * N if case["silu"] else 2 * M * N) + (2 * M * N if case["res"] else 0) + (2 * K if case["norm"] else 0),
                "flops": 2 * M * N * K}
    N, V, W = case["takes"], case["vocab"], case["window"]
    rows = 2 * N if case["guided"] else N
    seen = sum(min(n, W) if W else n for n in _lengths(case)) if case["penalties"] else 0
    masks = min(case["masks"], N)
    return {"bytes": 2 * (rows + N) * V + 8 * seen + (4 * V * (N if case["bias"] == 2 else 1) if case["bias"] else 0)
            + masks * (-(-V // 32) * 4), "flops": 6 * N * V}
