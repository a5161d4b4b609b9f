"""Timed cases of the operators behind speculation with trees of drafts.

  rope    rotary positions applied to heads at given positions (cache.Rotate)
  tree    attention of a tree of drafted tokens over the paged cache
          (KVCache.AttendTree)
  accept  acceptance of a tree of drafts against the target's logits
          (tree_accept_async)
  keep    a batch's trees appended, their accepted paths kept (KVCache.KeepPath)
          and the caches read back, layer by layer

Each has a plain form in elementary torch operations and, with `own` set, the
framework's call.  Lengths and tree shapes are part of the case (drawn from its
"mix"); values come from prepare()'s seed.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decode step of 16 users: the q and k heads of their new tokens, launch latency only.
        dict(name="rope_decode", op="rope", rows=16, heads=40, D=128, rd=128, layout="halves", dtype="bf16",
             pos=8192, scaling="none"),
        # Prompts of 8192 tokens, every q and k head of a layer: a stream through memory.
        dict(name="rope_prompt", op="rope", rows=8192, heads=40, D=128, rd=128, layout="pairs", dtype="bf16",
             pos=8192, scaling="linear"),
        # An odd chunk far into a context stretched by parts, a part of an 80-wide head rotated, f32 rows.
        dict(name="rope_far", op="rope", rows=3001, heads=32, D=80, rd=32, layout="halves", dtype="f32",
             pos=1000000, scaling="yarn"),
        # One user, a small tree on a short chat, the API's default f32 rows: launches and host time.
        dict(name="tree_one", op="tree", B=1, H=32, KVH=8, D=128, P=16, T_lo=200, T_hi=200, n_lo=7, n_hi=7,
             mix=1, dtype="f32", part=1.0),
        # The benchmark's 16 users at 8k of context, 16 drafts each: a stream over the cache.
        dict(name="tree_8k", op="tree", B=16, H=32, KVH=8, D=128, P=16, T_lo=8192, T_hi=8192, n_lo=16, n_hi=16,
             mix=2, dtype="bf16", part=1.0),
        # Wide trees for users at very different points, 8 heads a kv head: the most arithmetic.
        dict(name="tree_wide", op="tree", B=24, H=64, KVH=8, D=128, P=16, T_lo=1000, T_hi=12000, n_lo=40, n_hi=64,
             mix=3, dtype="bf16", part=1.0),
        # Odd sizes: 80-wide heads with a kv head each, trees of 1 to 31 nodes, the last levels as queries.
        dict(name="tree_odd", op="tree", B=5, H=16, KVH=16, D=80, P=32, T_lo=300, T_hi=3001, n_lo=1, n_hi=31,
             mix=4, dtype="bf16", part=0.5),
        # One user, drafts picked without probabilities: what a single step waits for.
        dict(name="accept_one", op="accept", B=1, V=32000, n_lo=8, n_hi=8, mix=5, T=0.8, draft=False),
        # A full serving batch of 32-node trees with the draft's own distribution.
        dict(name="accept_batch", op="accept", B=64, V=32000, n_lo=32, n_hi=32, mix=6, T=0.8, draft=True),
        # Rows that are not 16-byte aligned, uneven and larger trees.
        dict(name="accept_odd", op="accept", B=12, V=50257, n_lo=9, n_hi=61, mix=7, T=1.0, draft=True),
        # One layer of one user: what keeping a path costs at the least.
        dict(name="keep_one", op="keep", B=1, L=1, KVH=8, D=128, P=16, T_lo=200, T_hi=200, n_lo=8, n_hi=8, mix=8,
             dtype="bf16"),
        # Every layer of a batch at once.
        dict(name="keep_batch", op="keep", B=16, L=16, KVH=8, D=128, P=16, T_lo=100, T_hi=300, n_lo=24, n_hi=48,
             mix=9, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 8e14)


def draw(rng):
    while True:
        c = _draw(rng)
        if _cost(c) > max(_cost(k) for k in listed() if k["op"] == c["op"]):
            continue
        if c["op"] == "tree" and sum(map(sum, _lens(c))) * c["KVH"] > 2_000_000:
            continue
        if c["op"] == "accept" and sum(_lens(c)[1]) * c["V"] > 64 * 32 * 32000:
            continue
        return c


def _draw(rng):
    op = rng.choice(["rope", "rope", "tree", "tree", "tree", "tree", "accept", "accept", "accept", "keep"])
    if op == "rope":
        D = rng.choice([16, 64, 80, 96, 128, 192, 256])
        rd = rng.choice([D, D, D // 2])
        return dict(op=op, rows=_log(rng, 1, 8192), heads=rng.randint(1, 72), D=D, rd=rd,
                    layout=rng.choice(["pairs", "halves"]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                    pos=_log(rng, 64, 1000000), scaling=rng.choice(["none", "linear", "ntk", "yarn"]))
    c = dict(op=op, mix=rng.randint(100, 10 ** 6))
    if op == "accept":
        c["B"], c["V"], n = _log(rng, 1, 64), _log(rng, 4000, 128000), _log(rng, 2, 128)
        c["n_hi"], c["n_lo"] = n, rng.choice([n, max(1, n // 3)])
        c["T"], c["draft"] = round(rng.uniform(0.6, 1.1), 2), rng.choice([True, True, False])
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "f32"])
    if op == "keep":
        c["B"], c["L"], T, n = _log(rng, 1, 16), _log(rng, 1, 16), _log(rng, 1, 300), _log(rng, 1, 64)
        c["KVH"], c["D"], c["P"] = rng.choice([1, 2, 8, 16]), rng.choice([64, 80, 128]), rng.choice([16, 32, 64])
    else:
        c["B"], T, n = _log(rng, 1, 64), _log(rng, 16, 32768), _log(rng, 1, 128)
        c["H"], c["KVH"] = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (16, 16), (8, 2), (28, 4), (16, 1)])
        c["D"], c["P"] = rng.choice([128, 128, 128, 64, 80, 256]), rng.choice([16, 16, 32, 64])
        c["part"] = rng.choice([1.0, 1.0, 0.5])
    c["T_hi"], c["T_lo"] = T, rng.choice([T, max(1, T // 2), max(1, T // 8)])
    c["n_hi"], c["n_lo"] = n, rng.choice([n, max(1, n // 3)])
    return c


# ---- shapes: lengths, trees, paths -----------------------------------------------------

def _lens(case):
    """(context tokens, tree nodes) of every sequence."""
    r = random.Random(case["mix"])
    lo, hi = case.get("T_lo", 0), case.get("T_hi", 0)
    wide = lo > 0 and hi > 10 * lo
    T = [_log(r, lo, hi) if wide else r.randint(lo, hi) for _ in range(case["B"])]
    return T, [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["B"])]


def _trees(case):
    """The nodes' parents, a list for each sequence (node 0 is the root)."""
    r = random.Random(case["mix"] + 1)
    return [[-1] + [r.randint((j - 1) // 3, max((j - 1) // 3, 2 * (j - 1) // 3)) for j in range(1, n)]
            for n in _lens(case)[1]]


def _queries(case):
    """Nodes of every sequence that are queries: the last ones."""
    return [max(1, int(n * case["part"])) for n in _lens(case)[1]]


def _up(parents, j):
    """Node j and its ancestors, root first."""
    out = []
    while j >= 0:
        out.append(j)
        j = parents[j]
    return out[::-1]


def _paths(case):
    """An accepted path for each sequence: to one of its last nodes."""
    r = random.Random(case["mix"] + 2)
    return [_up(p, r.randint(len(p) // 2, len(p) - 1)) for p in _trees(case)]


def _rounds(case):
    """The contexts' appends, a page a sequence in a fresh random order each time, as a serving batch that
    grows together leaves its pages: [(sequence, first token, tokens)] lists."""
    T, _ = _lens(case)
    r = random.Random(case["mix"] + 3)
    out, P = [], case["P"]
    for at in range(0, max(T), P):
        order = [i for i in range(len(T)) if at < T[i]]
        r.shuffle(order)
        out.append([(i, at, min(P, T[i] - at)) for i in order])
    return out


def _freqs(case):
    """inv_freq (f32) and the factor of the rotated dims, in numpy: base 10000, contexts stretched 8 times."""
    rd, base, f = case["rd"], 10000.0, 8.0
    i = np.arange(rd // 2, dtype=np.float64)
    if case["scaling"] == "ntk":
        base *= f ** (rd / max(rd - 2, 1))
    inv = base ** (-2.0 * i / rd)
    scale = 1.0
    if case["scaling"] == "linear":
        inv = inv / f
    if case["scaling"] == "yarn":
        # dims that turn more than 32 times in the original 4096 positions stay, fewer than once are divided
        def dim(turns):
            return rd * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), rd - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        inv = inv / f * ramp + inv * (1 - ramp)
        scale = 0.1 * math.log(f) + 1.0
    return inv.astype(np.float32), float(np.float32(scale))


# ---- inputs ------------------------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, dtype=dtype, generator=g)

    op = case["op"]
    if op == "rope":
        dt = DTYPES[case["dtype"]]
        return dict(x=randn(case["rows"], case["heads"], case["D"], dtype=dt),
                    pos=torch.randint(0, case["pos"], (case["rows"],), device=DEV, generator=g, dtype=torch.int32))
    T, n = _lens(case)
    trees = _trees(case)
    s = dict(parents=torch.tensor(sum(trees, []), dtype=torch.int32, device=DEV))
    if op == "accept":
        rows, V = sum(n), case["V"]
        base = randn(rows, V) * 3.0
        t = base + randn(rows, V) * 0.7
        # children without replacement from their parent's draft distribution: the best of noisy logits
        wide = max(max((p.count(j) for j in range(len(p))), default=0) for p in trees)
        tok = torch.randint(0, V, (rows,), device=DEV, generator=g, dtype=torch.int32)
        if wide:
            noise = -torch.log(-torch.log(torch.rand(rows, V, device=DEV, generator=g).clamp_(1e-9, 1 - 1e-7)))
            best = torch.topk(base / case["T"] + noise, wide, dim=1).indices.to(torch.int32)
            kids, at, up, rank = [], 0, [], []
            for p in trees:
                seen = {}
                for j in range(1, len(p)):
                    kids.append(at + j)
                    up.append(at + p[j])
                    rank.append(seen.get(p[j], 0))
                    seen[p[j]] = rank[-1] + 1
                at += len(p)
            tok[torch.tensor(kids, device=DEV)] = best[torch.tensor(up, device=DEV), torch.tensor(rank, device=DEV)]
        s.update(t=t, d=base if case["draft"] else None, tok=tok, u=torch.rand(rows, device=DEV, generator=g))
        return s
    KVH, D, dt, bf = case["KVH"], case["D"], DTYPES[case["dtype"]], torch.bfloat16
    if op == "tree":
        live = sum(T) + sum(n)  # a sequence's context, then its nodes
        s["K"], s["V"] = randn(live, KVH, D, dtype=bf), randn(live, KVH, D, dtype=bf)
        s["q"] = (randn(sum(_queries(case)), case["H"], D) * 2.0).to(dt)
        return s
    L = case["L"]
    s["K"], s["V"] = randn(L, sum(T), KVH, D, dtype=bf), randn(L, sum(T), KVH, D, dtype=bf)
    s["k"], s["v"] = randn(L, sum(n), KVH, D, dtype=dt), randn(L, sum(n), KVH, D, dtype=dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], op = case, case["op"]
    if op == "rope":
        inv, s["scale"] = _freqs(case)
        s["inv"] = torch.from_numpy(inv).to(DEV)
    if op == "tree":
        s["nq"] = _queries(case)
    if op == "keep":
        s["paths"] = _paths(case)
    if op != "rope":
        s["T"], s["n"] = _lens(case)
    return _prepare_own(case, s) if own else s


def _prepare_own(case, s):
    import relux_amd as ra
    op, B = case["op"], case.get("B", 1)
    s["ra"], s["seqs"] = ra, list(range(B))
    if op in ("rope", "accept"):
        s["cache"] = ra.KVCache(num_layers=1, max_len=16, num_kv_heads=1, head_dim=64)  # any cache's stream
        if op == "rope":
            s["out"] = torch.empty_like(s["x"])
        else:
            s["sampler"] = ra.Sampler(temperature=case["T"])
            s["path"] = torch.empty(B, max(s["n"]), dtype=torch.int32, device=DEV)
            s["n_acc"] = torch.empty(B, dtype=torch.int32, device=DEV)
            s["next"] = torch.empty(B, dtype=torch.int32, device=DEV)
        return s
    T, n, P, L = s["T"], s["n"], case["P"], case.get("L", 1)
    c = ra.KVCache(num_layers=L, max_len=max(a + b for a, b in zip(T, n)), num_kv_heads=case["KVH"],
                   head_dim=case["D"], page_tokens=P, max_seqs=B,
                   pool_pages=sum(-(-(a + b) // P) for a, b in zip(T, n)) + 8)
    first = np.cumsum([0] + [a + (b if op == "tree" else 0) for a, b in zip(T, n)])
    K, V = (s["K"][None], s["V"][None]) if op == "tree" else (s["K"], s["V"])
    for todo in _rounds(case):
        rows = torch.from_numpy(np.concatenate([np.arange(first[i] + at, first[i] + at + m) for i, at, m in todo]))
        rows = rows.to(DEV)
        for layer in range(L):
            c.Append(layer, K[layer][rows], V[layer][rows], seq_ids=[t[0] for t in todo], n_tok=[t[2] for t in todo],
                     layout="SHD")
    if op == "tree":
        rows = torch.from_numpy(np.concatenate([np.arange(f + a, f + a + b) for f, a, b in zip(first, T, n)])).to(DEV)
        c.Append(0, s["K"][rows], s["V"][rows], seq_ids=s["seqs"], n_tok=n, layout="SHD")
        s["out"] = torch.empty_like(s["q"])
    else:
        live = sum(T) + sum(len(p) for p in s["paths"])
        s["ko"] = [torch.empty(live * case["KVH"] * case["D"], dtype=torch.bfloat16, device=DEV) for _ in range(L)]
        s["vo"] = [torch.empty_like(k) for k in s["ko"]]
        s["kept"] = [len(p) for p in s["paths"]]
    s["cache"] = c
    s["K"] = s["V"] = None
    return s


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else PLAIN[s["case"]["op"]](s)


def _run_own(s):
    case, c = s["case"], s["cache"]
    op = case["op"]
    if op == "rope":
        return c.Rotate(s["x"], s["pos"], s["inv"], layout=case["layout"], scale=s["scale"], out=s["out"])
    if op == "tree":
        return c.AttendTree(0, s["q"], case["H"], s["parents"], seq_ids=s["seqs"], n_nodes=s["n"], n_q=s["nq"],
                            out=s["out"])
    if op == "accept":
        return s["ra"].tree_accept_async(c, s["t"], s["tok"], s["parents"], s["n"], s["u"], s["sampler"],
                                         draft_logits=s["d"], path=s["path"], n_acc=s["n_acc"], next_tok=s["next"])
    for layer in range(case["L"]):
        c.Append(layer, s["k"][layer], s["v"][layer], seq_ids=s["seqs"], n_tok=s["n"], layout="SHD")
    c.KeepPath(s["seqs"], s["n"], s["paths"])
    for layer in range(case["L"]):
        c.Gather(layer, s["seqs"], s["ko"][layer], s["vo"][layer])
    c.Rollback(s["seqs"], s["kept"])  # back to the contexts, for the next pass
    return [s["ko"], s["vo"]]


def _plain_rope(s):
    x, rd = s["x"], s["case"]["rd"]
    a = s["pos"].double()[:, None] * s["inv"].double()[None, :]  # far positions need the 64 bits
    c, sn = (torch.cos(a) * s["scale"]).float()[:, None], (torch.sin(a) * s["scale"]).float()[:, None]
    r = x[..., :rd].float()
    if s["case"]["layout"] == "pairs":
        x0, x1 = r[..., 0::2], r[..., 1::2]
        y = torch.stack([x0 * c - x1 * sn, x0 * sn + x1 * c], dim=-1).flatten(-2)
    else:
        x0, x1 = r[..., :rd // 2], r[..., rd // 2:]
        y = torch.cat([x0 * c - x1 * sn, x0 * sn + x1 * c], dim=-1)
    return torch.cat([y.to(x.dtype), x[..., rd:]], dim=-1)


def _plain_tree(s):
    case = s["case"]
    H, KVH, D = case["H"], case["KVH"], case["D"]
    G, out, at, node, row = H // KVH, [], 0, 0, 0
    for T, n, m in zip(s["T"], s["n"], s["nq"]):
        # a node sees itself and its ancestors: the closure of the parent relation, by squaring
        parent = s["parents"][node:node + n]
        ids = torch.arange(n, device=DEV, dtype=torch.int32)
        see = ((parent[:, None] == ids[None, :]) | (ids[:, None] == ids[None, :])).float()
        step = 1
        while step < n:
            see = (torch.matmul(see, see) > 0).float()
            step *= 2
        mask = torch.cat([torch.ones(m, T, device=DEV), see[n - m:]], dim=1) > 0
        q = s["q"][row:row + m].float().view(m, KVH, G, D).permute(1, 0, 2, 3).reshape(KVH, m * G, D)
        k = s["K"][at:at + T + n].float().permute(1, 2, 0).contiguous()
        v = s["V"][at:at + T + n].float().permute(1, 0, 2).contiguous()
        w = torch.matmul(q, k) * (1.0 / math.sqrt(D))
        w = w.view(KVH, m, G, T + n).masked_fill_(~mask[None, :, None, :], -math.inf)
        w = torch.exp(w - w.amax(dim=-1, keepdim=True))
        w = (w / w.sum(dim=-1, keepdim=True)).view(KVH, m * G, T + n)
        o = torch.matmul(w, v).view(KVH, m, G, D).permute(1, 0, 2, 3).reshape(m, H, D)
        out.append(o.to(s["q"].dtype))
        at, node, row = at + T + n, node + n, row + m
    return torch.cat(out)


def _plain_accept(s):
    """The walk for the whole batch at once, a node index at a time; in 64 bits, since decisions and draws
    stand next to borders and the sums run over the vocabulary."""
    n, temp = s["n"], float(np.float32(s["case"]["T"]))
    B, V = len(n), s["case"]["V"]
    first = torch.tensor(np.cumsum([0] + n[:-1]), device=DEV)
    count = torch.tensor(n, device=DEV)

    def probs(logits, rows):
        x = logits[rows].double() / temp
        x = torch.exp(x - x.amax(dim=1, keepdim=True))
        return x / x.sum(dim=1, keepdim=True)

    pick = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.long, device=DEV)
    p = probs(s["t"], first)
    q = probs(s["d"], first) if s["d"] is not None else None
    c, left = torch.zeros(B, 1, dtype=torch.float64, device=DEV), torch.ones(B, dtype=torch.float64, device=DEV)
    path = torch.full((B, max(n)), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    taken = torch.zeros(B, dtype=torch.long, device=DEV)
    for j in range(1, max(n)):
        row = first + torch.clamp(count - 1, max=j)
        child = (j < count) & (s["parents"][row].long() == cur)
        x = s["tok"][row].long()
        u = s["u"][row].double()
        if q is None:
            have, mass = p[pick, x], p.sum(dim=1)
            yes = child & (u * mass < have)
            p[pick, x] = torch.where(child & ~yes, torch.zeros_like(have), have)
        else:
            rest = torch.clamp(p - c * q, min=0.0)
            mass, qx = rest.sum(dim=1), q[pick, x]
            yes = child & (u * qx * mass < rest[pick, x] * left)
            no = child & ~yes
            c = torch.where(no, c[:, 0] + mass / left, c[:, 0])[:, None]
            left = torch.where(no, left - qx, left)
        cur = torch.where(yes, torch.full_like(cur, j), cur)
        taken = taken + yes
        path[pick, taken] = torch.where(yes, torch.full_like(path[:, 0], j), path[pick, taken])
        new = probs(s["t"], first + cur)
        p = torch.where(yes[:, None], new, p)
        if q is not None:
            q = torch.where(yes[:, None], probs(s["d"], first + cur), q)
            c = torch.where(yes[:, None], torch.zeros_like(c), c)
            left = torch.where(yes, torch.ones_like(left), left)
    rest = p if q is None else torch.clamp(p - c * q, min=0.0)
    cum = torch.cumsum(rest, dim=1)
    nxt = (cum <= s["u"][first].double()[:, None] * cum[:, -1:]).sum(dim=1)
    return path, taken.to(torch.int32), torch.clamp(nxt, max=V - 1).to(torch.int32)


def _plain_keep(s):
    case = s["case"]
    rows = [torch.tensor(p, device=DEV) for p in s["paths"]]
    out = ([], [])
    for layer in range(case["L"]):
        for got, old, new in ((out[0], s["K"], s["k"]), (out[1], s["V"], s["v"])):
            at, node, parts = 0, 0, []
            for T, n, r in zip(s["T"], s["n"], rows):
                kept = torch.cat([old[layer, at:at + T], new[layer, node + r].to(torch.bfloat16)])
                parts.append(kept.transpose(0, 1).reshape(-1))
                at, node = at + T, node + n
            got.append(torch.cat(parts))
    return [out[0], out[1]]


PLAIN = dict(rope=_plain_rope, tree=_plain_tree, accept=_plain_accept, keep=_plain_keep)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "rope":
        e = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * case["D"] * e + 4 * case["rows"], "flops": 3 * n * case["rd"]}
    T, n = _lens(case)
    if op == "accept":
        # the root's rows of every sequence (where the walk goes from there is in the values)
        rows = case["B"] * (2 if case["draft"] else 1)
        return {"bytes": 4 * rows * case["V"] + 12 * sum(n), "flops": 4 * rows * case["V"]}
    KVH, D, e = case["KVH"], case["D"], 2 if case["dtype"] == "bf16" else 4
    if op == "keep":
        kept = sum(len(p) for p in _paths(case))
        row = case["L"] * KVH * D * 2  # K and V elements of a token
        return {"bytes": row * (e * sum(n) + 2 * sum(T) + 2 * (sum(T) + kept)), "flops": row * kept}
    H, nq = case["H"], _queries(case)
    pairs = 0
    for a, m, parents in zip(T, nq, _trees(case)):
        depth = []
        for p in parents:
            depth.append(1 + (depth[p] if p >= 0 else 0))
        pairs += m * a + sum(depth[len(parents) - m:])
    return {"bytes": (sum(T) + sum(n)) * KVH * D * 4 + 2 * sum(nq) * H * D * e + 4 * sum(n),
            "flops": 4 * pairs * H * D}


# ---- what the results are, in 64 bits ------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "rope":
        inv, scale = _freqs(case)
        x, rd = s["x"].double(), case["rd"]
        turn = torch.polar(torch.full((case["rows"], rd // 2), scale, dtype=torch.float64, device=DEV),
                           torch.outer(s["pos"].double(), torch.from_numpy(inv).to(DEV).double()))[:, None, :]
        if case["layout"] == "pairs":
            z = torch.view_as_complex(x[..., :rd].reshape(*x.shape[:2], rd // 2, 2).contiguous()) * turn
            x[..., :rd] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :rd // 2], x[..., rd // 2:rd]) * turn
            x[..., :rd] = torch.cat([z.real, z.imag], dim=-1)
        return x
    T, n = _lens(case)
    trees = _trees(case)
    if op == "tree":
        return _exact_tree(case, s, T, n, trees)
    if op == "accept":
        return _exact_accept(case, s, n, trees)
    out = [[], []]
    for layer in range(case["L"]):
        for i, (old, new) in enumerate(((s["K"], s["k"]), (s["V"], s["v"]))):
            ctx, add = torch.split(old[layer], T), torch.split(new[layer].to(torch.bfloat16), n)
            out[i].append(torch.cat([torch.cat([a, b[p]]).permute(1, 0, 2).flatten()
                                     for a, b, p in zip(ctx, add, _paths(case))]).double())
    return out


def _exact_tree(case, s, T, n, trees):
    H, KVH, D = case["H"], case["KVH"], case["D"]
    G, nq = H // KVH, _queries(case)
    K, V = torch.split(s["K"], [a + b for a, b in zip(T, n)]), torch.split(s["V"], [a + b for a, b in zip(T, n)])
    out = []
    for i, q in enumerate(torch.split(s["q"], nq)):
        bias = np.zeros((nq[i], T[i] + n[i]))
        bias[:, T[i]:] = -np.inf
        for m in range(nq[i]):
            bias[m, [T[i] + a for a in _up(trees[i], n[i] - nq[i] + m)]] = 0.0
        bias = torch.from_numpy(bias).to(DEV).repeat_interleave(G, dim=0)
        o = torch.empty(nq[i], H, D, dtype=torch.float64, device=DEV)
        for h in range(KVH):
            qh = q[:, h * G:(h + 1) * G].reshape(nq[i] * G, D).double() / math.sqrt(D)
            w = torch.softmax(torch.addmm(bias, qh, K[i][:, h].double().t().contiguous()), dim=-1)
            o[:, h * G:(h + 1) * G] = torch.matmul(w, V[i][:, h].double()).view(nq[i], G, D)
        out.append(o)
    return torch.cat(out)


def _exact_accept(case, s, n, trees):
    """Sequence by sequence: the residual distributions themselves, renormalised after every rejection."""
    temp = np.float64(np.float32(case["T"]))
    tok, us = s["tok"].cpu().numpy(), s["u"].cpu().numpy().astype(np.float64)

    def probs(row):
        x = row.cpu().numpy().astype(np.float64) / temp
        x = np.exp(x - x.max())
        return x / x.sum()

    path, acc, nxt, at = np.full((len(n), max(n)), -1, np.int32), [], [], 0
    for b, parents in enumerate(trees):
        node, steps = 0, [0]
        while True:
            p = probs(s["t"][at + node])
            q = probs(s["d"][at + node]) if case["draft"] else None
            went = None
            for c in [j for j in range(1, n[b]) if parents[j] == node]:
                x, u = tok[at + c], us[at + c]
                if q is None:
                    if u < p[x]:
                        went = c
                        break
                    p[x] = 0.0
                else:
                    if u * q[x] < p[x]:
                        went = c
                        break
                    p = np.maximum(p - q, 0.0)
                    q[x] = 0.0
                    q = q / q.sum()
                p = p / p.sum()
            if went is None:
                break
            node = went
            steps.append(node)
        path[b, :len(steps)] = steps
        acc.append(len(steps) - 1)
        nxt.append(min(int(np.searchsorted(np.cumsum(p), us[at] * p.sum(), side="right")), case["V"] - 1))
        at += n[b]
    return tuple(torch.tensor(np.asarray(a, np.int32), device=DEV) for a in (path, acc, nxt))
