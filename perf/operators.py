"""The cache-side operators of drafted decoding, as they are measured: attention of a
tree of drafted tokens over a KV cache (with or without the accumulated attention weight
of every cached row), acceptance of a verified tree with the append of its accepted rows,
and eviction of the rows that drew the least attention.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from a seed,
``run`` makes one pass: the plain form in elementary torch operations (``own = False``)
or the framework's entry points (``own = True``). Lengths, node counts and accepted
counts are functions of the case alone, so ``work`` knows them; every value is drawn.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# -----------------------------------------------------------------------------
# cases
# -----------------------------------------------------------------------------
def _attend(name, dtype, T, H, Hkv, d, m, lo, hi, Lmax, weights=False):
    return {"name": name, "op": "attend", "dtype": dtype, "T": T, "H": H, "Hkv": Hkv, "d": d, "m": m, "lo": lo,
            "hi": hi, "Lmax": Lmax, "weights": weights}


def _accept(name, dtype, layers, T, Hkv, d, m, longest, lo, hi, Lmax):
    return {"name": name, "op": "accept", "dtype": dtype, "layers": layers, "T": T, "Hkv": Hkv, "d": d, "m": m,
            "longest": longest, "lo": lo, "hi": hi, "Lmax": Lmax}


def _evict(name, dtype, layers, T, Hkv, d, lo, hi, Lmax, budget, recent, sinks):
    return {"name": name, "op": "evict", "dtype": dtype, "layers": layers, "T": T, "Hkv": Hkv, "d": d, "lo": lo,
            "hi": hi, "Lmax": Lmax, "budget": budget, "recent": recent, "sinks": sinks}


def listed():
    return [
        # one token of one trace over a short cache: the latency of a chat's first steps
        _attend("attend-one-token", "fp16", 1, 16, 16, 128, 1, 203, 203, 256),
        # the decoder's own shape: 16 traces after a 512-token prompt, 8 drafted tokens each
        _attend("attend-draft-8", "fp16", 16, 16, 16, 128, 8, 512, 752, 768),
        # a full tree over grouped heads of 64; one trace has nothing in its cache yet
        _attend("attend-tree-63-grouped", "bf16", 8, 32, 4, 64, 63, 0, 2041, 2112),
        # a batch of long, unequal traces with 32 nodes each: the largest call
        _attend("attend-tree-32-long", "bf16", 16, 32, 8, 128, 32, 3001, 16001, 16384),
        # one very long trace, one token: the cache has to be shared among all SMs
        _attend("attend-one-long", "fp16", 1, 32, 8, 128, 1, 130001, 130001, 131072),
        # a decode step that keeps the score of each cached row, one token per trace
        _attend("attend-score-4096", "fp16", 16, 16, 16, 128, 1, 4096, 4096, 4096, weights=True),
        # the same while verifying trees over grouped heads
        _attend("attend-score-tree-16", "bf16", 4, 32, 8, 128, 16, 1001, 8191, 8192, weights=True),
        # a small model's verified chain: nothing but latency
        _accept("accept-small", "fp16", 2, 1, 2, 64, 5, 3, 37, 37, 64),
        # all 24 layers of the decoder's shape after a verification step
        _accept("accept-24-layers", "fp16", 24, 16, 16, 128, 16, 6, 512, 740, 768),
        # a short cache that has just outgrown its budget
        _evict("evict-small", "fp16", 1, 1, 4, 64, 300, 300, 320, 256, 32, 4),
        # all 24 layers of the decoder's shape brought back to 512 rows
        _evict("evict-24-layers", "fp16", 24, 16, 16, 128, 600, 760, 768, 512, 64, 4),
        # long caches halved
        _evict("evict-long", "bf16", 2, 4, 8, 128, 60001, 65536, 65536, 32768, 1024, 4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        b, f = limits.get(c["op"], (0, 0))
        limits[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        op = rng.choice(["attend", "attend", "attend", "accept", "evict", "evict"])
        T = _log_int(rng, 1, 32)
        Hkv = rng.choice([1, 2, 4, 8, 16])
        d = rng.choice([64, 80, 96, 128, 128])
        dtype = rng.choice(["fp16", "bf16"])
        if op == "attend":
            m = _log_int(rng, 1, 64)
            hi = _log_int(rng, 16, 131000)
            lo = rng.choice([0, hi // 2, hi])
            c = _attend("", dtype, T, Hkv * rng.choice([1, 2, 4, 8]), Hkv, d, m, lo, hi, hi + rng.randrange(0, 65),
                        weights=rng.random() < 0.4)
        elif op == "accept":
            m = _log_int(rng, 2, 64)
            hi = _log_int(rng, 16, 2000)
            c = _accept("", dtype, rng.choice([1, 2, 12, 22, 24]), T, Hkv, d, m, rng.randint(1, min(m, 8)), hi // 2, hi,
                        hi + m + rng.randrange(0, 65))
        else:
            hi = _log_int(rng, 64, 65536)
            budget = max(16, int(hi * rng.uniform(0.3, 0.95)))
            c = _evict("", dtype, rng.choice([1, 2, 12, 22, 24]), T, Hkv, d, rng.choice([hi // 4, hi * 3 // 4, hi]), hi,
                       hi + rng.randrange(0, 65), budget, rng.randint(1, budget // 4), rng.randint(0, 4))
        w = work(c)
        state = (c.get("layers", 1) * T * Hkv * c["Lmax"] * d * 4 +
                 (T * c["H"] * c["m"] * c["Lmax"] * 4 if op == "attend" else 0))
        if w["bytes"] <= limits[op][0] and w["flops"] <= limits[op][1] and state <= 4.5e9:
            del c["name"]
            return c


def _lens(c):
    """Valid cache rows of each trace: spread evenly over [lo, hi] in a mixed order."""
    T = c["T"]
    if T == 1:
        return [c["hi"]]
    return [c["lo"] + (c["hi"] - c["lo"]) * ((t * 7 + 3) % T) // (T - 1) for t in range(T)]


def _nodes(c):
    """Drafted nodes of each trace: every third trace has drafted fewer than m."""
    return [c["m"] - (c["m"] // 3 if t % 3 == 2 else 0) for t in range(c["T"])]


def _accepted(c):
    return [1 + (t * 5 + c["longest"] // 2) % c["longest"] for t in range(c["T"])]


def work(case):
    c, lens = case, _lens(case)
    if c["op"] == "attend":
        nodes = _nodes(c)
        rows = c["T"] * c["m"]
        data = 2 * (2 * c["Hkv"] * c["d"] * (sum(lens) + rows) + 2 * rows * c["H"] * c["d"]) + 8 * rows + 4 * c["T"]
        if c["weights"]:
            data += 4 * c["Hkv"] * (2 * sum(lens) + rows)
        flops = 4 * c["H"] * c["d"] * sum(n * (length + 1) for n, length in zip(nodes, lens))
        return {"bytes": data, "flops": flops}
    if c["op"] == "accept":
        n = c["layers"] * c["Hkv"] * sum(_accepted(c))
        return {"bytes": n * (8 * c["d"] + 12) + 16 * c["T"] * c["m"] + 24 * c["T"], "flops": c["T"] * c["m"]}
    data = 0
    for length in lens:
        kept = min(length, c["budget"])
        if length > kept:  # rows of the tail that stay: the recent ones, and their share of the others
            tail, old = length - kept, length - c["recent"] - c["sinks"]
            recent = min(c["recent"], tail)
            moved = recent + (tail - recent) * (kept - c["recent"] - c["sinks"]) / old
        else:
            moved = 0
        data += 8 * length + 8 * kept + moved * 8 * c["d"]
    n = c["layers"] * c["Hkv"]
    return {"bytes": int(n * data) + 12 * c["T"], "flops": n * sum(lens)}


# -----------------------------------------------------------------------------
# inputs
# -----------------------------------------------------------------------------
def _tree(rng, n, m):
    """Parents of a random tree of n nodes in topological order, padded with -1 to m."""
    return [-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, n)] + [-1] * (m - n)


def _masks(parents, n):
    """Ancestors-or-self of each node as the bits of a signed 64-bit integer; 0 for padding."""
    out = []
    for i, p in enumerate(parents):
        bits = 0 if i >= n else (1 << i) | (out[p] & (2 ** 64 - 1) if p >= 0 else 0)
        out.append(bits - 2 ** 64 if bits >= 2 ** 63 else bits)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    rng = random.Random(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=dt):
        return torch.randn(shape, dtype=dtype, device="cuda", generator=g)

    T, Hkv, d, Lmax = c["T"], c["Hkv"], c["d"], c["Lmax"]
    lens = _lens(c)
    s = {"case": c, "lens": _i32(lens)}
    if c["op"] == "attend":
        H, m = c["H"], c["m"]
        s["k"], s["v"] = normal(T, Hkv, Lmax, d), normal(T, Hkv, Lmax, d)
        qkv = normal(T, m, (H + 2 * Hkv) * d)  # the projection's output; its values are read in place
        s["q"] = normal(T, m, H, d) * 1.5
        s["kd"] = normal(T, m, Hkv, d)
        s["vd"] = qkv[:, :, (H + Hkv) * d:].view(T, m, Hkv, d)
        s["masks"] = torch.tensor([_masks(_tree(rng, n, m), n) for n in _nodes(c)], dtype=torch.int64, device="cuda")
        s["out"] = torch.zeros_like(s["q"])
        if c["weights"]:
            rows = torch.arange(Lmax, device="cuda")
            seen = rows < s["lens"].view(T, 1, 1)
            s["scores"] = torch.where(seen, normal(T, Hkv, Lmax, dtype=torch.float32).exp(), 0.0)
            s["scores_out"] = torch.zeros_like(s["scores"])
            s["draft_scores"] = torch.zeros((T, Hkv, m), dtype=torch.float32, device="cuda")
        return s

    layers = c["layers"]
    s["k"], s["v"] = normal(layers, T, Hkv, Lmax, d), normal(layers, T, Hkv, Lmax, d)
    if c["op"] == "accept":
        m = c["m"]
        tokens, parents, target = [], [], []
        for t, count in enumerate(_accepted(c)):
            path = [0] + sorted(rng.sample(range(1, m), count - 1))
            par = [-1] + [rng.randrange(i) for i in range(1, m)]
            for a, b in zip(path, path[1:]):
                par[b] = a
            tok = rng.sample(range(32000), m)
            tgt = [rng.randrange(32000, 32064) for _ in range(m)]  # no drafted token unless on the path
            for a, b in zip(path, path[1:]):
                tgt[a] = tok[b]
            tokens.append(tok)
            parents.append(par)
            target.append(tgt)
        s.update(tokens=_i32(tokens), parents=_i32(parents), target=_i32(target))
        s["next_pos"] = s["lens"] + 100  # some rows have been evicted before
        s["kd"] = normal(layers, T, m, Hkv, d)
        s["vd"] = normal(layers, T, m, Hkv, d)
        s["draft_scores"] = normal(layers, T, Hkv, m, dtype=torch.float32).exp()
        s["scores"] = normal(layers, T, Hkv, Lmax, dtype=torch.float32).exp()
        s["positions"] = torch.arange(Lmax, dtype=torch.int32, device="cuda").repeat(layers, T, Hkv, 1)
        return s

    # Accumulated weights are heavy-tailed, and rows that no query ever looked at hold an
    # exact zero. Rows left by earlier evictions are out of order; the newest lie at the end.
    w = (1.5 * normal(layers, T, Hkv, Lmax, dtype=torch.float32)).exp()
    s["scores"] = torch.where(torch.rand(w.shape, device="cuda", generator=g) < 0.2, 0.0, w)
    pos = torch.empty((layers, T, Hkv, Lmax), dtype=torch.int32, device="cuda")
    for t, length in enumerate(lens):
        base = torch.arange(Lmax, dtype=torch.int32, device="cuda") * 2
        mixed = length * 3 // 4
        if mixed > 1:
            base[:mixed] = base[torch.randperm(mixed, device="cuda", generator=g)]
        pos[:, t] = base
    s["positions"] = pos
    s["next_pos"] = s["lens"] * 2
    s["scores_out"] = torch.zeros_like(s["scores"])
    s["positions_out"] = torch.zeros_like(pos)
    return s


# -----------------------------------------------------------------------------
# one pass
# -----------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _own_attend, "accept": _own_accept, "evict": _own_evict}[op](state)
    return {"attend": _plain_attend, "accept": _plain_accept, "evict": _plain_evict}[op](state)


def _own_attend(s):
    from moat_b200.tree import tree_attention
    if not s["case"]["weights"]:
        return tree_attention(s["q"], s["k"], s["v"], s["lens"], s["kd"], s["vd"], s["masks"], out=s["out"])
    return tree_attention(s["q"], s["k"], s["v"], s["lens"], s["kd"], s["vd"], s["masks"], out=s["out"],
                          scores=s["scores"], scores_out=s["scores_out"], draft_scores=s["draft_scores"])


def _own_accept(s):
    from moat_b200.tree import accept_tree
    a = accept_tree(s["tokens"], s["parents"], s["target"], s["lens"], s["next_pos"], s["k"], s["v"], s["kd"], s["vd"],
                    scores=s["scores"], draft_scores=s["draft_scores"], positions=s["positions"])
    return [a.path, a.counts, a.next_ids, a.lens, a.next_pos, s["k"], s["v"], s["scores"], s["positions"]]


def _own_evict(s):
    from moat_b200.evict import evict_cache
    c = s["case"]
    scores, positions, lens = evict_cache(s["k"], s["v"], s["scores"], s["positions"], s["lens"], s["next_pos"],
                                          c["budget"], recent=c["recent"], sinks=c["sinks"],
                                          scores_out=s["scores_out"], positions_out=s["positions_out"])
    return [scores, positions, lens, s["k"], s["v"]]


def _plain_attend(s):
    c = s["case"]
    T, H, Hkv, d, m, Lmax = c["T"], c["H"], c["Hkv"], c["d"], c["m"], c["Lmax"]
    G = H // Hkv
    q = s["q"].float().view(T, m, Hkv, G, d).permute(0, 2, 1, 3, 4).reshape(T, Hkv, m * G, d)
    keys = torch.cat([s["k"].float(), s["kd"].float().transpose(1, 2)], dim=2)
    values = torch.cat([s["v"].float(), s["vd"].float().transpose(1, 2)], dim=2)
    dev = q.device
    node = torch.arange(m, device=dev)
    in_tree = (s["masks"].unsqueeze(-1) >> node) & 1  # [T, m, m]
    real = s["masks"] != 0
    in_cache = (torch.arange(Lmax, device=dev) < s["lens"].view(T, 1)).view(T, 1, Lmax) & real.view(T, m, 1)
    see = torch.cat([in_cache, in_tree.bool()], dim=2)  # [T, m, Lmax + m]
    see = see.view(T, 1, m, 1, Lmax + m).expand(T, 1, m, G, Lmax + m).reshape(T, 1, m * G, Lmax + m)
    x = torch.matmul(q, keys.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    x.masked_fill_(~see, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(dim=-1, keepdim=True)
    x.div_(torch.where(total == 0.0, 1.0, total))
    out = torch.matmul(x, values).view(T, Hkv, m, G, d).permute(0, 2, 1, 3, 4).reshape(T, m, H, d).to(s["q"].dtype)
    if not c["weights"]:
        return out
    w = x.sum(dim=2)
    cached = torch.arange(Lmax, device=dev) < s["lens"].view(T, 1, 1)
    return [out, torch.where(cached, s["scores"] + w[:, :, :Lmax], s["scores_out"]), w[:, :, Lmax:].contiguous()]


def _plain_accept(s):
    c = s["case"]
    layers, T, Hkv, d, m = c["layers"], c["T"], c["Hkv"], c["d"], c["m"]
    tokens, parents, target = s["tokens"].long(), s["parents"].long(), s["target"].long()
    node = torch.arange(m, device=tokens.device)
    real = (parents >= 0) & (parents < node)
    up = torch.where(real, parents, 0)
    agrees = real & (tokens >= 0) & (tokens == target.gather(1, up))
    twin = ((parents.unsqueeze(1) == parents.unsqueeze(2)) & (tokens.unsqueeze(1) == tokens.unsqueeze(2))
            & agrees.unsqueeze(1) & (node < node.view(m, 1)))  # an earlier sibling drafted the same token
    good = (agrees & ~twin.any(dim=2)) | (node == 0)
    for _ in range(6):  # a node is accepted if it and all its ancestors agree
        good = good & good.gather(1, up)
        up = up.gather(1, up)
    counts = good.sum(dim=1)
    order = torch.where(good, node, m).sort(dim=1).values
    taken = order < m
    path = torch.where(taken, order, -1)
    last = order.gather(1, (counts - 1).unsqueeze(1))
    next_ids = target.gather(1, last).squeeze(1)
    src = torch.where(taken, order, 0)
    dst = s["lens"].long().unsqueeze(1) + node
    write = taken.view(1, T, 1, m, 1).expand(layers, T, Hkv, m, d)
    rows_src = src.view(1, T, m, 1, 1).expand(layers, T, m, Hkv, d)
    rows_dst = dst.view(1, T, 1, m, 1).expand(layers, T, Hkv, m, d)
    for cache, draft in ((s["k"], s["kd"]), (s["v"], s["vd"])):
        new = draft.gather(2, rows_src).transpose(2, 3)
        cache.scatter_(3, rows_dst, torch.where(write, new, cache.gather(3, rows_dst)))
    flat = dst.view(1, T, 1, m).expand(layers, T, Hkv, m)
    put = write[..., 0]
    new = s["draft_scores"].gather(3, src.view(1, T, 1, m).expand(layers, T, Hkv, m))
    s["scores"].scatter_(3, flat, torch.where(put, new, s["scores"].gather(3, flat)))
    new = (s["next_pos"].unsqueeze(1) + node).to(torch.int32).view(1, T, 1, m).expand(layers, T, Hkv, m)
    s["positions"].scatter_(3, flat, torch.where(put, new, s["positions"].gather(3, flat)))
    n = counts.to(torch.int32)
    return [path.to(torch.int32), n, next_ids.to(torch.int32), s["lens"] + n, s["next_pos"] + n, s["k"], s["v"],
            s["scores"], s["positions"]]


def _plain_evict(s):
    c = s["case"]
    T, Lmax, top = c["T"], c["Lmax"], min(c["budget"], c["Lmax"])
    dev = s["scores"].device
    rows = torch.arange(Lmax, device=dev)
    lens = s["lens"].view(1, T, 1, 1)
    kept = lens.clamp(max=c["budget"])
    pos = s["positions"]
    guarded = (pos >= s["next_pos"].view(1, T, 1, 1) - c["recent"]) | (pos < c["sinks"])
    key = torch.where(guarded, math.inf, s["scores"])
    key = torch.where(rows < lens, key, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    stays = torch.zeros_like(guarded).scatter_(3, order, (rows < kept).expand_as(guarded))
    hole = ~stays & (rows < kept)
    mover = stays & (rows >= kept)
    place = torch.where(mover, mover.cumsum(dim=-1) - 1, Lmax)
    source = torch.zeros(key.shape[:-1] + (Lmax + 1,), dtype=torch.int64, device=dev)
    source.scatter_(3, place, rows.expand_as(place))
    src = torch.where(hole, source.gather(3, (hole.cumsum(dim=-1) - 1).clamp(min=0)), rows)[..., :top]
    live = rows[:top] < kept
    for cache in (s["k"], s["v"]):
        cache[..., :top, :] = cache.gather(3, src.unsqueeze(-1).expand(*src.shape, c["d"]))
    scores, positions = s["scores_out"].clone(), s["positions_out"].clone()
    scores[..., :top] = torch.where(live, s["scores"].gather(3, src), scores[..., :top])
    positions[..., :top] = torch.where(live, pos.gather(3, src), positions[..., :top])
    return [scores, positions, s["lens"].clamp(max=c["budget"]), s["k"], s["v"]]


# -----------------------------------------------------------------------------
# the definitions in 64 bits
# -----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "accept": _exact_accept, "evict": _exact_evict}[case["op"]](s)


def _exact_attend(s):
    """Trace by trace and head by head: the visible rows alone, softmax by its logarithm."""
    c = s["case"]
    T, H, Hkv, m = c["T"], c["H"], c["Hkv"], c["m"]
    G = H // Hkv
    lens, masks = s["lens"].tolist(), s["masks"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if c["weights"]:
        scores = s["scores_out"].double()
        draft = torch.zeros(s["draft_scores"].shape, dtype=torch.float64, device="cuda")
    for t in range(T):
        n, nodes = lens[t], [i for i in range(m) if masks[t][i] != 0]
        hidden = torch.tensor([[not (masks[t][i] >> j) & 1 for j in range(m)] for i in nodes], device="cuda")
        for h in range(Hkv):
            k = torch.cat([s["k"][t, h, :n], s["kd"][t, :, h]]).double()
            v = torch.cat([s["v"][t, h, :n], s["vd"][t, :, h]]).double()
            seen = torch.zeros(n + m, dtype=torch.float64, device="cuda")
            for g in range(G):
                x = s["q"][t, nodes, h * G + g].double() @ k.T / c["d"] ** 0.5
                x[:, n:][hidden] = -math.inf
                p = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
                out[t, nodes, h * G + g] = p @ v
                seen += p.sum(dim=0)
            if c["weights"]:
                scores[t, h, :n] = s["scores"][t, h, :n].double() + seen[:n]
                draft[t, h] = seen[n:]
    return [out, scores, draft] if c["weights"] else out


def _exact_accept(s):
    """The walk itself on the host; rows that are copied have no computed value."""
    c = s["case"]
    tokens, parents, target = (s[n].tolist() for n in ("tokens", "parents", "target"))
    path = np.full((c["T"], c["m"]), -1, np.int32)
    counts, ids = [], []
    for t in range(c["T"]):
        node, n = 0, 0
        while node is not None:
            path[t, n], n, last = node, n + 1, node
            node = next((i for i in range(last + 1, c["m"])
                         if parents[t][i] == last and tokens[t][i] == target[t][last]), None)
        counts.append(n)
        ids.append(target[t][last])
    n = _i32(counts)
    return [torch.from_numpy(path).cuda(), n, _i32(ids), s["lens"] + n, s["next_pos"] + n, None, None, None, None]


def _exact_evict(s):
    """Row by row on the host: the rows that stay, and the holes filled in order."""
    c = s["case"]
    if c["layers"] * c["Hkv"] * sum(_lens(c)) > 3e7:
        return None
    score, pos = s["scores"].cpu().numpy(), s["positions"].cpu().numpy()
    new_score, new_pos = s["scores_out"].cpu().numpy().copy(), s["positions_out"].cpu().numpy().copy()
    for t, length in enumerate(_lens(c)):
        kept = min(length, c["budget"])
        for layer in range(c["layers"]):
            for h in range(c["Hkv"]):
                p, w = pos[layer, t, h, :length], score[layer, t, h, :length]
                safe = (p >= 2 * length - c["recent"]) | (p < c["sinks"])
                best = np.lexsort((np.arange(length), -w.astype(np.float64), ~safe))[:kept]
                src, inside = np.arange(kept), np.zeros(length, bool)
                inside[best] = True
                src[~inside[:kept]] = kept + np.flatnonzero(inside[kept:])
                new_score[layer, t, h, :kept], new_pos[layer, t, h, :kept] = w[src], p[src]
    lens = [min(n, c["budget"]) for n in _lens(c)]
    return [torch.from_numpy(new_score).double().cuda(), torch.from_numpy(new_pos).cuda(), _i32(lens), None, None]
