"""Cases of the draft-tree and cache operators: tree attention over a KV cache, the attention
weight each cached row receives, eviction by that weight, and committing an accepted path.

Every case can be computed in a plain form (elementary torch operations in fp32) and, with
``own`` true, by the library's kernels through ``jinf.kernels``. ``exact`` computes the same
outputs from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

# (query heads, kv heads, head size) of the model shapes: the tiny test model, 8B, 70B
TINY, B8, B70 = (8, 2, 64), (32, 8, 128), (64, 8, 128)


def _attn(name, op, shape, dtype, seqs, nodes, past, accepted=0, tree=True):
    d = {"op": op, "heads": shape[0], "kv_heads": shape[1], "hd": shape[2], "dtype": dtype, "seqs": seqs,
         "nodes": nodes, "past": past, "tree": tree}
    if op == "mass":
        d["accepted"] = accepted
    return dict(d, name=name) if name else d


def _evict(name, shape, dtype, seqs, rows, keep, sink, recent):
    d = {"op": "evict", "heads": shape[0], "kv_heads": shape[1], "hd": shape[2], "dtype": dtype, "seqs": seqs,
         "rows": rows, "keep": keep, "sink": sink, "recent": recent}
    return dict(d, name=name) if name else d


def _commit(name, shape, dtype, seqs, nodes, past, accepted):
    d = {"op": "commit", "heads": shape[0], "kv_heads": shape[1], "hd": shape[2], "dtype": dtype, "seqs": seqs,
         "nodes": nodes, "past": past, "accepted": accepted}
    return dict(d, name=name) if name else d


def listed():
    return [
        # the start of a generation with the tiny test model: five drafts after a short prompt, launch latency
        _attn("tree tiny 5 nodes", "tree", TINY, "f16", 1, 5, 37),
        # one token of each of eight sequences, 8B heads, lengths spread up to 8192: plain batched decode
        _attn("tree 8b 8 seqs 1 token", "tree", B8, "f16", 8, 1, 8191, tree=False),
        # an ordinary draft tree over an ordinary context, 8B heads
        _attn("tree 8b 26 nodes 4k", "tree", B8, "f16", 1, 26, 4097),
        # a wide tree at the 70B shape's full training context
        _attn("tree 70b 64 nodes 8k", "tree", B70, "bf16", 1, 64, 8128),
        # an odd tree over a long context, 70B heads
        _attn("tree 70b 33 nodes 128k", "tree", B70, "f16", 1, 33, 131001),
        # the accepted path of an ordinary tree, credited to the rows it attended to
        _attn("mass 8b 5 of 26 nodes 4k", "mass", B8, "f16", 1, 26, 4097, accepted=5),
        # the same for eight sequences of different lengths, every node counted
        _attn("mass 8b 8 seqs 16 nodes", "mass", B8, "f16", 8, 16, 8000, accepted=16),
        # a chunk of a long prompt, every row credited (causal, no tree)
        _attn("mass 70b 256 chunk 32k", "mass", B70, "bf16", 1, 256, 32769, accepted=256, tree=False),
        # one layer's cache cut back to a quarter at the 8B training context
        _evict("evict 8b 8k to 2k", B8, "f16", 1, 8192, 2048, 4, 256),
        # all 32 layers of an 8B model cut back from 32k rows at once
        _evict("evict 8b 32 layers 32k to 8k", B8, "f16", 32, 32771, 8192, 4, 1023),
        # the accepted path of one sequence, all 32 layers of an 8B model
        _commit("commit 8b 32 layers", B8, "f16", 32, 26, 1500, 5),
        # eight sequences of a 70B model, ten layers of each (one device's share of a pipeline)
        _commit("commit 70b 8 seqs 10 layers", B70, "bf16", 80, 64, 700, 9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "mass", "evict", "commit"])
    shape = rng.choice([TINY, B8, B70, (4, 4, 128), (24, 2, 64), (16, 1, 128)])
    dtype = rng.choice(["f16", "bf16"])
    if op == "evict":
        rows = _log(rng, 64, 65536)
        seqs = _log(rng, 1, max(1, min(32, 32 * 32768 * 8 // (rows * shape[1] * 2))))
        keep = _log(rng, 16, rows)
        sink = rng.randint(0, min(4, keep // 4))
        return _evict(None, shape, dtype, seqs, rows, keep, sink, rng.randint(0, (keep - sink) // 2))
    if op == "commit":
        nodes = _log(rng, 2, 128)
        return _commit(None, shape, dtype, _log(rng, 1, 80), nodes, rng.randint(0, 1500),
                       rng.randint(1, min(nodes, 12)))
    seqs = rng.choice([1, 1, 1, rng.randint(2, 8)])
    nodes = _log(rng, 1, 256)
    accepted = rng.choice([nodes, rng.randint(1, min(nodes, 8))]) if op == "mass" else 0
    past = _log(rng, 1, 131072)
    # no more than the largest listed case of the operator
    most = 64 * 33 * 131072 if op == "tree" else 64 * 256 * 32768
    past = min(past, max(1, most // (seqs * nodes * shape[0])))
    return _attn(None, op, shape, dtype, seqs, nodes, past, accepted, tree=rng.random() < 0.75)


def _kernels():
    root = os.path.join(os.getcwd(), "jetson-inference_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from jinf import kernels
    return kernels


def _type(case):
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _lengths(g, seqs, most):
    """One length per sequence: the first the longest, the others spread below it."""
    f = 0.25 + 0.75 * torch.rand(seqs, generator=g, device="cuda")
    f[0] = 1.0
    return (f * most).to(torch.int32)


def _tree(seed, nodes):
    """Parents of a random tree (parent < node, -1: a root) and the visibility it gives."""
    g = torch.Generator()
    g.manual_seed(int(seed) + 1)
    u = torch.rand(nodes, generator=g).tolist()
    parents = [int(t * u[t] ** 0.5) - 1 if t else -1 for t in range(nodes)]
    see = torch.zeros(nodes, nodes, dtype=torch.bool)
    for t in range(nodes):
        if parents[t] >= 0:
            see[t] = see[parents[t]]
        see[t, t] = True
    return parents, see


def _pack(see):
    """[nodes, nodes] truth values -> [nodes, ceil(nodes / 32)] words, bit u % 32 of word u / 32."""
    nodes = see.shape[0]
    words = (nodes + 31) // 32
    bits = torch.zeros(nodes, words * 32, dtype=torch.int64)
    bits[:, :nodes] = see
    w = (bits.view(nodes, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _path(parents, accepted):
    """Nodes of a root-to-leaf path of at most `accepted` nodes, ascending."""
    depth_of, best = [], 0
    for t, p in enumerate(parents):
        depth_of.append(1 if p < 0 else depth_of[p] + 1)
        if depth_of[t] > depth_of[best]:
            best = t
    path = []
    while best >= 0:
        path.append(best)
        best = parents[best]
    return path[::-1][:accepted]


def prepare(case, seed):
    g = _gen(seed)
    dt, hd, nkv, nh, seqs = _type(case), case["hd"], case["kv_heads"], case["heads"], case["seqs"]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=dt)  # noqa: E731
    st = {"case": case}
    if case["op"] in ("tree", "mass"):
        nodes, past = case["nodes"], case["past"]
        ctx = past + nodes + 5
        st["k"], st["v"] = rnd(seqs, nkv, ctx, hd), rnd(seqs, nkv, ctx, hd)
        st["q"] = rnd(seqs, nodes, nh, hd) * 1.5
        st["n_past"] = _lengths(g, seqs, past)
        parents, see = _tree(seed, nodes)
        st["mask"] = _pack(see).cuda() if case["tree"] else None
        st["out"] = torch.empty(seqs, nodes, nh, hd, dtype=dt, device="cuda")
        st["lse"] = torch.empty(seqs, nodes, nh, dtype=torch.float32, device="cuda")
        if case["op"] == "mass":
            st["lse"] = _plain_tree(st, want_out=False)["lse"]
            st["mass"] = torch.rand(seqs, nkv, ctx, generator=g, device="cuda") ** 4 * 3
            w = torch.ones(seqs, nodes)
            if case["accepted"] < nodes:
                chosen = _path(parents, case["accepted"]) if case["tree"] else range(case["accepted"])
                w.zero_()
                w[:, list(chosen)] = 1.0
            st["weight"] = w.cuda()
    elif case["op"] == "evict":
        rows, keep = case["rows"], case["keep"]
        st["k"], st["v"] = rnd(seqs, nkv, rows, hd), rnd(seqs, nkv, rows, hd)
        m = torch.rand(seqs, nkv, rows, generator=g, device="cuda")
        st["mass"] = torch.where(m < 0.02, torch.zeros_like(m), m ** 6 * 40)  # few rows carry most; some none
        st["n_rows"] = _lengths(g, seqs, rows)
        # the cut-back cache: rows past the new length are whatever that memory held
        st["k_out"] = torch.zeros(seqs, nkv, keep, hd, dtype=dt, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
        st["mass_out"] = torch.zeros(seqs, nkv, keep, device="cuda")
        st["ids"] = torch.empty(seqs, nkv, keep, dtype=torch.int32, device="cuda")
        st["n_out"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
    else:
        nodes, past = case["nodes"], case["past"]
        ctx = past + nodes + 5
        st["k"], st["v"] = rnd(seqs, nkv, ctx, hd), rnd(seqs, nkv, ctx, hd)
        st["mass"] = torch.rand(seqs, nkv, ctx, generator=g, device="cuda")
        st["n_past"] = _lengths(g, seqs, past)
        r = torch.rand(seqs, nodes, generator=g, device="cuda")
        n = torch.randint(1, case["accepted"] + 1, (seqs,), generator=g, device="cuda")
        n[0] = case["accepted"]
        first = r.argsort(dim=1)[:, : case["accepted"]]  # some nodes, ascending, -1 past each row's count
        first = torch.where(torch.arange(case["accepted"], device="cuda") < n[:, None], first, nodes)
        first = first.sort(dim=1).values
        st["accepted"] = torch.where(first < nodes, first, -1).to(torch.int32)
        st["n_accepted"] = n.to(torch.int32)
        st["n_out"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
    if own:
        K = _kernels()
        st["kernels"], st["view"] = K, K.KvView(st["k"], st["v"])
        if case["op"] == "evict":
            st["view_out"] = K.KvView(st["k_out"], st["v_out"])
        if case["op"] == "tree":
            st["ws"] = torch.zeros(K.tree_attention_workspace_bytes(st["view"], nh, nodes, past), dtype=torch.uint8,
                                   device="cuda")
    return st


# ---- plain forms ----


def _seen(st, length):
    """[seqs or 1, nodes, length] truth values: the rows each node attends to, of the first `length`."""
    nodes = st["q"].shape[1]
    j = torch.arange(length, device="cuda")
    past = st["n_past"].long()[:, None]
    u = j[None, :] - past  # tree row of each cache row, per sequence
    in_tree = (u >= 0) & (u < nodes)
    uc = u.clamp(0, nodes - 1)
    if st["mask"] is None:
        bit = uc[:, None, :] <= torch.arange(nodes, device="cuda")[None, :, None]
    else:
        words = st["mask"][:, uc // 32]                       # [nodes, seqs, length]
        bit = ((words >> (uc % 32)) & 1).bool().transpose(0, 1)
    return (u < 0)[:, None, :] | (in_tree[:, None, :] & bit)


def _scores(st):
    """fp32 scores [seqs, kv heads, nodes, group, rows], -inf where a node does not attend."""
    q, k = st["q"], st["k"]
    seqs, nodes, nh, hd = q.shape
    nkv = k.shape[1]
    length = min(st["case"]["past"] + nodes, k.shape[2])
    q = q.float().view(seqs, nodes, nkv, nh // nkv, hd).transpose(1, 2).reshape(seqs, nkv, -1, hd)
    s = torch.matmul(q * (1.0 / math.sqrt(hd)), k[:, :, :length].float().transpose(2, 3))
    s = s.view(seqs, nkv, nodes, nh // nkv, length)
    return s.masked_fill_(~_seen(st, length)[:, None, :, None, :], -math.inf)


def _plain_tree(st, want_out=True):
    s = _scores(st)
    seqs, nkv, nodes, group, length = s.shape
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(-1).transpose(1, 2).reshape(seqs, nodes, nkv * group)
    if not want_out:
        return {"lse": lse}
    o = torch.matmul(p.view(seqs, nkv, nodes * group, length), st["v"][:, :, :length].float())
    o = o.view(seqs, nkv, nodes, group, -1) / torch.where(total == 0, 1.0, total)
    out = o.transpose(1, 2).reshape(seqs, nodes, nkv * group, -1)
    return {"out": out.to(st["q"].dtype), "lse": lse}


def _plain_mass(st):
    s = _scores(st)
    seqs, nkv, nodes, group, length = s.shape
    lse = st["lse"].view(seqs, nodes, nkv, group).transpose(1, 2)[..., None]
    p = s.sub_(torch.where(lse == -math.inf, 0.0, lse)).exp_()
    add = (p * st["weight"][:, None, :, None, None]).sum((2, 3))
    rows = torch.arange(length, device="cuda")[None, None, :]
    past = st["n_past"][:, None, None]
    mass = st["mass"]  # updated in place, as it is from step to step
    old = torch.where(rows < past, mass[:, :, :length], 0.0)
    mass[:, :, :length] = torch.where(rows < past + nodes, old + add, mass[:, :, :length])
    return {"mass": mass}


def _plain_evict(st):
    c, mass, n = st["case"], st["mass"], st["n_rows"]
    keep, sink, recent = c["keep"], c["sink"], c["recent"]
    rows = torch.arange(mass.shape[2], device="cuda")[None, None, :]
    n3 = n[:, None, None]
    rank = torch.where(torch.isnan(mass), -math.inf, mass)
    rank = torch.where((rows < sink) | (rows >= n3 - recent) | (n3 <= keep), math.inf, rank)
    live = rows < n3
    # largest first, equal ones by row; rows past the length last
    order = torch.where(live, rank, -math.inf).argsort(dim=-1, descending=True, stable=True)
    order = order.gather(-1, (~live.expand_as(rank)).gather(-1, order).to(torch.int8).argsort(dim=-1, stable=True))
    n_out = n.clamp(max=keep)
    slot = torch.arange(keep, device="cuda")[None, None, :]
    ids = torch.where(slot < n_out[:, None, None], order[:, :, :keep], mass.shape[2]).sort(dim=-1).values
    valid = slot < n_out[:, None, None]
    at = ids.clamp(max=mass.shape[2] - 1)
    row = at[..., None].expand(-1, -1, -1, st["k"].shape[3])
    return {"k": torch.where(valid[..., None], st["k"].gather(2, row), st["k_out"]),
            "v": torch.where(valid[..., None], st["v"].gather(2, row), st["v_out"]),
            "mass": torch.where(valid, mass.gather(2, at), st["mass_out"]),
            "ids": torch.where(valid, ids, -1).to(torch.int32), "n": n_out}


def _plain_commit(st):
    acc, n, past = st["accepted"].long(), st["n_accepted"].long(), st["n_past"].long()
    i = torch.arange(acc.shape[1], device="cuda")[None, :]
    valid = i < n[:, None]
    dst = past[:, None] + i
    src = torch.where(valid, past[:, None] + acc, dst)  # rows past the count stay
    for name in ("k", "v", "mass"):
        t = st[name]
        tail = (1,) * (t.dim() - 3)
        nkv = t.shape[1]
        shape = (t.shape[0], nkv, i.shape[1]) + tuple(t.shape[3:])
        rows = t.gather(2, src.view(src.shape[0], 1, -1, *tail).expand(shape))
        t.scatter_(2, dst.view(dst.shape[0], 1, -1, *tail).expand(shape), rows)
    return {"k": st["k"], "v": st["v"], "mass": st["mass"], "n": (past + n).to(torch.int32)}


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        return {"tree": _plain_tree, "mass": _plain_mass, "evict": _plain_evict, "commit": _plain_commit}[op](st)
    K, c = st["kernels"], st["case"]
    if op == "tree":
        K.tree_attention(st["out"], st["q"], st["view"], st["n_past"], c["past"], st["ws"], mask=st["mask"],
                         lse=st["lse"])
        return {"out": st["out"], "lse": st["lse"]}
    if op == "mass":
        K.attention_mass(st["mass"], st["q"], st["view"], st["n_past"], c["past"], st["lse"], mask=st["mask"],
                         node_weight=st["weight"])
        return {"mass": st["mass"]}
    if op == "evict":
        K.kv_evict(st["view"], st["view_out"], st["mass"], st["mass_out"], st["n_rows"], st["ids"], st["n_out"],
                   c["keep"], c["sink"], c["recent"])
        return {"k": st["k_out"], "v": st["v_out"], "mass": st["mass_out"], "ids": st["ids"], "n": st["n_out"]}
    K.tree_commit(st["view"], st["mass"], st["n_past"], c["past"], st["accepted"], st["n_accepted"], c["nodes"],
                  st["n_out"])
    return {"k": st["k"], "v": st["v"], "mass": st["mass"], "n": st["n_out"]}


def work(case):
    """Each input read once and each output written once; the sequences' lengths by their mean."""
    nkv, nh, hd, seqs = case["kv_heads"], case["heads"], case["hd"], case["seqs"]
    if case["op"] in ("tree", "mass"):
        nodes = case["nodes"]
        mean = (1.0 + 0.625 * (seqs - 1)) / seqs  # lengths are spread over [1/4, 1] of the longest
        cached = seqs * nkv * (case["past"] * mean + nodes)
        mask = nodes * ((nodes + 31) // 32) * 4 if case["tree"] else 0
        if case["op"] == "tree":
            return {"bytes": cached * hd * 4 + seqs * nodes * nh * (hd * 4 + 4) + mask,
                    "flops": 4.0 * seqs * nodes * nh * hd * (case["past"] * mean + nodes)}
        acc = min(case["accepted"], nodes)
        return {"bytes": cached * (hd * 2 + 8) + seqs * acc * nh * (hd * 2 + 4) + seqs * nodes * 4 + mask,
                "flops": 2.0 * seqs * acc * nh * hd * (case["past"] * mean + nodes)}
    if case["op"] == "evict":
        mean = (1.0 + 0.625 * (seqs - 1)) / seqs
        return {"bytes": seqs * nkv * (case["rows"] * mean * 4 + case["keep"] * (hd * 8 + 12)), "flops": 0}
    mean = (case["accepted"] + (seqs - 1) * (case["accepted"] + 1) / 2.0) / seqs
    return {"bytes": seqs * nkv * mean * (hd * 8 + 8), "flops": 0}


# ---- the definitions in 64 bits, written apart from the plain forms: one sequence and kv head at a time ----


def _exact_attn(case, st):
    seqs, nodes, nh, hd = st["q"].shape
    nkv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(seqs, nodes, nh, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((seqs, nodes, nh), -math.inf, dtype=torch.float64, device="cuda")
    mass = st["mass"].double() if case["op"] == "mass" else None
    for s in range(seqs):
        past = int(st["n_past"][s])
        total = past + nodes
        see = torch.ones(nodes, total, dtype=torch.bool, device="cuda")
        for t in range(nodes):
            if st["mask"] is None:
                see[t, past + t + 1:] = False
            else:
                word = [w & 0xFFFFFFFF for w in st["mask"][t].tolist()]
                see[t, past:] = torch.tensor([(word[u >> 5] >> (u & 31)) & 1 for u in range(nodes)],
                                             dtype=torch.bool, device="cuda")
        for h in range(nkv):
            k, v = st["k"][s, h, :total].double(), st["v"][s, h, :total].double()
            if mass is not None:
                mass[s, h, past:total] = 0.0
            for g in range(group):
                head = h * group + g
                x = (st["q"][s, :, head].double() @ k.T) / math.sqrt(hd)
                x = torch.where(see, x, -math.inf)
                if mass is not None:
                    p = torch.exp(x - st["lse"][s, :, head].double()[:, None])
                    mass[s, h, :total] += st["weight"][s].double() @ p
                else:
                    lse[s, :, head] = torch.logsumexp(x, -1)
                    out[s, :, head] = torch.exp(x - lse[s, :, head][:, None]) @ v
    return {"mass": mass} if mass is not None else {"out": out, "lse": lse}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("tree", "mass"):
        return _exact_attn(case, st)
    return None  # whole numbers and copied values: nothing is computed
