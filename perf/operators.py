"""The operators of sampled and drafted generation, case by case: their inputs, their plain forms and their calls.

Four operators of the serving path, over the packed rows and the per-persona KV rings of ``UtttB200``:

* ``sample``: one token per row of logits by temperature, top-k, top-p and min-p from one given uniform
  number a row (``sampling.sample``);
* ``tree``: attention of a tree of drafted tokens over a persona's KV ring (``tree.tree_attention``);
* ``commit``: the accepted path of a drafted tree, and its keys and values copied into the rings of all layers,
  (2, layers, slots, KV heads, window, head dim) (``tree.tree_accept``, ``kv_cache.ring_commit``);
* ``fork``: the rings of a persona copied to other slots, all layers at once (``kv_cache.ring_fork``).

``own`` chooses between the plain forms (elementary torch operations) and the framework's calls.
"""

import math

import torch

own = False

# heads, KV heads and head dim of the framework's model configurations
TINY = dict(n_heads=4, n_kv=4, hd=64)
SMALL = dict(n_heads=12, n_kv=4, hd=64)
LARGE = dict(n_heads=20, n_kv=5, hd=128)


def listed():
    return [
        # one persona's next token: latency counts
        dict(name="sample one row", op="sample", rows=1, V=32000, limit=21478, f32=True, mix=False, temperature=0.7,
             top_k=0, top_p=0.9, min_p=0.0),
        # a packed decode batch whose turns ask for different settings, greedy ones among them
        dict(name="sample packed turns", op="sample", rows=64, V=32000, limit=32000, f32=True, mix=True,
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # every node of the drafted trees of a batch; odd sizes, BF16 rows
        dict(name="sample odd rows", op="sample", rows=333, V=8003, limit=7999, f32=False, mix=False,
             temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
        # a wide vocabulary and a large batch
        dict(name="sample wide", op="sample", rows=256, V=131072, limit=131072, f32=False, mix=False,
             temperature=1.0, top_k=0, top_p=0.95, min_p=0.0),
        # one persona, a short draft, a ring that is not full yet
        dict(name="tree one row", op="tree", B=1, N=5, W=512, lo=300, hi=300, ragged=False, **LARGE),
        # packed personas with ragged trees and lengths
        dict(name="tree packed", op="tree", B=64, N=16, W=512, lo=32, hi=4096, ragged=True, **LARGE),
        # the widest trees
        dict(name="tree wide", op="tree", B=33, N=64, W=512, lo=64, hi=1024, ragged=True, **SMALL),
        # a long window, one KV head for all query heads
        dict(name="tree long", op="tree", B=8, N=31, W=8192, lo=9000, hi=100000, ragged=False, n_heads=8, n_kv=1,
             hd=128),
        # after one persona's step
        dict(name="commit one row", op="commit", B=1, N=5, W=512, L=12, slots=4, lo=300, hi=300, ragged=False,
             n_kv=4, hd=64),
        # after a packed step of the largest model
        dict(name="commit packed", op="commit", B=16, N=32, W=512, L=34, slots=17, lo=32, hi=4096, ragged=True,
             n_kv=5, hd=128),
        # one prompt, several replies
        dict(name="fork short", op="fork", pairs=3, fan=3, W=512, L=12, slots=5, lo=77, hi=77, n_kv=4, hd=64),
        # a batch of prompts, two replies each
        dict(name="fork full rings", op="fork", pairs=16, fan=1, W=512, L=34, slots=33, lo=600, hi=4096, n_kv=5,
             hd=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "tree", "tree", "commit", "fork"])
    if op == "sample":
        V = _log(rng, 500, 131072)
        rows = max(1, min(_log(rng, 1, 512), (128 << 17) // V))
        return dict(op=op, rows=rows, V=V, limit=V - rng.choice([0, 0, 1, V // 3]), f32=rng.random() < 0.5,
                    mix=rng.random() < 0.4, temperature=rng.uniform(0.3, 1.6),
                    top_k=rng.choice([0, 0, 1, _log(rng, 2, 1000)]),
                    top_p=rng.choice([1.0, rng.uniform(0.3, 0.99)]), min_p=rng.choice([0.0, 0.0, rng.uniform(0.001, 0.3)]))
    if op == "tree":
        n_kv, rep, hd = rng.choice([1, 2, 4, 5]), rng.randint(1, 8), rng.choice([32, 64, 128])
        W = _log(rng, 16, 8192)
        B = max(1, min(_log(rng, 1, 64), 64 * 5 * 512 // (n_kv * W)))
        N = _log(rng, 1, 64)
        while B * N * W * rep * n_kv * hd > 8 * 31 * 8192 * 8 * 128:
            B, N = (B // 2, N) if B > 1 else (B, N // 2)
        lo = _log(rng, 1, 2 * W)
        return dict(op=op, B=B, N=N, W=W, lo=lo, hi=lo + rng.choice([0, _log(rng, 1, 4 * W)]),
                    ragged=rng.random() < 0.5, n_heads=n_kv * rep, n_kv=n_kv, hd=hd)
    n_kv, hd, L = rng.choice([1, 2, 4, 5]), rng.choice([32, 64, 128]), rng.randint(1, 34)
    W = _log(rng, 64, 1024)
    lo = _log(rng, 1, 2 * W)
    rest = dict(W=W, L=L, lo=lo, hi=lo + rng.choice([0, W]), n_kv=n_kv, hd=hd)
    most = max(1, (600 << 20) // (4 * L * n_kv * hd * W))
    if op == "commit":
        B = max(1, min(_log(rng, 1, 32), most - 1))
        return dict(op=op, B=B, N=_log(rng, 1, 64), slots=B + 1, ragged=rng.random() < 0.5, **rest)
    fan = rng.choice([1, 1, 2, 3])
    pairs = fan * max(1, min(_log(rng, 1, 16), most // (2 * fan)))
    return dict(op=op, pairs=pairs, fan=fan, slots=pairs + pairs // fan + 1, **rest)


# ------------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _nodes(c):
    return _spread(1, c["N"], c["B"]) if c["ragged"] and c["B"] > 1 else [c["N"]] * c["B"]


def _shuffled(values, g):
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t[torch.randperm(len(values), device="cuda", generator=g)].contiguous()


def _trees(c, g):
    """(parents, nodes per row): node 0 is the root, a node's parent is one of the few nodes before it."""
    B, N = c["B"], c["N"]
    i = torch.arange(N, device="cuda")
    back = 1 + (torch.rand(B, N, device="cuda", generator=g) * 4).long()
    parents = (i - back).clamp_min(0)
    parents[:, 0] = -1
    return parents.to(torch.int32).contiguous(), _shuffled(_nodes(c), g)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(torch.bfloat16)


def _bf16(g, *shape):
    return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(c)
    if c["op"] == "sample":
        rows, V = c["rows"], c["V"]
        # logits as a language model's: a broad bulk, a few likely ids, BF16 values as the LM head writes them
        x = torch.randn(rows, V, device="cuda", generator=g) * 2.0
        hot = torch.randint(0, V, (rows, 40), device="cuda", generator=g)
        x.scatter_add_(1, hot, torch.rand(rows, 40, device="cuda", generator=g) * 8.0)
        x = x.to(torch.bfloat16)
        st["logits"] = x.float() if c["f32"] else x
        st["u"] = torch.rand(rows, device="cuda", generator=g)
        if c["mix"]:
            r = torch.rand(4, rows, device="cuda", generator=g)
            st["temperature"] = torch.where(r[0] < 0.2, 0.0, 0.4 + r[0])
            st["top_k"] = torch.where(r[1] < 0.5, 0.0, r[1] * 200).to(torch.int32)
            st["top_p"] = torch.where(r[2] < 0.3, 1.0, 0.3 + 0.69 * r[2])
            st["min_p"] = torch.where(r[3] < 0.6, 0.0, 0.1 * r[3])
        return st
    W, n_kv, hd = c["W"], c["n_kv"], c["hd"]
    if c["op"] == "tree":
        B, N, nh = c["B"], c["N"], c["n_heads"]
        st["parents"], st["n_nodes"] = _trees(c, g)
        st["pos"] = _shuffled(_spread(c["lo"], c["hi"], B), g)
        st["slots"] = _shuffled(list(range(B + 1))[:B], g)
        st["qkv"] = _randn(g, B * N, (nh + 2 * n_kv) * hd)
        st["k_ring"], st["v_ring"] = _bf16(g, B + 1, n_kv, W, hd), _bf16(g, B + 1, n_kv, W, hd)
        freq = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd))
        a = torch.outer(torch.arange(c["hi"] + N + 1, dtype=torch.float64, device="cuda"), freq)
        a = torch.cat((a, a), dim=-1)
        st["rope_cos"], st["rope_sin"] = a.cos().float().contiguous(), a.sin().float().contiguous()
        # rows behind a row's last node are left as they were
        st["out"] = torch.zeros(B * N, nh * hd, dtype=torch.bfloat16, device="cuda")
        st["k_tree"] = torch.zeros(B, n_kv, N, hd, dtype=torch.bfloat16, device="cuda")
        st["v_tree"] = torch.zeros_like(st["k_tree"])
        return st
    L, slots = c["L"], c["slots"]
    st["rings"] = _bf16(g, 2, L, slots, n_kv, W, hd)
    if c["op"] == "commit":
        B, N = c["B"], c["N"]
        st["parents"], st["n_nodes"] = _trees(c, g)
        st["pos"] = _shuffled(_spread(c["lo"], c["hi"], B), g)
        st["slots"] = _shuffled(list(range(slots))[:B], g)
        st["picks"] = torch.randint(0, 32000, (B, N), device="cuda", generator=g, dtype=torch.int32)
        # most drafted tokens are what the model picks after their parents
        hit = torch.gather(st["picks"], 1, st["parents"].long().clamp_min(0))
        other = torch.randint(0, 32000, (B, N), device="cuda", generator=g, dtype=torch.int32)
        st["tokens"] = torch.where(torch.rand(B, N, device="cuda", generator=g) < 0.85, hit, other).contiguous()
        st["tree"] = _bf16(g, 2, L, B, n_kv, N, hd)
        return st
    order = torch.randperm(slots, device="cuda", generator=g).tolist()
    n_src = c["pairs"] // c["fan"]
    st["src"] = [order[i // c["fan"]] for i in range(c["pairs"])]
    st["dst"] = [order[n_src + i] for i in range(c["pairs"])]
    st["end"] = _spread(c["lo"], c["hi"], c["pairs"])
    for name in ("src", "dst", "end"):
        st[name + "_t"] = torch.tensor(st[name], device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _column(st, name, dtype):
    v = st[name]
    t = v if isinstance(v, torch.Tensor) else torch.full((st["rows"],), v, device="cuda")
    return t.to(torch.float32).to(dtype)[:, None]       # the values that a 32-bit argument holds


def _plain_sample(st):
    """Order a row's candidates by value (the lowest id first among equals); top-k keeps the first k, top-p those
    whose mass before them is at most top_p of the mass that top-k left, min-p those at least min_p as likely as
    the first.  The pick is the lowest id whose kept mass up to and with it exceeds u of the kept mass."""
    x = st["logits"].float()
    rows, V = x.shape
    i = torch.arange(V, device=x.device)
    out = (i == 0) | (i == 1) | (i == 3) | (i >= st["limit"])
    s = torch.where(out[None, :] | x.isnan(), -math.inf, x)
    T, k = _column(st, "temperature", torch.float64), _column(st, "top_k", torch.int64)
    p, mp = _column(st, "top_p", torch.float64), _column(st, "min_p", torch.float64)
    greedy = T <= 1e-5
    T, k = torch.where(greedy, 1.0, T), torch.where(greedy, 1, k)
    val, order = torch.sort(s, dim=1, descending=True, stable=True)
    val = val.double()
    w = torch.where(val == -math.inf, 0.0, torch.exp((val - val[:, :1]) / T))      # 64 bits: borders of long sums
    keep = (val > -math.inf) & ((k <= 0) | (i[None, :] < k))
    m = torch.where(keep, w, 0.0)
    before = torch.cumsum(m, dim=1) - m
    keep = keep & ((p >= 1.0) | (before <= p * m.sum(1, keepdim=True))) & (w >= mp)
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    weight = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))
    run_up = torch.cumsum(weight, dim=1)
    total = weight.sum(1, keepdim=True)
    ids = (run_up > st["u"].double()[:, None] * total).to(torch.uint8).argmax(1, keepdim=True)
    prob = weight.gather(1, ids) / total
    return {"ids": ids[:, 0].to(torch.int32), "kept": kept.sum(1).to(torch.int32), "prob": prob[:, 0].float()}


def _closure(parents, n):
    """(B, N, N): whether node j is node i or one of its ancestors."""
    N = parents.shape[1]
    step = torch.eye(N, device="cuda", dtype=torch.float64) + (
        parents.long()[:, :, None] == torch.arange(N, device="cuda")[None, None, :])
    return torch.linalg.matrix_power(step, N) > 0.5


def _turned(x, cos, sin):
    """The rotation as the framework's rings hold it: tables, products and sum each rounded to BF16."""
    half = x.shape[-1] // 2
    other = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    a = (x.float() * cos.to(torch.bfloat16).float()).to(torch.bfloat16).float()
    b = (other.float() * sin.to(torch.bfloat16).float()).to(torch.bfloat16).float()
    return (a + b).to(torch.bfloat16)


def _plain_tree(st):
    B, N, W, nh, n_kv, hd = (st[k] for k in ("B", "N", "W", "n_heads", "n_kv", "hd"))
    pos, n = st["pos"].long(), st["n_nodes"].long()
    above = _closure(st["parents"], n)
    live = torch.arange(N, device="cuda")[None, :] < n[:, None]
    depth = above.sum(2) - 1
    at = pos[:, None] + depth                                                   # (B, N)
    cos, sin = st["rope_cos"][at][:, :, None, :], st["rope_sin"][at][:, :, None, :]
    q, k, v = st["qkv"].reshape(B, N, nh + 2 * n_kv, hd).split((nh, n_kv, n_kv), dim=2)
    q, k = _turned(q, cos, sin), _turned(k, cos, sin)
    rows = st["slots"].long()
    keys = torch.cat((st["k_ring"][rows], k.transpose(1, 2)), dim=2).float()     # (B, n_kv, W + N, hd)
    vals = torch.cat((st["v_ring"][rows], v.transpose(1, 2)), dim=2).float()
    j = torch.arange(W, device="cuda")[None, :]
    held = pos[:, None] - 1 - (pos[:, None] - 1 - j) % W                        # the position in each ring place
    see = torch.cat(((held >= 0)[:, None, :] & (held[:, None, :] > at[:, :, None] - W),
                     above & (depth[:, :, None] - depth[:, None, :] < W)), dim=2)          # (B, N, W + N)
    qh = q.float().reshape(B, N, n_kv, nh // n_kv, hd).permute(0, 2, 3, 1, 4)
    s = torch.matmul(qh, keys[:, :, None].transpose(-1, -2)) / math.sqrt(hd)    # (B, n_kv, rep, N, W + N)
    s = s.masked_fill(~see[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(e, vals[:, :, None]) / e.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, nh * hd).to(torch.bfloat16)
    zero = torch.zeros((), dtype=torch.bfloat16, device="cuda")
    return {"out": torch.where(live[:, :, None], o, zero).reshape(B * N, nh * hd),
            "k_tree": torch.where(live[:, :, None, None], k, zero).transpose(1, 2).contiguous(),
            "v_tree": torch.where(live[:, :, None, None], v, zero).transpose(1, 2).contiguous()}


def _plain_commit(st):
    """The accepted path: from the root on to the lowest child that holds what was picked after its parent."""
    B, N, W = st["B"], st["N"], st["W"]
    parents, n = st["parents"].long(), st["n_nodes"].long()
    i = torch.arange(N, device="cuda")
    live = i[None, :] < n[:, None]
    up = parents.clamp_min(0)
    match = live & (parents >= 0) & (st["tokens"] == torch.gather(st["picks"], 1, up))
    same = (parents[:, :, None] == parents[:, None, :]) & match[:, None, :] & (i[None, None, :] < i[None, :, None])
    first = match & ~same.any(2)                                 # the lowest matching child of its parent
    above = _closure(st["parents"], n)
    ok = first | (i == 0)[None, :]
    taken = live & (above <= ok[:, None, :]).all(2) & above[:, :, 0]
    depth = above.sum(2) - 1
    n_path = taken.sum(1)
    spare = torch.full((B, N + 1), -1, dtype=torch.long, device="cuda")
    path = spare.scatter(1, torch.where(taken, depth, N), i[None, :].expand(B, N))[:, :N]
    path = torch.where(i[None, :] < n_path[:, None], path, -1)
    last = torch.gather(path, 1, (n_path - 1).clamp_min(0)[:, None])
    following = torch.gather(st["picks"], 1, last.clamp_min(0))[:, 0]
    slots = st["slots"].long()[:, None]
    place = (st["pos"].long()[:, None] + i[None, :]) % W
    # only the last W positions of a path stay in a ring
    put = (i[None, :] < n_path[:, None]) & (i[None, :] >= n_path[:, None] - W)
    rows = torch.arange(B, device="cuda")[:, None]
    new = st["tree"][:, :, rows, :, path.clamp_min(0)]           # (B, N, 2, L, n_kv, hd)
    old = st["rings"][:, :, slots, :, place]
    st["rings"][:, :, slots, :, place] = torch.where(put[:, :, None, None, None, None], new, old)
    return {"path": path.to(torch.int32), "n_path": n_path.to(torch.int32), "next": following, "rings": st["rings"]}


def _plain_fork(st):
    there = torch.arange(st["W"], device="cuda")[None, :] < st["end_t"][:, None]
    new, old = st["rings"][:, :, st["src_t"]], st["rings"][:, :, st["dst_t"]]
    st["rings"][:, :, st["dst_t"]] = torch.where(there[None, None, :, None, :, None], new, old)
    return st["rings"]


def run(state):
    st = state
    if own:
        from utttcompanion_b200 import kv_cache, sampling, tree
        if st["op"] == "sample":
            return sampling.sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                   top_p=st["top_p"], min_p=st["min_p"], active_limit=st["limit"])._asdict()
        if st["op"] == "tree":
            tree.tree_attention(st["qkv"], st["parents"], st["pos"], st["slots"], st["k_ring"], st["v_ring"],
                                st["rope_cos"], st["rope_sin"], st["n_heads"], n_nodes=st["n_nodes"], out=st["out"],
                                k_tree=st["k_tree"], v_tree=st["v_tree"])
            return {"out": st["out"], "k_tree": st["k_tree"], "v_tree": st["v_tree"]}
        if st["op"] == "commit":
            path, n_path, following = tree.tree_accept(st["tokens"], st["parents"], st["picks"], st["n_nodes"])
            kv_cache.ring_commit(st["rings"], st["tree"], st["pos"], st["slots"], path, n_path)
            return {"path": path, "n_path": n_path, "next": following, "rings": st["rings"]}
        kv_cache.ring_fork(st["rings"], st["src"], st["dst"], st["end"])
        return st["rings"]
    if st["op"] == "sample":
        return _plain_sample(st)
    if st["op"] == "tree":
        return _plain_tree(st)
    if st["op"] == "commit":
        return _plain_commit(st)
    return _plain_fork(st)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    c = case
    if c["op"] == "sample":
        n = c["rows"] * min(c["limit"], c["V"])
        return {"bytes": n * (4 if c["f32"] else 2) + c["rows"] * (4 + 12 + (16 if c["mix"] else 0)), "flops": 4 * n}
    n_kv, hd, W = c["n_kv"], c["hd"], c["W"]
    if c["op"] == "tree":
        nh, nodes, pos = c["n_heads"], _nodes(c), _spread(c["lo"], c["hi"], c["B"])
        ring, new = sum(min(p, W) for p in pos), sum(nodes)
        per_row = sum(nodes) / len(nodes)
        return {"bytes": 4 * n_kv * hd * ring + new * (2 * (nh + 2 * n_kv) * hd + 2 * nh * hd + 4 * n_kv * hd + 4),
                "flops": 4 * nh * hd * per_row * (ring + new / 2)}
    if c["op"] == "commit":
        # the accepted paths' lengths depend on the draft: a third of the nodes stands for them
        nodes = sum(max(1, n // 3) for n in _nodes(c))
        return {"bytes": 2 * 4 * c["L"] * n_kv * hd * nodes + 16 * c["B"] * c["N"], "flops": 0}
    copied = sum(min(e, W) for e in _spread(c["lo"], c["hi"], c["pairs"]))
    read = copied / c["fan"]
    return {"bytes": 4 * c["L"] * n_kv * hd * (copied + read), "flops": 0}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions, in 64 bits and row by row."""
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] == "tree":
        return _exact_tree(st)
    if case["op"] == "commit":
        return _exact_commit(st)
    rings = st["rings"].clone()
    for s, d, e in zip(st["src"], st["dst"], st["end"]):
        n = min(e, st["W"])
        rings[:, :, d, :, :n] = st["rings"][:, :, s, :, :n]
    return rings


def _exact_sample(st):
    import numpy as np
    logits = st["logits"].float().cpu().numpy().astype(np.float64)
    u = st["u"].cpu().numpy().astype(np.float64)

    def given(name, r):
        v = st[name]
        return float(v[r]) if isinstance(v, torch.Tensor) else float(np.float32(v))
    prob = np.zeros(st["rows"])
    for r in range(st["rows"]):
        x = logits[r, :st["limit"]].copy()
        x[[0, 1, 3]] = -np.inf
        T, k = given("temperature", r), int(given("top_k", r))
        if T <= 1e-5:
            prob[r] = 1.0
            continue
        order = np.lexsort((np.arange(x.size), -x))
        order = order[np.isfinite(x[order])]
        if k > 0:
            order = order[:k]
        w = np.exp((x[order] - x[order[0]]) / T)
        if given("top_p", r) < 1.0:
            lower = np.concatenate(([0.0], np.cumsum(w)[:-1]))
            order = order[lower <= given("top_p", r) * w.sum()]
            w = w[:order.size]
        order = order[w >= given("min_p", r)]
        ids = np.sort(order)
        w = np.exp((x[ids] - x.max()) / T)
        c = np.cumsum(w)
        pick = int(np.searchsorted(c, u[r] * c[-1], side="right"))
        prob[r] = w[pick] / c[-1]
    return {"ids": None, "kept": None, "prob": torch.from_numpy(prob)}


def _exact_tree(st):
    B, N, W, nh, n_kv, hd = (st[k] for k in ("B", "N", "W", "n_heads", "n_kv", "hd"))
    rep, half = nh // n_kv, hd // 2
    out = torch.zeros(B, N, nh, hd, dtype=torch.float64, device="cuda")
    kt = torch.zeros(B, n_kv, N, hd, dtype=torch.float64, device="cuda")
    vt = torch.zeros_like(kt)
    parents, nodes, pos, slots = (st[k].tolist() for k in ("parents", "n_nodes", "pos", "slots"))
    x = st["qkv"].reshape(B, N, nh + 2 * n_kv, hd)
    for b in range(B):
        n, p0 = nodes[b], pos[b]
        lines = []
        for i in range(n):
            lines.append(([] if parents[b][i] < 0 else lines[parents[b][i]]) + [i])
        at = torch.tensor([p0 + len(line) - 1 for line in lines], device="cuda")
        cos, sin = st["rope_cos"][at].bfloat16()[:, None], st["rope_sin"][at].bfloat16()[:, None]
        y = x[b, :n, :nh + n_kv]
        # the rotation is defined with BF16 products and sum: the rings hold such keys
        lo = y[..., :half] * cos[..., :half] - y[..., half:] * sin[..., :half]
        hi = y[..., half:] * cos[..., half:] + y[..., :half] * sin[..., half:]
        y = torch.cat((lo, hi), -1).double()
        v = x[b, :n, nh + n_kv:].double().transpose(0, 1)
        kt[b, :, :n], vt[b, :, :n] = y[:, nh:].transpose(0, 1), v
        first = max(0, p0 - W)
        old = torch.arange(first, p0, device="cuda")
        keys = torch.cat((st["k_ring"][slots[b]][:, old % W].double(), kt[b, :, :n]), 1)
        vals = torch.cat((st["v_ring"][slots[b]][:, old % W].double(), v), 1)
        hidden = torch.ones(n, old.numel() + n, dtype=torch.bool, device="cuda")
        hidden[:, :old.numel()] = old[None, :] <= (at[:, None] - W)
        line = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            line[i, [j for j in lines[i] if len(lines[i]) - len(lines[j]) < W]] = True
        hidden[:, old.numel():] = ~line.to("cuda")
        for h in range(nh):
            s = (y[:, h] @ keys[h // rep].T) / hd ** 0.5
            out[b, :n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vals[h // rep]
    return {"out": out.reshape(B * N, nh * hd), "k_tree": kt, "v_tree": vt}


def _exact_commit(st):
    rings = st["rings"].clone()
    tokens, parents, picks = st["tokens"].tolist(), st["parents"].tolist(), st["picks"].tolist()
    nodes, pos, slots = (st[k].tolist() for k in ("n_nodes", "pos", "slots"))
    for b in range(st["B"]):
        at, step = 0, 0
        while at is not None:
            rings[:, :, slots[b], :, (pos[b] + step) % st["W"]] = st["tree"][:, :, b, :, at]
            step += 1
            at = next((j for j in range(at + 1, nodes[b])
                       if parents[b][j] == at and tokens[b][j] == picks[b][at]), None)
    return {"path": None, "n_path": None, "next": None, "rings": rings}
