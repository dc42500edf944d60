"""Plain 64-bit implementations of sampling, tree attention, path acceptance and ring copies (numpy), row by row."""

import numpy as np


def sample_row(s, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, limit=None, stop_free=False):
    """(id, kept, prob) of one row of float32 logits ``s``; settings are taken as float32 values."""
    s = np.asarray(s, np.float32)
    lim = s.size if limit is None else min(limit, s.size)
    x = s[:lim].astype(np.float64)
    ids = np.array([i for i in range(lim) if not (i in (0, 1, 3) or (stop_free and i < 6))
                    and not np.isnan(x[i]) and x[i] != -np.inf], np.int64)
    if ids.size == 0:
        return (6 if stop_free else 2) % lim, 0, 0.0
    T = float(np.float32(temperature))
    order = ids[np.lexsort((ids, -x[ids]))]
    if not T > float(np.float32(1e-5)):
        return int(order[0]), 1, 1.0
    m = x[order[0]]

    def weight(i):
        with np.errstate(invalid="ignore"):
            return np.where(x[i] == m, 1.0, np.exp((x[i] - m) / T))
    if top_k > 0:
        order = order[:top_k]
    w = weight(order)
    p = float(np.float32(top_p))
    if p < 1.0:
        before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        order = order[before <= p * w.sum()]
        w = w[:order.size]
    order = order[w >= float(np.float32(min_p))]
    kept = np.sort(order)
    w = weight(kept)
    run = np.cumsum(w)
    pick = int(np.searchsorted(run, float(np.float32(u)) * run[-1], side="right"))
    return int(kept[pick]), int(kept.size), float(w[pick] / run[-1])


def bf16(x):
    """Round float values to the nearest BF16 value (ties to even), returned as float64."""
    b = np.asarray(x, np.float32).view(np.uint32)
    return ((b + 0x7fff + ((b >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32).astype(np.float64)


def rope(x, cos, sin):
    """apply_rope on BF16 values: tables, products and sum rounded to BF16 (FP32 arithmetic before each)."""
    half = x.shape[-1] // 2
    rot = np.concatenate((-x[..., half:], x[..., :half]), -1)
    f = np.float32
    a = bf16((x.astype(f) * bf16(cos).astype(f)))
    b = bf16((rot.astype(f) * bf16(sin).astype(f)))
    return bf16(a.astype(f) + b.astype(f))


def lines(parents, n):
    """Each node's path from its root, itself last; a parent that is not an earlier node makes a root."""
    out = []
    for i in range(n):
        out.append((out[parents[i]] if 0 <= parents[i] < i else []) + [i])
    return out


def tree_row(qkv, parents, n, pos, k_ring, v_ring, cos, sin, n_heads):
    """(out (n, n_heads, hd), keys (n_kv, n, hd), values) of one row: qkv (N, heads * hd), rings (n_kv, W, hd)."""
    n_kv, W, hd = k_ring.shape
    rep = n_heads // n_kv
    x = qkv.reshape(qkv.shape[0], -1, hd)[:n]
    path = lines(parents, n)
    at = [pos + len(p) - 1 for p in path]
    row = np.minimum(np.array(at, np.int64), cos.shape[0] - 1)
    c, s = cos[row][:, None], sin[row][:, None]
    q, k = rope(x[:, :n_heads], c, s), rope(x[:, n_heads:n_heads + n_kv], c, s)
    v = x[:, n_heads + n_kv:n_heads + 2 * n_kv]
    out = np.zeros((n, n_heads, hd))
    for i in range(n):
        old = [p % W for p in range(max(0, at[i] - W + 1), pos)]
        new = [j for j in path[i] if at[i] - at[j] < W]
        for h in range(n_heads):
            g = h // rep
            kk = np.concatenate((k_ring[g, old].reshape(-1, hd), k[new, g]))
            vv = np.concatenate((v_ring[g, old].reshape(-1, hd), v[new, g]))
            sc = kk @ q[i, h] / np.sqrt(hd)
            e = np.exp(sc - sc.max())
            out[i, h] = e @ vv / e.sum()
    return out, k.transpose(1, 0, 2), v.transpose(1, 0, 2)


def accept_row(tokens, parents, picks, n):
    """(path, next) of one tree."""
    if n < 1:
        return [], -1
    path = [0]
    while True:
        cur = path[-1]
        nxt = [j for j in range(cur + 1, n) if parents[j] == cur and tokens[j] == picks[cur]]
        if not nxt:
            return path, picks[cur]
        path.append(nxt[0])
