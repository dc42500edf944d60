"""GPU: tree attention, path acceptance and the ring copies against plain 64-bit forms.

Attention bound, |out - ref| <= 2^-8 |ref| + 2^-9 vmax with vmax the largest |v| a node sees: the output's rounding to
BF16 is at most 2^-8 |ref| (2^-9 for a value at the top of its binade, 2^-8 covers every value), and everything in
FP32 before it (scores of |s| <= 32 off by at most 2^-15, so weights by 2^-14 of themselves; sums of at most 8256 terms)
stays below 2^-9 vmax.  Keys, values, paths and copies must be equal.
"""

import numpy as np
import pytest
import torch

from drafting_refs import accept_row, tree_row
from utttcompanion_b200 import kv_cache, sampling, tree
from utttcompanion_b200.model import rope_tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tree(kind, N, rng):
    if kind == "chain":
        return [-1] + list(range(N - 1))
    if kind == "star":
        return [-1] + [0] * (N - 1)
    return [-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, N)]


def _case(B, N, nh, nkv, hd, W, pos, kind="random", nodes=None, seed=0, n_pos=None):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    bf = torch.bfloat16
    c = dict(parents=torch.tensor([_tree(kind, N, rng) for _ in range(B)], dtype=torch.int32, device=DEV),
             pos=torch.tensor(pos, dtype=torch.int32, device=DEV),
             slots=torch.tensor(rng.permutation(B + 2)[:B].tolist(), dtype=torch.int32, device=DEV),
             qkv=torch.randn(B * N, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(bf),
             k_ring=torch.randn(B + 2, nkv, W, hd, device=DEV, generator=g).to(bf),
             v_ring=torch.randn(B + 2, nkv, W, hd, device=DEV, generator=g).to(bf),
             n_nodes=None if nodes is None else torch.tensor(nodes, dtype=torch.int32, device=DEV))
    cos, sin = rope_tables(hd, n_pos or max(pos) + N + 1, 10000.0)
    c["rope_cos"], c["rope_sin"] = cos.to(DEV).contiguous(), sin.to(DEV).contiguous()
    return c


def _run(c, nh, **kw):
    return tree.tree_attention(c["qkv"], c["parents"], c["pos"], c["slots"], c["k_ring"], c["v_ring"], c["rope_cos"],
                               c["rope_sin"], nh, n_nodes=c["n_nodes"], **kw)


def _check(c, nh, out, kt, vt, rows=None):
    B, N = c["parents"].shape
    nkv, W, hd = c["k_ring"].shape[1:]
    np64 = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
    cos, sin = c["rope_cos"].cpu().numpy(), c["rope_sin"].cpu().numpy()
    got, kt, vt = np64(out).reshape(B, N, nh, hd), np64(kt), np64(vt)
    for b in range(B) if rows is None else rows:
        n = N if c["n_nodes"] is None else max(0, min(N, int(c["n_nodes"][b])))
        sl = int(c["slots"][b])
        x = np64(c["qkv"].reshape(B, N, -1)[b][:, :(nh + 2 * nkv) * hd])
        ref, k, v = tree_row(x, c["parents"][b].tolist(), n, int(c["pos"][b]), np64(c["k_ring"][sl]),
                             np64(c["v_ring"][sl]), cos, sin, nh)
        vmax = max(np.nanmax(np.abs(np.where(np.isfinite(y), y, 0)), initial=0) for y in (np64(c["v_ring"][sl]), v))
        np.testing.assert_array_equal(kt[b, :, :n], k)
        np.testing.assert_array_equal(vt[b, :, :n], v)
        err = np.abs(got[b, :n] - ref)
        assert np.isfinite(got[b, :n]).all()
        assert (err <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * vmax).all(), (b, float(err.max()))
        assert (got[b, n:] == 0).all() and (kt[b, :, n:] == 0).all() and (vt[b, :, n:] == 0).all()


@pytest.mark.parametrize("B,N,nh,nkv,hd,W,pos,kind,nodes", [
    (1, 1, 4, 4, 64, 128, [0], "chain", None),                    # a single token, an empty ring
    (1, 1, 20, 5, 128, 512, [700], "chain", None),                # the decode step's own case
    (2, 5, 20, 5, 128, 512, [300, 511], "random", None),
    (3, 16, 12, 4, 64, 512, [512, 513, 5000], "random", [16, 9, 1]),
    (2, 64, 12, 4, 64, 512, [40, 1000], "random", None),
    (2, 64, 4, 4, 32, 16, [3, 100], "chain", [64, 33]),           # paths longer than the window
    (3, 7, 2, 2, 32, 1, [0, 1, 9], "random", None),               # a window of one: each node sees itself
    (2, 13, 8, 1, 128, 1000, [999, 2500], "star", None),          # eight heads on one KV head
    (4, 33, 7, 1, 64, 77, [1, 76, 77, 78], "random", [33, 0, 32, 17]),   # a row without nodes
    (1, 31, 8, 1, 128, 8192, [100000], "random", None),
    (2, 64, 24, 3, 128, 130, [129, 131], "random", None),         # 512 queries a KV head
    (40, 3, 6, 2, 64, 65, list(range(50, 90)), "random", None),
    (1, 9, 15, 3, 64, 200, [63], "random", None),                 # five heads a KV head; tiles that end inside
    (1, 17, 18, 3, 32, 63, [62], "star", None),
    (1, 2, 3, 3, 128, 64, [64], "chain", None),
    # enough rows that nothing splits the keys; ragged trees and lengths
    (64, 16, 20, 5, 128, 512, [32 + 64 * i for i in range(64)], "random", [1 + i % 16 for i in range(64)]),
    (40, 64, 12, 4, 64, 300, [1 + 37 * i for i in range(40)], "random", [1 + (i * 7) % 64 for i in range(40)]),
    (80, 9, 8, 2, 64, 130, [100 + i for i in range(80)], "star", None),
])
def test_tree_attention(B, N, nh, nkv, hd, W, pos, kind, nodes):
    c = _case(B, N, nh, nkv, hd, W, pos, kind, nodes, seed=N * W + hd)
    rings = c["k_ring"].clone(), c["v_ring"].clone()
    _check(c, nh, *_run(c, nh), rows=None if B < 10 else (0, 2, 13, 14, 15, 31, B - 2, B - 1))
    assert torch.equal(rings[0], c["k_ring"]) and torch.equal(rings[1], c["v_ring"])


@pytest.mark.parametrize("hd,W,N", [(64, 96, 12), (128, 40, 33), (32, 256, 64)])
def test_what_a_node_does_not_see_does_not_reach_it(hd, W, N):
    """NaN and infinities in the ring's empty places, in places that only some nodes still see, in nodes off a
    node's path, and in the rows behind a row's last node."""
    nh, nkv = 4, 2
    nodes = [N, N - 3, N]
    c = _case(3, N, nh, nkv, hd, W, [W // 2, W + 7, W + 50], nodes=nodes, seed=3)
    clean = [t.clone() for t in _run(c, nh)]
    par = c["parents"].tolist()
    sl = c["slots"].tolist()
    for t in (c["k_ring"], c["v_ring"]):
        t[sl[0], :, W // 2:] = float("nan")                       # never written
        for b in (1, 2):
            t[sl[b], :, (int(c["pos"][b]) - W) % W] = float("inf")   # the oldest place: no node sees position pos - W
    x = c["qkv"].reshape(3, N, -1)
    x[1, N - 3:] = float("nan")                                   # behind the last node
    last = N - 1
    assert last not in par[2]
    x[2, last] = float("nan")                                     # a leaf: only itself sees it
    got = _run(c, nh)
    assert torch.equal(got[0].reshape(3, N, -1)[:2], clean[0].reshape(3, N, -1)[:2])
    assert torch.equal(got[0].reshape(3, N, -1)[2, :last], clean[0].reshape(3, N, -1)[2, :last])
    # a place that roots still see and deeper nodes do not
    c = _case(1, N, nh, nkv, hd, W, [W + 20], kind="chain", seed=4)
    clean = _run(c, nh)[0]
    edge = (W + 20 + 1 - W) % W                                   # position pos - W + 1: seen at depth 0 alone
    c["v_ring"][:, :, edge] = float("nan")
    c["k_ring"][:, :, (edge + 1) % W] = float("inf")              # seen at depths 0 and 1
    got = _run(c, nh)[0]
    assert torch.equal(got[2:], clean[2:]) and bool(torch.isnan(got[0]).all())


def test_bad_device_values_leave_rows_alone():
    c = _case(4, 6, 4, 2, 64, 32, [10, 20, 30, 40], seed=5)
    want = [t.clone() for t in _run(c, 4)]
    c["slots"][1] = 6
    c["pos"][2] = -1
    c["parents"][3] = torch.tensor([5, 0, 1, 3, 77, -9], dtype=torch.int32)   # 5, 3, 77, -9: roots
    got = _run(c, 4)
    for a, b in zip(got, want):
        a, b = a.reshape(4, -1), b.reshape(4, -1)
        assert torch.equal(a[0], b[0]) and (a[1:3] == 0).all()
    c["slots"][1], c["pos"][2] = int(c["slots"][0]), 30
    _check(c, 4, *_run(c, 4), rows=[0, 3])
    c["n_nodes"] = torch.tensor([-3, 99, 6, 2], dtype=torch.int32, device=DEV)
    _check(c, 4, *_run(c, 4))


def test_positions_past_the_table_take_its_last_row():
    c = _case(1, 4, 4, 2, 64, 32, [10], kind="chain", seed=6, n_pos=12)
    _check(c, 4, *_run(c, 4))


def test_strides_and_given_outputs():
    c = _case(2, 5, 4, 2, 64, 32, [10, 50], nodes=[5, 3], seed=7)
    want = _run(c, 4)
    big = torch.randn(10, 600, device=DEV).to(torch.bfloat16)
    big[:, 8:8 + 512] = c["qkv"]
    c["qkv"] = big[:, 8:520]
    wide = torch.full((10, 300), 7.0, dtype=torch.bfloat16, device=DEV)
    kt = torch.full((2, 2, 5, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    vt = kt.clone()
    _run(c, 4, out=wide[:, 5:261], k_tree=kt, v_tree=vt)
    live = torch.tensor([i < n for n in (5, 3) for i in range(5)], device=DEV)
    assert torch.equal(wide[:, 5:261][live], want[0][live]) and (wide[~live] == 7).all()
    assert (wide[:, :5] == 7).all() and (wide[:, 261:] == 7).all()
    assert torch.equal(kt[0], want[1][0]) and torch.equal(vt[1, :, :3], want[2][1, :, :3])
    assert (kt[1, :, 3:] == 7).all() and (vt[1, :, 3:] == 7).all()
    odd = torch.zeros(10, 601, device=DEV, dtype=torch.bfloat16)   # rows 1202 bytes apart, from byte 2 on
    odd[:, 1:513] = c["qkv"]
    c["qkv"] = odd[:, 1:513]
    assert torch.equal(_run(c, 4)[0], want[0])


def test_captured_and_replayed_with_other_rows():
    c = _case(3, 8, 12, 4, 64, 128, [100, 200, 300], nodes=[8, 4, 6], seed=8)
    d = _case(3, 8, 12, 4, 64, 128, [127, 90, 301], nodes=[2, 8, 0], seed=9)
    out = _run(c, 12)[0]
    kt = torch.zeros(3, 4, 8, 64, dtype=torch.bfloat16, device=DEV)
    vt = torch.zeros_like(kt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _run(c, 12, out=out, k_tree=kt, v_tree=vt)
    for name in c:
        if name.startswith("rope"):
            continue
        c[name].copy_(d[name])
    for t in (out, kt, vt):
        t.zero_()
    c["rope_cos"].copy_(c["rope_cos"])
    graph.replay()
    torch.cuda.synchronize()
    _check(c, 12, out, kt, vt)


def _wave(seed):
    """320 CTAs where the GPU holds 296: a full wave and a second launch for the rest of the rows."""
    return _case(64, 16, 20, 5, 128, 512, [32 + 64 * i for i in range(64)], "random", [1 + i % 16 for i in range(64)],
                 seed=seed)


def test_a_second_launch_is_captured_and_replayed():
    c, d = _wave(11), _wave(12)
    want = [[t.clone() for t in _run(x, 20)] for x in (c, d)]
    got = [torch.zeros_like(t) for t in want[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _run(c, 20, out=got[0], k_tree=got[1], v_tree=got[2])
    for x, w in ((c, want[0]), (d, want[1])):
        for name in c:
            c[name].copy_(x[name])
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_what_follows_waits_for_both_launches():
    """The next kernel starts early (its grid is launched while the last one runs): it must not read early."""
    cases = [_wave(13 + i) for i in range(3)]
    u = torch.zeros(1024, device=DEV)
    outs = [_run(c, 20)[0].clone() for c in cases]
    want = [sampling.sample(o, u, temperature=0.0).ids for o in outs]
    out = torch.zeros_like(outs[0])
    for i in range(30):
        out.zero_()
        _run(cases[i % 3], 20, out=out)
        ids = sampling.sample(out, u, temperature=0.0).ids
        assert torch.equal(ids, want[i % 3])


def test_two_streams_at_once():
    a, b = _wave(16), _case(5, 64, 12, 4, 64, 300, [10, 200, 299, 300, 9000], seed=17)
    g = torch.Generator(device=DEV).manual_seed(18)
    x = (torch.randn(40, 32000, device=DEV, generator=g) * 3).to(torch.bfloat16)
    u = torch.rand(40, device=DEV, generator=g)

    def both():
        return _run(a, 20) + _run(b, 12) + tuple(sampling.sample(x, u, top_p=0.9, temperature=0.8))
    want = [t.clone() for t in both()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s, r in zip(streams, got):
            with torch.cuda.stream(s):
                r.append(both())
    torch.cuda.synchronize()
    for r in got[0] + got[1]:
        assert all(torch.equal(p, q) for p, q in zip(r, want))


def test_attention_refusals():
    c = _case(2, 4, 4, 2, 64, 32, [1, 2], seed=10)
    for bad in (dict(qkv=c["qkv"].float()), dict(qkv=c["qkv"][:, :500]), dict(parents=c["parents"].long()),
                dict(pos=c["pos"][:1]), dict(slots=c["slots"].cpu()), dict(k_ring=c["k_ring"].float()),
                dict(v_ring=c["v_ring"][:, :1]), dict(k_ring=c["k_ring"].transpose(1, 2)),
                dict(rope_cos=c["rope_cos"].double()), dict(rope_sin=c["rope_sin"][:-1]),
                dict(n_nodes=torch.ones(3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            _run({**c, **bad}, 4)
    with pytest.raises(ValueError):
        _run(c, 3)
    with pytest.raises(ValueError):
        _run(c, 4, out=torch.zeros(8, 255, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError):
        _run(c, 4, k_tree=torch.zeros(2, 2, 5, 64, dtype=torch.bfloat16, device=DEV))
    c = _case(1, 2, 4, 2, 64, 32, [1], seed=10)
    far = torch.empty(2 ** 31 + 512, dtype=torch.bfloat16, device=DEV)      # rows 2^31 elements apart
    with pytest.raises(ValueError):
        _run({**c, "qkv": far.as_strided((2, 512), (2 ** 31, 1))}, 4)
    with pytest.raises(ValueError):
        _run(c, 4, out=far.as_strided((2, 256), (2 ** 31, 1)))


# ------------------------------------------------------------------------------------------------ accepted path
@pytest.mark.parametrize("N", [1, 2, 5, 31, 32, 33, 64])
def test_accepted_path(N):
    rng = np.random.default_rng(N)
    B = 37
    parents = np.array([_tree(("chain", "star", "random")[b % 3], N, rng) for b in range(B)])
    picks = rng.integers(0, 3, (B, N))
    tokens = np.where(rng.random((B, N)) < 0.7, picks[np.arange(B)[:, None], np.maximum(parents, 0)],
                      rng.integers(0, 3, (B, N)))
    nodes = rng.integers(-1, N + 2, B)
    parents[B - 1] = rng.integers(-3, 70, N)                      # not a tree: never out of range, always ends
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    for n in (None, nodes):
        path, n_path, nxt = tree.tree_accept(dev(tokens), dev(parents), dev(picks), None if n is None else dev(n))
        for b in range(B):
            m = N if n is None else max(0, min(N, int(n[b])))
            want, follow = accept_row(tokens[b], parents[b], picks[b], m)
            assert path[b].tolist() == want + [-1] * (N - len(want))
            assert (int(n_path[b]), int(nxt[b])) == (len(want), follow)


# ------------------------------------------------------------------------------------------------ ring copies
def _rings(L, S, nkv, W, hd, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(2, L, S, nkv, W, hd, device=DEV, generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("L,B,N,nkv,hd,W", [(3, 4, 6, 2, 64, 32), (1, 1, 1, 1, 32, 1), (2, 3, 64, 3, 128, 48),
                                            (34, 2, 9, 5, 128, 20), (2, 5, 20, 1, 8, 33)])
def test_commit(L, B, N, nkv, hd, W):
    rng = np.random.default_rng(N + W)
    rings = _rings(L, B + 2, nkv, W, hd)
    kv = _rings(L, B, nkv, N, hd, 1)
    pos = rng.integers(0, 3 * W, B)
    slots = rng.permutation(B + 2)[:B]
    lens = rng.integers(0, N + 1, B)
    lens[0] = N
    path = np.array([np.sort(rng.permutation(N)) for _ in range(B)])
    path[:, 0] = 0
    want = rings.clone()
    for b in range(B):
        for t in range(lens[b]):                                   # in order: later positions replace earlier ones
            want[:, :, slots[b], :, (pos[b] + t) % W] = kv[:, :, b, :, path[b, t]]
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    kv_cache.ring_commit(rings, kv, dev(pos), dev(slots), dev(path), dev(lens))
    assert torch.equal(rings, want)


def test_commit_leaves_bad_rows_out():
    rings = _rings(2, 4, 2, 16, 64)
    kv = _rings(2, 4, 2, 4, 64, 1)
    want = rings.clone()
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    path = dev([[0, 1, 2, 3], [0, 1, 2, 3], [0, 9, -1, 3], [0, 1, 2, 3]])
    kv_cache.ring_commit(rings, kv, dev([0, -1, 2147483647, 3]), dev([4, 1, 2, 3]), path, dev([4, 4, 4, -2]))
    for t, n in ((0, 0), (3, 3)):                                  # nodes 9 and -1 do not exist
        want[:, :, 2, :, (2147483647 + t) % 16] = kv[:, :, 2, :, n]
    assert torch.equal(rings, want)


@pytest.mark.parametrize("src,dst,end", [
    ([0], [1], None), ([0, 0, 0], [1, 2, 3], [5, 16, 40]), ([2, 4], [0, 1], [0, 7]),
    ([5, 3, 1], [3, 1, 0], None),                                  # a chain: slots move down
    ([1, 3, 5], [0, 1, 3], [16, 3, 9]),                            # compaction
    ([2, 2, 4], [2, 3, 2], None),                                  # one copy to itself refused below; here none
])
@pytest.mark.parametrize("L,nkv,W,hd", [(3, 2, 16, 64), (1, 1, 1, 8), (2, 3, 37, 128)])
def test_fork(src, dst, end, L, nkv, W, hd):
    rings = _rings(L, 6, nkv, W, hd)
    before = rings.clone()
    if len(set(dst)) < len(dst):
        with pytest.raises(ValueError):
            kv_cache.ring_fork(rings, src, dst, end)
        assert torch.equal(rings, before)
        return
    want = before.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        n = W if end is None else min(W, end[i])
        want[:, :, d, :, :n] = before[:, :, s, :, :n]
    kv_cache.ring_fork(rings, src, dst, end)
    assert torch.equal(rings, want)


def test_fork_many_pairs_and_refusals():
    rings = _rings(2, 600, 1, 4, 16)
    before = rings.clone()
    kv_cache.ring_fork(rings, [i % 7 for i in range(300)], list(range(300, 600)))
    assert torch.equal(rings[:, :, 300:], before[:, :, torch.arange(300, device=DEV) % 7])
    assert torch.equal(rings[:, :, :300], before[:, :, :300])
    kv_cache.ring_fork(rings, [], [])
    kv_cache.ring_fork(rings, [3], [3])
    now = rings.clone()
    for src, dst in (([0, 1], [1, 0]), ([0], [600]), ([-1], [2]), ([0, 1], [5, 5]), ([2 ** 32], [1]),
                     ([0], [2 ** 32 + 1])):
        with pytest.raises(ValueError):
            kv_cache.ring_fork(rings, src, dst)
    with pytest.raises(ValueError):
        kv_cache.ring_fork(rings[:, :, ::2], [0], [1])
    with pytest.raises(ValueError):
        kv_cache.ring_fork(rings, [0], [1], [-2 ** 33])
    assert torch.equal(rings, now)
