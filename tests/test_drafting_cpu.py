"""CPU: refusals of the sampling, tree-attention, path and ring-copy entry points, all before any launch."""

import ctypes as C

import pytest
import torch

from utttcompanion_b200 import _lib, kv_cache, sampling, tree

BAD, SIZE = _lib.UTTT_ERR_INVALID, _lib.UTTT_ERR_UNSUPPORTED


def _buf():
    b = C.create_string_buffer(4096)
    return b, (C.addressof(b) + 255) // 256 * 256


def test_sample_rejects_bad_arguments_on_the_host():
    lib = _lib.load()
    keep, p = _buf()
    opt = _lib.Sampling(None, None, None, None, 1.0, 0, 1.0, 0.0)
    ok = dict(rows=2, V=16, x=p, f32=1, ld=16, lim=16, sf=0, opt=C.byref(opt), u=p, u_ld=1, ui=None, un=1, ids=p)

    def call(**kw):
        a = {**ok, **kw}
        return lib.uttt_sample(a["rows"], a["V"], a["x"], a["f32"], a["ld"], a["lim"], a["sf"], a["opt"], a["u"],
                               a["u_ld"], a["ui"], a["un"], a["ids"], None, None, None)
    for kw in (dict(rows=0), dict(V=6), dict(x=None), dict(opt=None), dict(u=None), dict(ids=None), dict(lim=2),
               dict(ld=15), dict(u_ld=-1), dict(ui=p, un=0)):
        assert call(**kw) == BAD, kw
    assert call(V=262145, ld=262145) == SIZE
    assert call(rows=65536) == SIZE


def test_tree_attention_rejects_bad_arguments_on_the_host():
    lib = _lib.load()
    keep, p = _buf()
    ok = dict(B=1, N=4, nh=4, nkv=2, hd=64, W=8, S=2, P=16, qld=512, par=p, n=None, old=256, qkv=p, pos=p)

    def call(**kw):
        a = {**ok, **kw}
        return lib.uttt_attn_tree(a["B"], a["N"], a["nh"], a["nkv"], a["hd"], a["W"], a["S"], a["P"], a["qkv"],
                                  a["qld"], a["par"], a["n"], a["pos"], p, p, p, p, p, p, p, p, a["old"], None)
    for kw in (dict(B=0), dict(N=0), dict(nkv=0), dict(W=0), dict(S=0), dict(P=0), dict(qkv=None), dict(par=None),
               dict(pos=None), dict(qld=511), dict(old=255)):
        assert call(**kw) == BAD, kw
    for kw in (dict(N=65), dict(hd=96, qld=4096, old=4096), dict(nh=18, qld=4096, old=4096), dict(nh=5, qld=4096, old=4096)):
        assert call(**kw) == SIZE, kw
    assert lib.uttt_tree_accept(0, 4, p, p, None, p, p, p, p, None) == BAD
    assert lib.uttt_tree_accept(1, 4, p, None, None, p, p, p, p, None) == BAD
    assert lib.uttt_tree_accept(1, 65, p, p, None, p, p, p, p, None) == SIZE


def test_ring_commit_rejects_bad_arguments_on_the_host():
    lib = _lib.load()
    keep, p = _buf()
    ok = dict(L=2, B=1, N=4, nkv=2, hd=64, W=8, S=3, t=p, ts=2 * 4 * 64, r=p, rs=3 * 2 * 8 * 64)

    def call(**kw):
        a = {**ok, **kw}
        return lib.uttt_kv_ring_commit(a["L"], a["B"], a["N"], a["nkv"], a["hd"], a["W"], a["S"], a["t"], p, a["ts"],
                                       a["r"], p, a["rs"], p, p, p, p, None)
    for kw in (dict(L=0), dict(B=0), dict(N=0), dict(W=0), dict(S=0), dict(t=None), dict(r=None), dict(ts=511),
               dict(rs=3071)):
        assert call(**kw) == BAD, kw
    for kw in (dict(N=65, ts=1 << 20), dict(hd=60), dict(t=p + 2), dict(r=p + 8), dict(ts=516)):
        assert call(**kw) == SIZE, kw


@pytest.mark.parametrize("src,dst,end", [
    ([0, 1], [2, 2], None),              # one destination twice
    ([0, 1], [1, 0], None),              # a swap
    ([0, 1, 2], [1, 2, 0], None),        # a longer cycle
    ([0, 3], [1, 2], None),              # a source out of range
    ([0], [-1], None),                   # a destination out of range
    ([0], [1], [-1]),                    # a negative position
    ([0, 1], [2, 0, 1], None),
])
def test_ring_fork_rejects_bad_pairs_before_it_copies(src, dst, end):
    lib = _lib.load()
    keep, p = _buf()
    n = max(len(src), len(dst))
    if len(src) == len(dst):
        arr = C.c_int * n
        st = lib.uttt_kv_ring_fork(2, n, 2, 64, 8, 3, p, p, 3 * 2 * 8 * 64, arr(*src), arr(*dst),
                                   None if end is None else arr(*end), None)
        assert st == BAD
    with pytest.raises(ValueError):
        kv_cache.ring_fork(torch.zeros(2, 2, 3, 2, 8, 64, dtype=torch.bfloat16), src, dst, end)


def test_ring_fork_rejects_bad_shapes_on_the_host():
    lib = _lib.load()
    keep, p = _buf()
    one = (C.c_int * 1)(0)
    two = (C.c_int * 1)(1)

    def call(L=2, n=1, nkv=2, hd=64, W=8, S=3, k=p, rs=3 * 2 * 8 * 64, src=one):
        return lib.uttt_kv_ring_fork(L, n, nkv, hd, W, S, k, p, rs, src, two, None, None)
    assert call(L=0) == BAD and call(n=0) == BAD and call(k=None) == BAD and call(src=None) == BAD
    assert call(rs=3071) == BAD
    assert call(hd=60) == SIZE and call(k=p + 2) == SIZE and call(L=20000) == SIZE


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 16)
    with pytest.raises(ValueError):
        sampling.sample(x, torch.zeros(2))
    i = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        tree.tree_accept(i, i, i)
    with pytest.raises(ValueError):
        kv_cache.ring_fork(torch.zeros(2, 1, 2, 1, 8, 32, dtype=torch.bfloat16), [0], [1])


@pytest.mark.parametrize("kw", [dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")),
                                dict(top_k=-1), dict(top_k=1.5), dict(top_p=0.0), dict(top_p=1.01),
                                dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.5)])
def test_settings_that_no_call_takes(kw):
    with pytest.raises(ValueError):
        sampling.check_settings(**kw)


def test_settings_at_their_limits():
    sampling.check_settings(0.0, 0, 1.0, 0.0)
    sampling.check_settings(2.0, 2 ** 31 - 1, 1e-6, 1.0)


@pytest.mark.parametrize("parents", [[], [0], [-1, 1], [-1, -1], [-1, 0, 3], [-1] + [0] * 64])
def test_trees_that_no_call_takes(parents):
    with pytest.raises(ValueError):
        tree.check_tree(parents)


def test_trees_at_their_limits():
    tree.check_tree([-1])
    tree.check_tree([-1] + [0] * 63)
    tree.check_tree([-1] + list(range(63)))


# ------------------------------------------------------------------------------------------------ host logic
def test_depths_and_pruning():
    parents = [-1, 0, 1, 1, 3, 0]
    depth = tree.depths(parents)
    assert depth == [0, 1, 2, 2, 3, 1]
    tokens, par, d = tree.prune([10, 11, 12, 13, 14, 15], parents, depth, 1)
    assert (tokens, par, d) == ([10, 11, 15], [-1, 0, 0], [0, 1, 1])
    assert tree.prune([10, 11], [-1, 0], [0, 1], 5) == ([10, 11], [-1, 0], [0, 1])
    assert tree.prune([10, 11, 12], [-1, 0, 0], [0, 1, 1], 0) == ([10], [-1], [0])


def test_prompt_lookup_drafts_what_followed_before():
    draft = tree.PromptLookup(match=2, depth=3, nodes=5)
    #      5 6 followed by 7 8 9 first and by 7 1 later: the later one first, merged
    ids = [5, 6, 7, 8, 9, 5, 6, 7, 1, 2, 5, 6]
    tokens, parents = draft(ids)
    assert tokens == [7, 1, 2, 8, 9] and parents == [0, 1, 2, 1, 4]
    tree.check_tree([-1, *parents])
    assert tree.PromptLookup(match=2, depth=3, nodes=2)(ids) == ([7, 1], [0, 1])
    assert draft([1, 2, 3]) == ([], [])
    assert draft([4, 4, 4, 4])[0] == [4, 4]            # what follows may run into the end
    assert draft([7]) == ([], [])
    with pytest.raises(ValueError):
        tree.PromptLookup(nodes=64)


def test_reply_uniforms_are_repeatable_and_in_range():
    a = sampling.reply_uniforms(1000, 5)
    assert torch.equal(a, sampling.reply_uniforms(1000, 5)) and not torch.equal(a, sampling.reply_uniforms(1000, 6))
    assert torch.equal(sampling.reply_uniforms(10, 5), a[:10])
    assert float(a.min()) >= 0.0 and float(a.max()) < 1.0


def test_sampling_rows_hold_each_rows_settings():
    rows = sampling.SamplingRows(torch.device("cpu"), 3, 4)
    rows.set(1, 0.7, 5, 0.9, 0.1, torch.tensor([0.25, 0.5]))
    f = rows.first(2)
    assert f["temperature"].tolist() == [0.0, pytest.approx(0.7)] and f["top_k"].tolist() == [0, 5]
    assert f["top_p"].tolist() == [1.0, pytest.approx(0.9)] and f["u"][1].tolist() == [0.25, 0.5, 0.0, 0.0]
    rows.set(1)
    assert rows.temperature.tolist() == [0.0, 0.0, 0.0] and rows.top_p.tolist() == [1.0, 1.0, 1.0]
    for bad in (dict(row=3), dict(row=0, top_p=0.0), dict(row=0, u=torch.zeros(5))):
        with pytest.raises(ValueError):
            rows.set(**bad)
