"""GPU: a device wait that expires in a tree's attention reaches the caller, and nothing of that step is committed.

The wait is made to run out by a short limit: a CTA that has more than two tiles to load gives up after two looks for a
free slot, ends the copies it has under way and returns.  No wait is left out and no access leaves its buffers.
"""

import pytest
import torch

from utttcompanion_b200 import _lib, tree
from utttcompanion_b200.model import UtttB200, rope_tables
from utttcompanion_b200.workloads import ModelConfig, reference_init_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(B, N, nh, nkv, hd, W, pos):
    g = torch.Generator(device=DEV).manual_seed(B + W)
    c = dict(B=B, N=N, nh=nh, nkv=nkv, hd=hd, W=W,
             parents=torch.tensor([[-1] + [i // 2 for i in range(N - 1)]] * B, dtype=torch.int32, device=DEV),
             pos=torch.full((B,), pos, dtype=torch.int32, device=DEV),
             slots=torch.arange(B, dtype=torch.int32, device=DEV),
             qkv=torch.randn(B * N, (nh + 2 * nkv) * hd, device=DEV, generator=g).to(torch.bfloat16))
    c["k_ring"], c["v_ring"] = (torch.randn(B, nkv, W, hd, device=DEV, generator=g).to(torch.bfloat16)
                                for _ in range(2))
    c["cos"], c["sin"] = (t.to(DEV).contiguous() for t in rope_tables(hd, pos + N + 1, 10000.0))
    return c


def _call(c, status, max_polls=0):
    out = torch.zeros(c["B"] * c["N"], c["nh"] * c["hd"], dtype=torch.bfloat16, device=DEV)
    kt = torch.zeros(c["B"], c["nkv"], c["N"], c["hd"], dtype=torch.bfloat16, device=DEV)
    vt = torch.zeros_like(kt)
    _lib.check(_lib.load().uttt_attn_tree_status(
        c["B"], c["N"], c["nh"], c["nkv"], c["hd"], c["W"], c["B"], c["cos"].shape[0], c["qkv"].data_ptr(),
        c["qkv"].shape[1], c["parents"].data_ptr(), None, c["pos"].data_ptr(), c["slots"].data_ptr(),
        c["k_ring"].data_ptr(), c["v_ring"].data_ptr(), c["cos"].data_ptr(), c["sin"].data_ptr(), kt.data_ptr(),
        vt.data_ptr(), out.data_ptr(), out.shape[1], None if status is None else status.data_ptr(), max_polls,
        torch.cuda.current_stream().cuda_stream), "uttt_attn_tree_status")
    return out, kt, vt


@pytest.mark.parametrize("shape", [(2, 9, 8, 1, 128, 8192, 9000),      # a cluster's CTAs, 17 tiles each
                                   (40, 16, 20, 5, 64, 512, 700),      # one CTA a row and KV head, 9 tiles
                                   (64, 4, 20, 5, 128, 512, 700)])     # two launches
def test_a_wait_that_expires_is_reported(shape):
    c = _case(*shape)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = _call(c, word)
    assert int(word) == 0
    out, kt, vt = _call(c, word, 2)
    torch.cuda.synchronize()
    assert int(word) == _lib.UTTT_ERR_TIMEOUT
    assert bool(torch.isnan(out).any(dim=1).any())
    assert bool((torch.isnan(out) | (out == want[0])).all())           # NaN, never a wrong number
    assert torch.equal(kt, want[1]) and torch.equal(vt, want[2])       # the nodes' own keys and values do not wait
    again = _call(c, word)                                             # the word keeps what it holds, the GPU works on
    assert int(word) == _lib.UTTT_ERR_TIMEOUT and all(torch.equal(a, b) for a, b in zip(again, want))
    assert all(torch.equal(a, b) for a, b in zip(_call(c, None), want))


def _engine():
    cfg = ModelConfig(vocab_size=512, d_model=256, n_layers=3, n_heads=4, n_kv_heads=2, d_ff_fast=384,
                      sliding_window_size=24, chunk_size=64, max_seq_len=512)
    return UtttB200(reference_init_state_dict(cfg, seed=3), cfg, max_personas=2)


def test_nothing_of_a_failed_step_is_committed(monkeypatch):
    """The word as an expired wait leaves it, put there behind the second layer's attention of the second step."""
    eng = _engine()
    st = eng.init_fast_state(1)
    prompt = torch.randint(6, 512, (30,), generator=torch.Generator().manual_seed(1))
    want, _ = eng.generate_drafted(prompt, st, 8, tree.PromptLookup(match=1))
    plain, calls, rings = tree.tree_attention, [0], []

    def expires(*a, **kw):
        out = plain(*a, **kw)
        calls[0] += 1
        if calls[0] == 4:
            rings.append(eng.rings.clone())
        if calls[0] == 5:
            kw["status"].fill_(_lib.UTTT_ERR_TIMEOUT)
        return out
    with monkeypatch.context() as m:
        m.setattr(tree, "tree_attention", expires)
        with pytest.raises(RuntimeError, match="wait"):
            eng.generate_drafted(prompt, st, 8, tree.PromptLookup(match=1))
    assert calls[0] == 6                                               # the step ran to its end, then was refused
    assert torch.equal(eng.rings, rings[0])
    assert int(eng.tree_status) == 0
    eng.check_tree_step()
    assert eng.generate_drafted(prompt, st, 8, tree.PromptLookup(match=1))[0] == want


def test_commits_wait_until_the_failure_is_raised():
    eng = _engine()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    kv = torch.ones(2, 3, 2, 2, 3, 64, dtype=torch.bfloat16, device=DEV)
    args = (i32([[5, 6, 7]] * 2), i32([[-1, 0, 1]] * 2), i32([[6, 7, 8]] * 2), kv, i32([4, 30]), i32([1, 0]))
    eng.tree_status.fill_(_lib.UTTT_ERR_TIMEOUT)
    assert eng.tree_commit(*args)[1].tolist() == [0, 0] and not bool(eng.rings.any())
    with pytest.raises(RuntimeError):
        eng.check_tree_step()
    assert eng.tree_commit(*args)[1].tolist() == [3, 3] and bool(eng.rings[:, :, 1, :, 4:7].all())


def test_status_must_be_one_int32_beside_the_rest():
    c = _case(1, 2, 4, 2, 64, 32, 5)
    for bad in (torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(1, device=DEV),
                torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            tree.tree_attention(c["qkv"], c["parents"], c["pos"], c["slots"], c["k_ring"], c["v_ring"], c["cos"],
                                c["sin"], 4, status=bad)
