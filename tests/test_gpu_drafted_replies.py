"""GPU: what a draft may change in a reply: nothing but near-ties.

Every token of a drafted reply must be the rule's own pick (64 bits, on the host) from the logits that its step computed
after the path before it, with the token's own number, whatever was drafted; those logits are the undrafted ones along
the same reply up to the rounding that separates the two paths (a tree's readout runs on the tensor-core tiles, which
keep z in FP32, a decode step's on the GEMV, which rounds it to BF16).  So a drafted reply leaves the undrafted one only
where logits that close pick differently, and up to there every correct draft must have been accepted.

CLOSE: the largest difference of a logit measured over the cases below is 0.078, at logits of up to 9 (two BF16 steps
of 2^-5 there and a little; this model's LM head is six times the initial one); the bound is twice that.
"""

import numpy as np
import pytest
import torch

from drafting_refs import sample_row
from utttcompanion_b200 import sampling, tree
from utttcompanion_b200.model import UtttB200
from utttcompanion_b200.workloads import ModelConfig, reference_init_state_dict

pytestmark = pytest.mark.gpu
CLOSE = 0.16


@pytest.fixture(scope="module")
def eng():
    cfg = ModelConfig(vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, d_ff_fast=384,
                      sliding_window_size=24, chunk_size=64, max_seq_len=512)
    sd = reference_init_state_dict(cfg, seed=3)
    sd = {k: (v * 6.0 if k in ("tok_embeddings.weight", "lm_head.weight") else v) for k, v in sd.items()}
    return UtttB200(sd, cfg, max_personas=2)


def _run(eng, prompt, st, n, draft, monkeypatch, **kw):
    """(reply, steps, [(token index, its logits)], [tokens drafted along the way, accepted] per step)."""
    seen, per_step, step = [], [], {}
    plain_step, plain_commit = eng.tree_step, eng.tree_commit

    def tree_step(*a, **k):
        step["lg"], kv = plain_step(*a, **k)
        return step["lg"], kv

    def tree_commit(*a, **k):
        out = plain_commit(*a, **k)
        path = out[0][0, :int(out[1])].tolist()
        base = 1 + sum(per_step)
        seen.extend((base + d, step["lg"][0, node].cpu().numpy()) for d, node in enumerate(path))
        per_step.append(len(path))
        return out
    with monkeypatch.context() as m:
        m.setattr(eng, "tree_step", tree_step)
        m.setattr(eng, "tree_commit", tree_commit)
        ids, steps = eng.generate_drafted(prompt, st, n, draft, **kw)
    assert steps == len(per_step)
    return ids, seen, per_step


@pytest.mark.parametrize("temperature,settings", [(0.0, {}), (1.0, {}), (0.8, dict(top_p=0.9)), (1.2, dict(top_k=20))])
@pytest.mark.parametrize("length", [5, 30, 100])
def test_a_draft_changes_nothing_but_near_ties(eng, length, temperature, settings, monkeypatch):
    st, n = eng.init_fast_state(1), 40
    prompt = torch.randint(6, 512, (length,), generator=torch.Generator().manual_seed(length))
    u = sampling.reply_uniforms(n, 11 + length)
    kw = dict(temperature=temperature, u=u, **settings)
    start = prompt.tolist()
    undrafted, _, _ = _run(eng, prompt, st, n, lambda ids: ([], []), monkeypatch, **kw)

    def perfect(ids):                                  # the undrafted reply, with wrong branches beside it
        at = len(ids) - len(start)
        good = undrafted[at:at + 5] if ids[len(start):] == undrafted[:at] else []
        tokens, parents, node = [], [], 0
        for tok in good:
            tokens += [(tok + 1) % 500 + 6, tok]
            parents += [node, node]
            node = len(tokens)
        return tokens, parents
    for draft in (lambda ids: ([], []), perfect, lambda ids: ([ids[-1], 9, 8], [0, 1, 0]), tree.PromptLookup(match=1)):
        ids, seen, per_step = _run(eng, prompt, st, n, draft, monkeypatch, **kw)
        assert len(ids) == n
        along = [lg.cpu().numpy() for lg in eng.teacher_forced_logits(prompt, ids, st)]
        at = dict(seen)
        for t in range(1, n):
            want = sample_row(at[t], float(u[t]), temperature=temperature, limit=eng.active_limit, stop_free=True,
                              **settings)
            assert ids[t] == want[0], t
            assert np.abs(at[t] - along[t]).max() <= CLOSE, t
        if draft is perfect:
            same = next((t for t in range(n) if ids[t] != undrafted[t]), n)
            base = 1
            for k in per_step:                         # a step's whole draft is right: all of it is accepted
                drafted = min(5, n - base - 1)
                if base + drafted < same:
                    assert k == drafted + 1, (base, k, same)
                base += k
