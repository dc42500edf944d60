"""GPU: sampled and drafted generation through the engine, the serving engine and the personalizer.

A drafted reply is the undrafted one, up to the rounding that separates the paths (a tree's readout runs on the
tensor-core tiles, a decode step's on the GEMV).  Logits of packed paths are held to 2e-2 elsewhere, with weights as
initialised; these models' LM head is SCALE = 6 times that, so that some ids are likely, and logits are linear in it
(their BF16 rounding is relative): EPS = 6 * 2e-2.  So every token is checked against the undrafted logits along the same reply.  Greedy: the
token's logit is within 2 EPS of the largest.  Sampled without truncation: weights move by at most a factor
exp(+-EPS / T), so a border of the distribution function moves by at most 1 - exp(-2 EPS / T), and the token's own
interval, widened by that, must hold the number it was picked with.
"""

import math

import numpy as np
import pytest
import torch

from utttcompanion_b200 import sampling, tree
from utttcompanion_b200.dropin import uTTTPersonalizerB200
from utttcompanion_b200.model import UtttB200
from utttcompanion_b200.serving import ServingEngine
from utttcompanion_b200.workloads import ModelConfig, reference_init_state_dict

pytestmark = pytest.mark.gpu
SCALE = 6.0
EPS = SCALE * 2e-2


def _engine(personas=6, seed=3):
    cfg = ModelConfig(vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, d_ff_fast=384,
                      sliding_window_size=24, chunk_size=64, max_seq_len=512)
    sd = reference_init_state_dict(cfg, seed=seed)
    sd = {k: (v * SCALE if k in ("tok_embeddings.weight", "lm_head.weight") else v) for k, v in sd.items()}
    return cfg, UtttB200(sd, cfg, max_personas=personas)


def _prompt(n, seed, vocab=512):
    return torch.randint(6, vocab, (n,), generator=torch.Generator().manual_seed(seed))


def _allowed(lg, limit):
    lg = lg.double().cpu().numpy().copy()
    lg[[0, 1, 2, 3, 4, 5]] = -np.inf
    lg[limit:] = -np.inf
    return lg


def _check_reply(eng, prompt, state, ids, temperature=0.0, u=None, slot=0):
    logits = eng.teacher_forced_logits(prompt, list(ids), state, slot=slot)
    for t, tok in enumerate(ids):
        lg = _allowed(logits[t], eng.active_limit)
        if temperature <= 1e-5:
            assert lg[tok] >= lg.max() - 2 * EPS, (t, tok)
            continue
        w = np.exp((lg - lg.max()) / temperature)
        run = np.cumsum(w) / w.sum()
        d = 1 - math.exp(-2 * EPS / temperature)
        lo = run[tok] - w[tok] / w.sum()
        assert lo - d <= float(u[t]) <= run[tok] + d, (t, tok, lo, run[tok], float(u[t]))


def test_tree_logits_are_the_decode_logits_along_every_path():
    cfg, eng = _engine()
    st = eng.init_fast_state(1)
    packed, down = eng.read_copies(st.w_up, st.w_gate, st.w_down)
    dev = eng.device
    parents = [-1, 0, 0, 1, 1, 3, 5, 6]
    tokens = _prompt(8, 1).tolist()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    for n, slot in ((9, 0), (40, 3)):                 # a ring not full yet, and one past its window
        prompt = _prompt(n, n)
        eng.prefill(prompt, slot, packed, down, 0)
        before = eng.rings.clone()
        lg, kv = eng.tree_step(i32([tokens]), i32([parents]), i32([n]), i32([slot]), packed, down, i32([0]))
        assert torch.equal(before, eng.rings)
        for leaf in (2, 4, 7):
            line = [leaf]
            while parents[line[0]] >= 0:
                line.insert(0, parents[line[0]])
            eng.rings.copy_(before)
            for d, node in enumerate(line):
                ref = eng.decode_step(i32([tokens[node]]), i32([n + d]), i32([slot]), packed, down, i32([0]))
                assert float((lg[0, node] - ref[0]).abs().max()) <= EPS, (n, node)
        # committing the path to node 4 leaves the ring that decoding it leaves
        eng.rings.copy_(before)
        for d, node in enumerate((0, 1, 4)):
            eng.decode_step(i32([tokens[node]]), i32([n + d]), i32([slot]), packed, down, i32([0]))
        decoded = eng.rings.clone()
        eng.rings.copy_(before)
        picks = [[0] * 8]
        picks[0][0], picks[0][1], picks[0][4] = tokens[1], tokens[4], 77
        path, n_path, nxt = eng.tree_commit(i32([tokens]), i32([parents]), i32(picks), kv, i32([n]), i32([slot]))
        assert path[0].tolist() == [0, 1, 4] + [-1] * 5 and int(n_path) == 3 and int(nxt) == 77
        places = [(n + d) % cfg.sliding_window_size for d in range(3)]
        rest = [p for p in range(cfg.sliding_window_size) if p not in places]
        assert torch.equal(eng.rings[:, :, :, :, rest], before[:, :, :, :, rest])
        a, b = eng.rings[:, :, slot][:, :, :, places].float(), decoded[:, :, slot][:, :, :, places].float()
        assert float((a - b).norm() / b.norm()) <= 2e-2       # as batched and single prefills' rings


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_drafted_reply_is_the_undrafted_one(temperature):
    cfg, eng = _engine()
    st = eng.init_fast_state(1)
    prompt, n = _prompt(30, 7), 40
    u = sampling.reply_uniforms(n, 11)
    plain, plain_steps = eng.generate_drafted(prompt, st, n, lambda ids: ([], []), temperature=temperature, u=u)
    assert len(plain) == n and plain_steps == n - 1
    _check_reply(eng, prompt, st, plain, temperature, u)
    start = prompt.tolist()

    def perfect(ids):                                  # the undrafted reply, with wrong branches beside it
        at = len(ids) - len(start)
        good = plain[at:at + 5] if ids[len(start):] == plain[:at] else []
        tokens, parents, node = [], [], 0
        for tok in good:
            tokens += [(tok + 1) % 500 + 6, tok]
            parents += [node, node]
            node = len(tokens)
        return tokens, parents
    drafted, steps = eng.generate_drafted(prompt, st, n, perfect, temperature=temperature, u=u)
    _check_reply(eng, prompt, st, drafted, temperature, u)
    if drafted == plain:
        assert steps <= -(-(n - 1) // 6) + 1
    wrong, wrong_steps = eng.generate_drafted(prompt, st, n, lambda ids: ([ids[-1], 9, 8], [0, 1, 0]),
                                              temperature=temperature, u=u)
    _check_reply(eng, prompt, st, wrong, temperature, u)
    looked, looked_steps = eng.generate_drafted(prompt, st, n, tree.PromptLookup(match=1), temperature=temperature, u=u)
    _check_reply(eng, prompt, st, looked, temperature, u)
    assert looked_steps <= n - 1


def test_drafted_generation_limits_and_refusals():
    cfg, eng = _engine()
    st = eng.init_fast_state(1)
    prompt = _prompt(5, 9)
    one, steps = eng.generate_drafted(prompt, st, 1, tree.PromptLookup())
    assert len(one) == 1 and steps == 0
    assert eng.generate_drafted(prompt, st, 0, tree.PromptLookup())[0] == []
    assert eng.generate_drafted(prompt, st, 0, tree.PromptLookup(), temperature=0.5, u=torch.zeros(0))[0] == []
    three, _ = eng.generate_drafted(prompt, st, 3, lambda ids: (list(range(6, 26)), list(range(20))))
    assert len(three) == 3
    for bad in (lambda ids: ([7], []), lambda ids: ([7], [1]), lambda ids: ([512], [0]), lambda ids: ([-1], [0]),
                lambda ids: ([7] * 64, [0] * 64)):
        with pytest.raises(ValueError):
            eng.generate_drafted(prompt, st, 4, bad)
    with pytest.raises(ValueError):
        eng.generate_drafted(prompt, st, 4, tree.PromptLookup(), temperature=0.5)          # no numbers
    with pytest.raises(ValueError):
        eng.generate_drafted(prompt, st, 4, tree.PromptLookup(), temperature=-1.0)
    with pytest.raises(ValueError):
        eng.tree_step(torch.zeros(1, 65, dtype=torch.int32), torch.zeros(1, 65, dtype=torch.int32),
                      torch.zeros(1), torch.zeros(1), *eng.read_copies(st.w_up, st.w_gate, st.w_down), torch.zeros(1))


def test_packed_trees_of_several_personas():
    """Three personas with their own weights, positions and tree sizes in one step, one row without a tree."""
    cfg, eng = _engine()
    st = eng.init_fast_state(3)
    g = torch.Generator(device=eng.device).manual_seed(5)
    for w in (st.w_up, st.w_gate, st.w_down):
        w += 0.02 * w.abs().mean() * torch.randn(w.shape, generator=g, device=eng.device)
    packed, down = eng.read_copies(st.w_up, st.w_gate, st.w_down)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=eng.device)  # noqa: E731
    lens, slots, nodes = [12, 31, 24, 7], [4, 0, 2, 1], [5, 3, 0, 1]
    state = [0, 1, 2, 2]
    for n, s, w in zip(lens, slots, state):
        eng.prefill(_prompt(n, n), s, packed, down, w)
    parents = [[-1, 0, 1, 1, 0]] * 4
    tokens = [_prompt(5, 50 + r).tolist() for r in range(4)]
    before = eng.rings.clone()
    lg, kv = eng.tree_step(i32(tokens), i32(parents), i32(lens), i32(slots), packed, down, i32(state), i32(nodes))
    assert bool(torch.isfinite(lg).all())
    for r in range(4):
        if nodes[r] == 0:
            continue
        one, one_kv = eng.tree_step(i32([tokens[r][:nodes[r]]]), i32([parents[r][:nodes[r]]]), i32([lens[r]]),
                                    i32([slots[r]]), packed, down, i32([state[r]]))
        assert float((lg[r, :nodes[r]] - one[0]).abs().max()) <= EPS
    picks = i32([[t[1], t[3], 0, 9, 0] for t in tokens])
    path, n_path, nxt = eng.tree_commit(i32(tokens), i32(parents), picks, kv, i32(lens), i32(slots), i32(nodes))
    assert n_path.tolist() == [3, 2, 0, 1] and nxt.tolist()[2] == -1
    changed = (eng.rings != before).any(dim=-1).any(dim=3).any(dim=0).any(dim=0)          # (slots, W)
    for r in range(4):
        want = {(lens[r] + d) % cfg.sliding_window_size for d in range(n_path[r])}
        assert set(torch.nonzero(changed[slots[r]]).flatten().tolist()) == want
    assert not bool(changed[[3, 5]].any())


def test_replies_of_one_prompt_from_forked_rings():
    cfg, eng = _engine()
    st = eng.init_fast_state(1)
    prompt, n = _prompt(33, 21), 20
    kw = dict(temperature=0.9, top_p=None, seed=100, slots=[5, 1, 3])
    replies = eng.generate_replies(prompt, st, n, 3, **kw)
    assert replies == eng.generate_replies(prompt, st, n, 3, **kw)
    assert len({tuple(r) for r in replies}) == 3
    for i, r in enumerate(replies):
        assert len(r) == n
        _check_reply(eng, prompt, st, r, 0.9, sampling.reply_uniforms(n, 100 + i))
    short = eng.generate_replies(prompt, st, n, 2, temperature=0.9, top_k=1)
    greedy, _, _ = eng.generate_greedy(prompt, st, n)
    assert short[0] == short[1]
    _check_reply(eng, prompt, st, short[0])
    for bad in (dict(n_replies=7), dict(n_replies=0), dict(n_replies=2, slots=[1, 1]), dict(n_replies=1, slots=[6]),
                dict(n_replies=1, temperature=-0.5), dict(n_replies=1, top_p=0.0)):
        with pytest.raises(ValueError):
            eng.generate_replies(prompt, st, n, **bad)


def test_serving_samples_each_turn_with_its_own_settings():
    cfg, eng = _engine(personas=5)
    srv = ServingEngine(eng, capacity=4, max_batch=3, online_ttt=False, stop_free=True, max_sampled_tokens=24)
    prompts = [_prompt(10 + 9 * i, 60 + i).tolist() for i in range(4)]
    temps = [0.0, 0.8, 1.2, 0.8]
    turns = [srv.submit(f"u{i}", p, 24, temperature=temps[i], seed=None if i == 2 else 5 + i)
             for i, p in enumerate(prompts)]
    assert turns[0].seed == 5 and turns[2].seed is not None
    srv.run()
    st = eng.init_fast_state(1)
    for i, t in enumerate(turns):
        assert len(t.reply) == 24
        u = sampling.reply_uniforms(24, t.seed) if temps[i] else None
        _check_reply(eng, torch.tensor(prompts[i]), st, t.reply, temps[i], u, slot=4)
    again = srv.submit("u0", prompts[0], 24, temperature=1.0, top_k=1)      # one candidate: greedy
    srv.run()
    _check_reply(eng, torch.tensor(prompts[0]), st, again.reply, slot=4)
    for bad in (dict(max_new_tokens=25, temperature=0.5), dict(temperature=float("nan")), dict(top_p=2.0),
                dict(min_p=-1.0), dict(temperature=0.5, seed=-1), dict(temperature=0.5, seed=2 ** 63)):
        with pytest.raises(ValueError):
            srv.submit("x", prompts[0], **{"max_new_tokens": 8, **bad})
    with pytest.raises(ValueError):
        ServingEngine(eng, capacity=4, max_batch=1, online_ttt=False).submit("x", prompts[0], 8, temperature=0.7)


def test_personalizer_samples_where_its_engine_does():
    cfg, eng = _engine(personas=3)
    srv = ServingEngine(eng, capacity=2, max_batch=1, stop_free=True, max_sampled_tokens=16)
    p = uTTTPersonalizerB200(srv)
    prompt = _prompt(12, 70).tolist()
    a = p.interact_and_evolve("alice", prompt, max_new_tokens=16, temperature=0.9, top_p=0.95, seed=3)
    b = p.interact_and_evolve("bob", prompt, max_new_tokens=16, temperature=0.9, top_p=0.95, seed=3)
    assert len(a.reply_ids) == 16 and a.seed == 3 and a.reply_ids == b.reply_ids    # both start from W_0
    c = p.interact_and_evolve("bob", prompt, max_new_tokens=16, temperature=0.9)
    assert c.seed is not None
    with pytest.raises(ValueError):
        p.interact_and_evolve("bob", prompt, max_new_tokens=17, temperature=0.9)
