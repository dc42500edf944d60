"""GPU: tree steps whose attention is two launches, in the order the engine makes them: a projection that rewrites the
packed q, k and v before each, one that takes tensor memory early behind each, the same buffers in every layer.

A step repeats itself bit for bit, so a read of a value from before, or a product that starts too early, shows against
the same step with the GPU waited for around every attention.
"""

import pytest
import torch

from utttcompanion_b200 import tree
from utttcompanion_b200.model import UtttB200
from utttcompanion_b200.workloads import ModelConfig, reference_init_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def step():
    """64 rows of up to 16 nodes at 20/5 heads of 128: 320 CTAs where the GPU holds 296."""
    cfg = ModelConfig(vocab_size=512, d_model=2560, n_layers=4, n_heads=20, n_kv_heads=5, d_ff_fast=256,
                      sliding_window_size=512, chunk_size=64, max_seq_len=4096)
    eng = UtttB200(reference_init_state_dict(cfg, seed=5), cfg, max_personas=64)
    g = torch.Generator(device=DEV).manual_seed(6)
    eng.rings.normal_(generator=g)
    st = eng.init_fast_state(1)
    packed, down = eng.read_copies(st.w_up, st.w_gate, st.w_down)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    parents = i32([[-1] + [max(0, i - 1 - (i * r) % 4) for i in range(1, 16)] for r in range(64)])
    pos, slots = i32([32 + 60 * i for i in range(64)]), i32(list(range(64)))
    nodes, zero = i32([1 + (7 * i) % 16 for i in range(64)]), torch.zeros(64, dtype=torch.int32, device=DEV)
    tokens = [torch.randint(6, 512, (64, 16), device=DEV, generator=g, dtype=torch.int32) for _ in range(3)]

    def run(k, toks=None):
        return eng.tree_step(tokens[k] if toks is None else toks, parents, pos, slots, packed, down, zero, nodes)
    live = torch.arange(16, device=DEV)[None, :] < nodes[:, None]
    return run, tokens, live


def _apart(run, k, monkeypatch):
    """The step with nothing running beside an attention."""
    plain = tree.tree_attention

    def alone(*a, **kw):
        torch.cuda.synchronize()
        out = plain(*a, **kw)
        torch.cuda.synchronize()
        return out
    with monkeypatch.context() as m:
        m.setattr(tree, "tree_attention", alone)
        return run(k)


def _same(a, b, live):
    return torch.equal(a[0][live], b[0][live]) and torch.equal(a[1], b[1])


def test_two_launches_between_projections(step, monkeypatch):
    run, _, live = step
    want = [_apart(run, k, monkeypatch) for k in range(3)]
    assert all(bool(torch.isfinite(lg[live]).all()) for lg, _ in want)
    for i in range(30):                                    # step after step, nothing waited for in between
        got = [run(k) for k in range(3)]
        assert all(_same(a, b, live) for a, b in zip(got, want)), i


def test_two_launches_captured_with_their_projections(step, monkeypatch):
    run, tokens, live = step
    want = [_apart(run, k, monkeypatch) for k in range(3)]
    toks = tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(0, toks)                                       # the stream's workspaces
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run(0, toks)
    for i in range(15):
        toks.copy_(tokens[i % 3])
        graph.replay()
        torch.cuda.synchronize()
        assert _same(got, want[i % 3], live), i
