"""GPU: sizes of uttt_sample around which a row is split over more CTAs, with flat rows (every sum at its largest).

A lane adds its weights, whole numbers of at most 2^45, in a double: exact for 256 of them and no more.  With rows enough
to fill the GPU, limits of 131073 and 131074 used to leave a row to one CTA whose lanes added 264.  A row's
outputs must not depend on the batch, so every one is held against the same row in a batch of two, which is split
otherwise, and some against the 64-bit rule.
"""

import pytest
import torch

from drafting_refs import sample_row
from utttcompanion_b200 import sampling

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("V", [131065, 131072, 131073, 131074, 131075, 131081])
@pytest.mark.parametrize("settings", [dict(temperature=3e4), dict(temperature=3e4, top_p=0.99), dict(min_p=1e-6)])
def test_flat_rows_do_not_depend_on_the_batch(V, settings):
    rows = 160
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(rows, V, device=DEV, generator=g).to(torch.bfloat16)
    u = torch.rand(rows, device=DEV, generator=g)
    u[:4] = torch.tensor([0.0, 0.99999994, 0.5, 0.0644], device=DEV)      # 0.0644: a border between two warps' pieces
    ids, kept, prob = sampling.sample(x, u, **settings)
    assert bool(((ids >= 2) & (ids < V)).all())
    for r in range(0, rows, 2):
        two = sampling.sample(x[r:r + 2], u[r:r + 2], **settings)
        assert torch.equal(ids[r:r + 2], two.ids) and torch.equal(kept[r:r + 2], two.kept)
        assert torch.equal(prob[r:r + 2], two.prob)
    for r in (0, 1, 2):
        want = sample_row(x[r].float().cpu().numpy(), float(u[r]), **settings)
        assert (int(ids[r]), int(kept[r])) == want[:2]


def test_limits_inside_a_wider_row():
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(150, 140000, device=DEV, generator=g).to(torch.bfloat16)
    u = torch.rand(150, device=DEV, generator=g)
    for limit in (131073, 131074):
        st = dict(temperature=1e3, active_limit=limit)
        whole, two = sampling.sample(x, u, **st), sampling.sample(x[:2], u[:2], **st)
        assert all(torch.equal(a[:2], b) for a, b in zip(whole, two))
        want = sample_row(x[0].float().cpu().numpy(), float(u[0]), temperature=1e3, limit=limit)
        assert (int(whole.ids[0]), int(whole.kept[0])) == want[:2]


def test_numbers_of_no_row_are_refused():
    x = torch.randn(1, 100, device=DEV)
    for u in (torch.tensor(0.5, device=DEV), torch.rand(1, 1, 1, device=DEV)):
        with pytest.raises(ValueError):
            sampling.sample(x, u)
    assert sampling.sample(x, torch.rand(1, 1, device=DEV)).ids.shape == (1,)
