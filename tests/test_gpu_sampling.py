"""GPU: uttt_sample against the 64-bit rule, row by row.

The pick and the number of kept ids must be equal.  A probability is one rounding to FP32 (2^-24 relative) of a
quotient w / sum w of weights.  Each weight is a whole number of 2^-45 of the largest; from 2^-24 on it is off by at most
2^-38 of itself before that rounding (the polynomial), below by 2^-19 (x of at most 64 from three FP32 roundings, 2^-24
each, and 2^-x by 2^-22), which is 2^-43 of the largest.  So |error| <= (2^-24 + 2^-37 + n 2^-42) p + n 2^-46.
"""

import math

import numpy as np
import pytest
import torch

from drafting_refs import sample_row
from utttcompanion_b200 import sampling

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _check(x, u, ids, kept, prob, settings, limit=None, stop_free=False):
    x, u = x.float().cpu().numpy(), u.cpu().numpy()
    ids, kept, prob = ids.tolist(), kept.tolist(), prob.tolist()
    for r in range(x.shape[0]):
        s = {k: (v[r].item() if isinstance(v, torch.Tensor) else v) for k, v in settings.items() if v is not None}
        want = sample_row(x[r], u[r], limit=limit, stop_free=stop_free, **s)
        assert (ids[r], kept[r]) == want[:2], (r, s, ids[r], kept[r], want)
        assert abs(prob[r] - want[2]) <= (2.0 ** -24 + 2.0 ** -37 + x.shape[1] * 2.0 ** -42) * want[2] + x.shape[1] * 2.0 ** -46, (r, prob[r], want)


def _logits(rows, V, dtype, seed, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, V, device=DEV, generator=g) * std
    hot = torch.randint(0, V, (rows, 10), device=DEV, generator=g)
    x.scatter_add_(1, hot, torch.rand(rows, 10, device=DEV, generator=g) * 8.0)
    return x.to(torch.bfloat16).to(dtype), torch.rand(rows, device=DEV, generator=g)


@pytest.mark.parametrize("settings", [
    dict(), dict(temperature=0.0), dict(temperature=0.6), dict(top_k=1), dict(top_k=50), dict(top_k=700),
    dict(top_p=0.9), dict(top_p=0.3, temperature=1.5), dict(min_p=0.05), dict(min_p=1.0),
    dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02), dict(top_k=1000, top_p=0.99), dict(top_k=10 ** 9),
    dict(temperature=0.02, top_p=0.5), dict(temperature=50.0, top_p=0.7), dict(top_p=1e-6),
])
@pytest.mark.parametrize("rows,V,dtype", [(1, 32000, torch.float32), (5, 8003, torch.bfloat16)])
def test_settings(rows, V, dtype, settings):
    x, u = _logits(rows, V, dtype, 1)
    _check(x, u, *sampling.sample(x, u, **settings), settings)


@pytest.mark.parametrize("rows,V,dtype,limit,stop_free", [
    (1, 7, torch.float32, None, True),           # one candidate
    (3, 8, torch.bfloat16, 3, False),            # id 2 alone
    (2, 33, torch.float32, 21, False),
    (300, 257, torch.float32, None, False),      # more rows than SMs
    (200, 2048, torch.bfloat16, 2001, True),
    (2, 40001, torch.float32, 40000, False),
    (1, 262144, torch.bfloat16, None, False),    # the widest vocabulary: 32768 logits a CTA
    (150, 36000, torch.float32, None, False),
])
@pytest.mark.parametrize("settings", [dict(temperature=0.9, top_p=0.92), dict(top_k=7, min_p=0.01), dict()])
def test_sizes(rows, V, dtype, limit, stop_free, settings):
    x, u = _logits(rows, V, dtype, 2)
    _check(x, u, *sampling.sample(x, u, active_limit=limit, stop_free=stop_free, **settings), settings, limit,
           stop_free)


@pytest.mark.parametrize("V", [131072, 131080, 262144])
def test_the_most_that_one_cta_takes(V):
    """Around the sizes that split a row whatever the batch; equal logits fill one bin with all of a CTA's weights."""
    x, u = _logits(150, V, torch.bfloat16, 17)
    x[0] = 0.0
    x[1] = 0.0
    x[1, 7] = 1.0
    for st in (dict(top_p=0.7), dict(top_k=V - 100, top_p=0.999), dict()):
        for rows in (2, 150):
            got = sampling.sample(x[:rows], u[:rows], **st)
            n = min(rows, 3)
            _check(x[:n], u[:n], *(t[:n] for t in got), st)


def test_settings_per_row():
    rows = 64
    x, u = _logits(rows, 5000, torch.float32, 3)
    g = torch.Generator(device=DEV).manual_seed(4)
    r = torch.rand(4, rows, device=DEV, generator=g)
    st = dict(temperature=torch.where(r[0] < 0.3, 0.0, r[0] * 2), top_k=(r[1] * 100 - 30).to(torch.int32),
              top_p=torch.where(r[2] < 0.3, 1.0, r[2]), min_p=torch.where(r[3] < 0.5, 0.0, r[3] * 0.2))
    _check(x, u, *sampling.sample(x, u, **st), {**st, "top_k": st["top_k"].clamp_min(0)})


@pytest.mark.parametrize("V", [300, 9000])
def test_device_values_out_of_range(V):
    """Per-row values that the host checks would refuse: each has a meaning, none an effect beyond its row."""
    nan, inf = float("nan"), float("inf")
    st = dict(temperature=[nan, -1.0, 0.8, 0.8, 0.8, 0.8, 0.8, 0.8], top_k=[0, 0, -5, 0, 20, 0, 0, 2 ** 31 - 1],
              top_p=[1, 1, 0.9, 0.0, -1.0, nan, 7.0, 0.9], min_p=[0, 0, 0, 0, 0, nan, 3.0, -1.0])
    means = dict(temperature=[0, 0] + [0.8] * 6, top_k=[0, 0, 0, 1, 1, 0, 0, 0], top_p=[1, 1, 0.9, 1, 1, 1, 1, 0.9],
                 min_p=[0, 0, 0, 0, 0, 0, 1.0, 0])
    x, u = _logits(8, V, torch.float32, 14)

    def tensors(d):
        return {k: torch.tensor(v, device=DEV, dtype=torch.int32 if k == "top_k" else torch.float32)
                for k, v in d.items()}
    _check(x, u, *sampling.sample(x, u, **tensors(st)), tensors(means))
    for given, used in ((-1.0, 0.0), (1.0, 0.99999994), (inf, 0.99999994), (nan, 0.99999994)):
        got = sampling.sample(x, torch.full((8,), given, device=DEV), top_p=0.9)
        _check(x, torch.full((8,), used, device=DEV), *got, dict(top_p=0.9))


@pytest.mark.parametrize("V", [700, 40000])
@pytest.mark.parametrize("settings", [
    dict(top_k=400), dict(top_k=512), dict(top_k=513, top_p=0.8), dict(top_p=0.9999), dict(top_p=0.5, min_p=0.2),
    dict(top_k=100, top_p=0.999999, min_p=1e-9), dict(temperature=0.1, top_p=0.99), dict(temperature=9.0, top_k=64),
])
@pytest.mark.parametrize("std", [0.0, 0.01, 6.0])
def test_few_and_many_candidates_down_to_the_cut(V, settings, std):
    x, u = _logits(4, V, torch.float32, 15, std)
    x[2] = x[2].round()                            # many equals
    _check(x, u, *sampling.sample(x, u, **settings), settings)


def _special(V, dtype):
    """Rows whose values go to the edges of the type."""
    low = torch.finfo(dtype).min
    g = torch.Generator(device=DEV).manual_seed(5)
    base = (torch.randn(V, device=DEV, generator=g) * 2).to(dtype)
    rows = []

    def row(f):
        t = base.clone()
        f(t)
        rows.append(t)
    row(lambda t: t.fill_(0.0))                                       # every logit equal
    row(lambda t: t.fill_(-math.inf))                                 # nothing left
    row(lambda t: t.fill_(math.nan))
    row(lambda t: t.fill_(low))                                       # everything at the type's lowest value
    row(lambda t: t[10:].fill_(low))                                  # a mask of the lowest value
    row(lambda t: t[:-1].fill_(-math.inf))                            # one candidate, the last id
    row(lambda t: t[::3].fill_(math.nan))
    row(lambda t: t[20:23].fill_(math.inf))                           # several infinities: they alone have mass
    row(lambda t: t[::2].fill_(-math.inf))
    row(lambda t: t.copy_(torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0)))   # both zeros are equal
    row(lambda t: t.mul_(1e-40 if dtype == torch.float32 else 1e-39))  # subnormal numbers
    row(lambda t: t.mul_(1e30))
    row(lambda t: t.copy_((t * 0.5).round()))                         # a few values, thousands of equals
    row(lambda t: t.copy_(torch.linspace(1.0, 1.0 + 1e-3, V)))        # neighbours
    return torch.stack(rows)


@pytest.mark.parametrize("settings", [
    dict(), dict(top_k=3), dict(top_k=999), dict(top_p=0.5), dict(top_p=0.37, top_k=700), dict(min_p=0.5),
    dict(temperature=0.0), dict(temperature=1e30), dict(top_k=1500, top_p=0.9, min_p=0.3, temperature=3.0),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2049, 12000])
def test_values_at_the_edges(V, dtype, settings):
    x = _special(V, dtype)
    n = x.shape[0]
    for uv in (0.0, 0.25, 0.7310586, 0.99999994):
        u = torch.full((n,), uv, device=DEV)
        _check(x, u, *sampling.sample(x, u, **settings), settings)


@pytest.mark.parametrize("temperature", [1.01e-5, 1e29, 1e31, 2e37, 3.4e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperatures_and_logits_over_the_whole_range(dtype, temperature):
    """Differences of logits beyond the largest FP32 number, and temperatures whose inverse FP32 does not hold."""
    V, top = 5000, torch.finfo(dtype).max
    x, u = _logits(6, V, dtype, 16)
    x[1] *= top / 64
    x[2] = torch.linspace(-1.0, 1.0, V, device=DEV).to(dtype) * top
    x[3, 9:12] = torch.inf
    x[3, 12:15] = top                                                 # no weight beside an infinity
    x[4, :] = -top
    x[4, 6:20] = top
    x[5, ::2] = -torch.inf
    for st in (dict(), dict(top_p=0.6), dict(top_k=1700, min_p=0.2), dict(top_k=9, top_p=0.8)):
        _check(x, u, *sampling.sample(x, u, temperature=temperature, **st), dict(temperature=temperature, **st))


def test_strides_alignment_and_u_index():
    x, _ = _logits(6, 1003, torch.bfloat16, 6)
    big = torch.full((6, 1100), 50.0, device=DEV, dtype=torch.bfloat16)
    big[:, 3:1006] = x                                                # rows 2200 bytes apart, from byte 6 on
    u = torch.rand(6, 9, device=DEV, generator=torch.Generator(device=DEV).manual_seed(7))
    at = torch.tensor([0, 8, 3, 3, -5, 100], dtype=torch.int32, device=DEV)
    want = u[torch.arange(6, device=DEV), at.long().clamp(0, 8)]
    got = sampling.sample(big[:, 3:1006], u, temperature=0.7, top_p=0.9, u_index=at)
    _check(x, want, *got, dict(temperature=0.7, top_p=0.9))
    cols = x.t().contiguous().t()                                     # columns apart: taken as a copy
    again = sampling.sample(cols, want, temperature=0.7, top_p=0.9)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_pick_does_not_depend_on_the_batch():
    x, u = _logits(40, 32000, torch.float32, 8)
    st = dict(temperature=0.9, top_k=400, top_p=0.97)
    whole = sampling.sample(x, u, **st)
    for r in (0, 17, 39):
        one = sampling.sample(x[r:r + 1], u[r:r + 1], **st)
        assert all(torch.equal(a[r:r + 1], b) for a, b in zip(whole, one))
    assert all(torch.equal(a, b) for a, b in zip(whole, sampling.sample(x, u, **st)))


def test_picks_follow_the_distribution():
    V, n = 64, 60000
    x = _logits(1, V, torch.float32, 9)[0]
    u = (torch.arange(n, device=DEV) + 0.5) / n                        # evenly spread numbers: counts are exact to 1
    ids = sampling.sample(x.expand(n, V).contiguous(), u.float(), temperature=1.2, top_p=0.9).ids
    got = torch.bincount(ids.long(), minlength=V).cpu().numpy()
    w = np.exp((x[0].double().cpu().numpy() - float(x[0, 4:].max().cpu())) / float(np.float32(1.2)))
    w[[0, 1, 3]] = 0
    order = np.argsort(-w, kind="stable")
    before = np.cumsum(w[order]) - w[order]
    w[order[before > float(np.float32(0.9)) * w.sum()]] = 0
    # a border between two picks moves by less than one number; FP32 numbers are off by at most 2^-25
    assert np.abs(got - w / w.sum() * n).max() <= 2 + n * 2.0 ** -24


def test_captured_on_another_stream_and_replayed():
    x, u = _logits(9, 9000, torch.float32, 10)
    st = dict(temperature=torch.full((9,), 0.8, device=DEV), top_p=torch.full((9,), 0.9, device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampling.sample(x, u, **st)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = sampling.sample(x, u, **st)
    for seed in (11, 12):
        a, b = _logits(9, 9000, torch.float32, seed)
        x.copy_(a)
        u.copy_(b)
        st["top_p"].fill_(0.5 + 0.03 * seed)
        graph.replay()
        torch.cuda.synchronize()
        _check(x, u, *got, st)


def test_no_rows_and_refusals():
    x, u = _logits(2, 100, torch.float32, 13)
    assert sampling.sample(x[:0], u[:0]).ids.shape == (0,)
    for bad in (dict(logits=x.double()), dict(u=u[:1]), dict(u=u.double()), dict(logits=x[:, :6]),
                dict(top_k=torch.ones(2, device=DEV)), dict(top_p=torch.ones(3, device=DEV)),
                dict(u=torch.rand(2, 3, device=DEV)), dict(u_index=torch.zeros(2, device=DEV)),
                dict(active_limit=2), dict(active_limit=-2 ** 32 + 9), dict(temperature=-1.0), dict(u=u.cpu()),
                dict(logits=x[:1, :1].expand(2, 2 ** 32 + 64)), dict(logits=x[:1].expand(2 ** 16, 100))):
        a = {**dict(logits=x, u=u), **bad}
        with pytest.raises(ValueError):
            sampling.sample(a.pop("logits"), a.pop("u"), **a)
    _check(x, u, *sampling.sample(x, u, active_limit=2 ** 32 + 5), {})   # no more than there are
