"""GPU: equal calls give equal bits, whatever order their CTAs finish in.

Sums that several CTAs add to are taken in a fixed order (split-K projections) or in 64 bits, where FP32 numbers no more
than 2^23 apart add up exactly (the hidden tiles of a readout).  A repeated call therefore has nothing to differ by,
so the outputs are compared bit for bit; a second stream keeps the CTAs from arriving in the same order every time.
"""

import pytest
import torch

from utttcompanion_b200 import _lib
from utttcompanion_b200 import fastweight as fw
from utttcompanion_b200.model import UtttB200
from utttcompanion_b200.readout import fast_readout
from utttcompanion_b200.workloads import ModelConfig, reference_init_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _repeat(call, n=30):
    """The results of n calls, other work running beside every second one."""
    side, junk = torch.cuda.Stream(), torch.zeros(1 << 22, device=DEV)
    out = []
    for i in range(n):
        if i % 2:
            with torch.cuda.stream(side):
                junk.add_(1.0)
        out.append(call())
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("M,N,K", [(1, 512, 256), (3, 384, 640), (1, 2560, 2560), (64, 3840, 2560), (200, 640, 768),
                                   (500, 256, 1024), (5, 130, 64)])
def test_linear_repeats_itself_and_is_right(M, N, K):
    lib = _lib.load()
    g = torch.Generator(device=DEV).manual_seed(M + N)
    x = torch.randn(M, K, device=DEV, generator=g).to(torch.bfloat16)
    w = (torch.randn(N, K, device=DEV, generator=g) * 0.05).to(torch.bfloat16)
    ws = fw.workspace(lib.uttt_linear_workspace(M, N), torch.device(DEV, torch.cuda.current_device()), slot=2)
    ws[256:].fill_(255)                                # every bit set: FP32 NaNs; a call needs nothing of it

    def call():
        y = torch.empty(M, N, device=DEV)
        seg = (_lib.Segment * 1)(_lib.Segment(0, N, _lib.SEG_STORE, 1, y.data_ptr(), N, None, 0, 0.0, None))
        _lib.check(lib.uttt_linear(M, N, K, x.data_ptr(), w.data_ptr(), 1, seg, 1e-5, ws.data_ptr(), ws.numel(),
                                   torch.cuda.current_stream().cuda_stream), "uttt_linear")
        return y
    got = _repeat(call)
    assert all(torch.equal(got[0], y) for y in got[1:])
    # K products, exact in FP32, summed in FP32: each of the K + 8 or so roundings is 2^-24 of a partial sum, and none
    # exceeds the sum of the products' magnitudes
    ref, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    assert bool(((got[0].double() - ref).abs() <= (K + 16) * 2.0 ** -24 * mag).all())


@pytest.mark.parametrize("op", [_lib.SEG_RMSNORM, _lib.SEG_RESID])
@pytest.mark.parametrize("M,N,K", [(1, 512, 256), (3, 2560, 2560), (64, 768, 768), (200, 640, 768)])
def test_linear_epilogues_over_several_k_ranges(op, M, N, K):
    """The finishing pass against the same pass over a projection of one K range (W stacked until its tiles alone
    fill the GPU).  Both sum the same products, in another order, so y differs by at most mag = 2 (K + 16) 2^-24 of the
    products' magnitudes.  Numbers e apart, each rounded to BF16 (off by at most 2^-8 of itself), are at most
    e + 2 * 2^-8 of the larger apart.  RESID rounds y and the sum.  RMSNORM rounds y, takes the root of the mean square
    of such values (off by no more than the largest of them, relatively) and rounds the product."""
    lib = _lib.load()
    g = torch.Generator(device=DEV).manual_seed(M + N + op)
    x = torch.randn(M, K, device=DEV, generator=g).to(torch.bfloat16)
    w = (torch.randn(N, K, device=DEV, generator=g) * 0.05).to(torch.bfloat16)
    aux = torch.randn(M, N, device=DEV, generator=g).to(torch.bfloat16) if op == _lib.SEG_RESID else \
        torch.rand(N, device=DEV, generator=g) + 0.5
    many = w.repeat(-(-148 * 128 // N) + 1, 1).contiguous()

    def call(weight):
        n = weight.shape[0]
        out = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
        ws = torch.full((lib.uttt_linear_workspace(M, n),), 255, dtype=torch.uint8, device=DEV)
        ws[:256] = 0
        seg = (_lib.Segment * 1)(_lib.Segment(0, N, op, 0, out.data_ptr(), N, aux.data_ptr(), N, 0.0, None))
        _lib.check(lib.uttt_linear(M, n, K, x.data_ptr(), weight.data_ptr(), 1, seg, 1e-5, ws.data_ptr(), ws.numel(),
                                   torch.cuda.current_stream().cuda_stream), "uttt_linear")
        return out
    a, b = call(w).double(), call(many).double()
    mag = (x.double().abs() @ w.double().abs().t()) * 2 * (K + 16) * 2.0 ** -24
    y = (x.double() @ w.double().t()).abs() + mag
    big = torch.maximum(a.abs(), b.abs())
    if op == _lib.SEG_RESID:
        bound = mag + 2.0 ** -7 * (y + big) * 1.01
    else:
        off = mag / y + 2.0 ** -7                      # of y, relatively
        bound = (off + (mag.amax(1, keepdim=True) / y.square().mean(1, keepdim=True).sqrt() + 2.0 ** -7) + 2.0 ** -7) \
            * big * 1.02
    assert bool(((a - b).abs() <= bound).all())


@pytest.mark.parametrize("B,T,d,h", [(1, 1, 256, 384), (3, 1, 2560, 6912), (1, 1, 768, 2048), (70, 1, 256, 640)])
def test_decode_readout_repeats_itself(B, T, d, h):
    _readouts(B, T, d, h)


@pytest.mark.parametrize("B,T,d,h", [(1, 33, 256, 384), (1, 12, 2560, 6912), (2, 70, 768, 2048), (5, 64, 256, 640)])
def test_tiled_readout_repeats_itself(B, T, d, h):
    _readouts(B, T, d, h)


def _readouts(B, T, d, h):
    g = torch.Generator(device=DEV).manual_seed(B + T + h)
    x = torch.randn(B, T, d, device=DEV, generator=g).to(torch.bfloat16)
    packed = (torch.randn(B, d, 2 * h, device=DEV, generator=g) * d ** -0.5).to(torch.bfloat16)
    down = (torch.randn(B, h, d, device=DEV, generator=g) * h ** -0.5).to(torch.bfloat16)
    lw, lb = torch.rand(d, device=DEV, generator=g) + 0.5, torch.randn(d, device=DEV, generator=g)
    got = _repeat(lambda: fast_readout(x, packed, None, down, lw, lb, out_dtype=torch.float32, packed=True))
    assert all(torch.equal(got[0], y) for y in got[1:])


def _tiny(personas):
    cfg = ModelConfig(vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, d_ff_fast=384,
                      sliding_window_size=24, chunk_size=64, max_seq_len=512)
    sd = reference_init_state_dict(cfg, seed=3)
    sd = {k: (v * 6.0 if k in ("tok_embeddings.weight", "lm_head.weight") else v) for k, v in sd.items()}
    return UtttB200(sd, cfg, max_personas=personas)


def test_sampled_replies_repeat_themselves():
    """Prefill, packed decode steps and picks: one turned rounding in any of them would change some reply sooner or
    later (at temperature 1.2 the picks' borders lie close)."""
    eng = _tiny(6)
    st = eng.init_fast_state(1)
    for n in (33, 200):
        prompt = torch.randint(6, 512, (n,), generator=torch.Generator().manual_seed(n))
        first = eng.generate_replies(prompt, st, 40, 5, temperature=1.2, top_p=None, seed=7)
        for _ in range(12):
            assert eng.generate_replies(prompt, st, 40, 5, temperature=1.2, top_p=None, seed=7) == first


def test_logits_repeat_themselves():
    eng = _tiny(6)
    st = eng.init_fast_state(1)
    packed, down = eng.read_copies(st.w_up, st.w_gate, st.w_down)
    prompt = torch.randint(6, 512, (90,), generator=torch.Generator().manual_seed(4))
    ids, pos = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([7, 8, 9], [90, 90, 90]))
    slots, zero = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    want = None
    for _ in range(25):
        lg = eng.prefill(prompt, 0, packed, down, 0)
        eng.fork_kv([0, 0], [1, 2], [90, 90])
        got = [lg, eng.decode_step(ids, pos, slots, packed, down, zero), eng.rings[:, :, :3].clone()]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_replies_may_use_every_position_of_the_table():
    """The last reply token is picked but never decoded from: T prompt ids and n tokens use T + n - 1 positions."""
    cfg = ModelConfig(vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, d_ff_fast=384,
                      sliding_window_size=24, chunk_size=64, max_seq_len=512)
    sd = reference_init_state_dict(cfg, seed=3)
    small, large = UtttB200(sd, cfg, max_personas=2, max_positions=64), UtttB200(sd, cfg, max_personas=2)
    prompt = torch.randint(6, 512, (30,), generator=torch.Generator().manual_seed(4))
    for n in (33, 34, 35):
        got = small.generate_replies(prompt, small.init_fast_state(1), n, 2, seed=1)
        assert got == large.generate_replies(prompt, large.init_fast_state(1), n, 2, seed=1)
        assert [len(r) for r in got] == [n, n]
    with pytest.raises(ValueError):
        small.generate_replies(prompt, small.init_fast_state(1), 36, 2, seed=1)
