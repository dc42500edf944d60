"""Sampling of one token per row from given random numbers (``uttt_sample``).

``UtttB200.greedy``'s counterpart at temperature > 0: the rules of
``uTTTModel._sample_next_token`` (``model/uttt_model.py:1181-1235``) without its
repetition penalty (``check_penalty``), with top-k and min-p beside top-p, for
every row of a packed batch in one launch, each row with its own settings.  The
uniform numbers are inputs, so a pick depends on its row's logits, settings and
number alone (the logits' own last bits may depend on how many rows a step has).
"""

from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from .fastweight import _launch, _require_cuda

Setting = Union[None, int, float, torch.Tensor]
MAX_VOCAB = 262144


class Sampled(NamedTuple):
    """``ids`` int32 (rows,); ``kept`` int32 (rows,), the ids that the settings left; ``prob`` FP32 (rows,), the
    pick's share of their mass."""
    ids: torch.Tensor
    kept: torch.Tensor
    prob: torch.Tensor


def check_settings(temperature: float = 1.0, top_k: Optional[int] = None, top_p: Optional[float] = None,
                   min_p: Optional[float] = None) -> None:
    """The ``ValueError`` of settings that no call takes (the reference's checks, ``:1190-1197``)."""
    if not math.isfinite(temperature) or temperature < 0:
        raise ValueError("temperature must be finite and nonnegative")
    if top_k is not None and (not math.isfinite(top_k) or int(top_k) != top_k or not 0 <= top_k < 2 ** 31):
        raise ValueError("top_k must be a nonnegative integer")
    if top_p is not None and (not math.isfinite(top_p) or not 0 < top_p <= 1):
        raise ValueError("top_p must be finite and in (0, 1]")
    if min_p is not None and (not math.isfinite(min_p) or not 0 <= min_p <= 1):
        raise ValueError("min_p must be finite and in [0, 1]")


def check_penalty(engine, temperature: float) -> None:
    """The ``ValueError`` of sampled generation on an engine whose model asks for a repetition penalty (``:1181-1235``:
    the scores of the last 48 ids).  The packed paths keep no ids beside the logits; ``dropin.uTTTModelB200``'s
    ``stream_generate`` applies it."""
    if temperature > 1e-5 and getattr(engine, "repetition_penalty", 1.0) > 1.0:
        raise ValueError("packed sampling applies no repetition penalty: set repetition_penalty to 1, or use "
                         "uTTTModelB200.stream_generate")


def reply_uniforms(n: int, seed: int) -> torch.Tensor:
    """The ``n`` uniform numbers in [0, 1) of a reply with this seed (host FP32): token t is picked with number t."""
    return torch.rand(n, generator=torch.Generator().manual_seed(seed), dtype=torch.float32)


class SamplingRows:
    """The sampling settings and random numbers of a packed batch's rows, in device memory, where captured steps
    read them.  A row at temperature 0, as all are at first, picks greedily."""

    def __init__(self, device: torch.device, rows: int, uniforms: int):
        self.device = torch.device(device)
        self.uniforms = int(uniforms)
        self.temperature = torch.zeros(rows, device=device)
        self.top_k = torch.zeros(rows, dtype=torch.int32, device=device)
        self.top_p = torch.ones(rows, device=device)
        self.min_p = torch.zeros(rows, device=device)
        self.u = torch.zeros(rows, self.uniforms, device=device)

    def set(self, row: int, temperature: float = 0.0, top_k: Optional[int] = None, top_p: Optional[float] = None,
            min_p: Optional[float] = None, u: Optional[torch.Tensor] = None) -> None:
        """Give ``row`` its settings and, at temperature > 0, its numbers (host FP32), on the current stream."""
        check_settings(temperature, top_k, top_p, min_p)
        if not 0 <= row < self.temperature.shape[0]:
            raise ValueError("row outside the table")
        if temperature > 1e-5 and (u is None or u.numel() == 0):
            raise ValueError("a sampled row needs its random numbers")
        if u is not None and u.numel() > self.uniforms:
            raise ValueError(f"a row holds {self.uniforms} random numbers")

        def put(dst: torch.Tensor, values: torch.Tensor) -> None:
            if self.device.type == "cuda":
                values = values.pin_memory()
            dst.copy_(values, non_blocking=True)
        put(self.temperature[row:row + 1], torch.tensor([float(temperature)]))
        put(self.top_k[row:row + 1], torch.tensor([int(top_k or 0)], dtype=torch.int32))
        put(self.top_p[row:row + 1], torch.tensor([1.0 if top_p is None else float(top_p)]))
        put(self.min_p[row:row + 1], torch.tensor([float(min_p or 0.0)]))
        if u is not None and u.numel():
            put(self.u[row, :u.numel()], u.to(torch.float32).reshape(-1))

    def first(self, n: int) -> dict:
        """The arguments of ``sample`` for the first ``n`` rows."""
        return dict(u=self.u[:n], temperature=self.temperature[:n], top_k=self.top_k[:n], top_p=self.top_p[:n],
                    min_p=self.min_p[:n])


def _per_row(name: str, v: Setting, off, dtype: torch.dtype, rows: int, index: int):
    """(device pointer or None, value for all rows)."""
    if isinstance(v, torch.Tensor):
        if v.get_device() != index or v.dtype is not dtype or v.shape != (rows,) or not v.is_contiguous():
            raise ValueError(f"{name} per row must be a contiguous {dtype} tensor of {rows} on cuda:{index}")
        return v.data_ptr(), off
    return None, off if v is None else v


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = None,
           top_p: Setting = None, min_p: Setting = None, active_limit: Optional[int] = None,
           stop_free: bool = False, u_index: Optional[torch.Tensor] = None) -> Sampled:
    """One id per row of FP32 or BF16 ``logits`` (rows, V).

    ``u``: FP32 uniform numbers in [0, 1), (rows,), or (rows, n) with ``u_index`` int32 (rows,) naming each
    row's column.  ``temperature``, ``top_k``, ``top_p``, ``min_p``: a number for all rows or a device tensor
    (FP32; ``top_k`` int32) of one per row, whose values the device takes as ``include/uttt_b200.h`` says;
    a temperature of at most 1e-5 picks greedily, ``top_k`` 0, ``top_p`` 1 and ``min_p`` 0 are off.
    PAD / BOS / UNK and ids from ``active_limit`` on are never picked (nor ids 2, 4 and 5 when
    ``stop_free``), as by ``UtttB200.greedy``.  Runs on the current stream of the logits' device."""
    _require_cuda(logits, u)
    f, index = torch.float32, logits.get_device()
    is_f32 = logits.dtype is f
    if logits.dim() != 2 or not (is_f32 or logits.dtype is torch.bfloat16):
        raise ValueError("logits must be FP32 or BF16 (rows, V) with V > 6")
    rows, V = logits.shape
    if not 6 < V <= MAX_VOCAB:
        raise ValueError(f"logits must be FP32 or BF16 (rows, V) with 6 < V <= {MAX_VOCAB}")
    if u.get_device() != index or u.dtype is not f or u.dim() not in (1, 2) or u.shape[0] != rows \
            or not u.is_contiguous():
        raise ValueError("u must be a contiguous FP32 (rows,) or (rows, n) tensor beside the logits")
    n_u = 1 if u.dim() == 1 else u.shape[1]
    if rows == 0:
        return Sampled(*(torch.empty(0, dtype=t, device=logits.device) for t in (torch.int32, torch.int32, f)))
    ld, step = logits.stride()
    if step != 1 or (rows > 1 and ld < V):
        logits = logits.contiguous()
        ld = V
    if u_index is None:
        at = None
        if n_u != 1:
            raise ValueError("u of several numbers a row needs u_index")
    elif u_index.get_device() != index or u_index.dtype is not torch.int32 or u_index.shape != (rows,) \
            or not u_index.is_contiguous() or n_u == 0:
        raise ValueError("u_index must be a contiguous int32 (rows,) tensor beside the logits")
    else:
        at = u_index.data_ptr()
    limit = V if active_limit is None else min(V, int(active_limit))
    if limit <= 2:
        raise ValueError("Active vocabulary must include EOS")
    tp, t0 = _per_row("temperature", temperature, 1.0, f, rows, index)
    kp, k0 = _per_row("top_k", top_k, 0, torch.int32, rows, index)
    pp, p0 = _per_row("top_p", top_p, 1.0, f, rows, index)
    mp, m0 = _per_row("min_p", min_p, 0.0, f, rows, index)
    check_settings(t0, k0, p0, m0)
    opt = _lib.Sampling(tp, kp, pp, mp, t0, int(k0), p0, m0)
    prob = torch.empty_like(u) if u.dim() == 1 else torch.empty(rows, dtype=f, device=u.device)
    ids = torch.empty(rows, dtype=torch.int32, device=u.device)
    kept = torch.empty_like(ids)
    on, stream = _launch(u.device)
    with on:
        st = _lib.load().uttt_sample(rows, V, logits.data_ptr(), is_f32, ld if rows > 1 else V, limit, bool(stop_free),
                                     C.byref(opt), u.data_ptr(), n_u, at, n_u, ids.data_ptr(), kept.data_ptr(),
                                     prob.data_ptr(), stream)
    if st:
        _lib.check(st, "uttt_sample")
    return Sampled(ids, kept, prob)
