"""Copies of the KV rings of all layers at once (``uttt_kv_ring_commit``, ``uttt_kv_ring_fork``).

``rings`` is BF16 (2, layers, slots, n_kv, W, hd): keys, then values; ``UtttB200.rings`` holds an engine's, and
``k_ring[i]`` / ``v_ring[i]`` are its layers.  Position p of a persona is at place p % W of its slot.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch

from . import _lib
from .fastweight import _launch, _require_cuda
from .tree import MAX_NODES, _int_rows


def _check_rings(rings: torch.Tensor) -> None:
    if rings.dim() != 6 or rings.shape[0] != 2 or rings.dtype is not torch.bfloat16 or not rings.is_contiguous() \
            or 0 in rings.shape:
        raise ValueError("rings must be contiguous BF16 (2, layers, slots, n_kv, W, hd)")


def ring_commit(rings: torch.Tensor, tree_kv: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor,
                path: torch.Tensor, n_path: torch.Tensor) -> None:
    """Put an accepted path into the rings, in place: node ``path[b, t]`` of ``tree_kv`` BF16
    (2, layers, B, n_kv, N, hd) at position ``pos[b] + t`` of slot ``slots[b]``, t < ``n_path[b]``
    (int32 device tensors of ``tree.tree_accept``; the slots of a batch must differ)."""
    _require_cuda(rings)
    _check_rings(rings)
    _, L, S, n_kv, W, hd = rings.shape
    index = rings.get_device()
    if tree_kv.get_device() != index or tree_kv.dtype is not torch.bfloat16 or tree_kv.dim() != 6 \
            or not tree_kv.is_contiguous():
        raise ValueError("tree_kv must be contiguous BF16 (2, layers, B, n_kv, N, hd) beside the rings")
    two, layers, B, heads, N, width = tree_kv.shape
    if (two, layers, heads, width) != (2, L, n_kv, hd) or not 1 <= N <= MAX_NODES:
        raise ValueError("tree_kv does not fit the rings' layers and heads")
    rows = (B,)
    ptrs = (_int_rows("pos", pos, rows, index), _int_rows("slots", slots, rows, index),
            _int_rows("path", path, (B, N), index), _int_rows("n_path", n_path, rows, index))
    if B == 0:
        return
    tree_stride, ring_stride = B * n_kv * N * hd, S * n_kv * W * hd
    t, r = tree_kv.data_ptr(), rings.data_ptr()
    on, stream = _launch(rings.device)
    with on:
        st = _lib.load().uttt_kv_ring_commit(L, B, N, n_kv, hd, W, S, t, t + 2 * L * tree_stride, tree_stride, r,
                                             r + 2 * L * ring_stride, ring_stride, *ptrs, stream)
    if st:
        _lib.check(st, "uttt_kv_ring_commit")


def ring_fork(rings: torch.Tensor, src: Sequence[int], dst: Sequence[int],
              end_pos: Optional[Sequence[int]] = None) -> None:
    """Copy slot ``src[i]``'s rings of all layers to slot ``dst[i]``, in place, for host lists of slots: the places
    of its first ``end_pos[i]`` positions (default: all).  Every source is read as it was before the call, so a
    list of moves can compact slots; equal destinations and swaps in a cycle raise ``ValueError``."""
    _require_cuda(rings)
    _check_rings(rings)
    _, L, S, n_kv, W, hd = rings.shape
    n = len(src)
    if len(dst) != n or (end_pos is not None and len(end_pos) != n):
        raise ValueError("src, dst and end_pos must have one entry per pair")
    if n == 0:
        return
    if min(src) < 0 or max(src) >= S or min(dst) < 0 or max(dst) >= S or (end_pos is not None and min(end_pos) < 0):
        raise ValueError("slot out of range, or a negative position")
    arr = C.c_int * n
    ring_stride, r = S * n_kv * W * hd, rings.data_ptr()
    dev = rings.device
    on, stream = _launch(dev)
    with on:
        st = _lib.load().uttt_kv_ring_fork(L, n, n_kv, hd, W, S, r, r + 2 * L * ring_stride, ring_stride, arr(*src),
                                           arr(*dst), None if end_pos is None else arr(*(min(e, W) for e in end_pos)),
                                           stream)
    _lib.check(st, "uttt_kv_ring_fork")
