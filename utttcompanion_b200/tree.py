"""Drafted tokens as a tree: attention of all its nodes over the KV rings, and the path that the picks accept.

One packed step verifies a tree of drafted tokens per persona (``UtttB200.tree_step``): every node attends to the
persona's KV ring and to its own path of the tree (``tree_attention``), the model's pick after each node decides
which path stands (``tree_accept``), and ``kv_cache.ring_commit`` puts that path's keys and values into the rings.
The reference drafts along one line (``model/uttt_model.py:1052-1179``).
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .fastweight import _launch, _require_cuda

MAX_NODES = 64
MAX_LD = 2 ** 31                     # elements from one row to the next


def check_tree(parents: Sequence[int]) -> None:
    """The ``ValueError`` of a host-side tree that no call takes: node 0 is the root (-1), every other node's
    parent comes before it, and there are at most ``MAX_NODES``."""
    if not 1 <= len(parents) <= MAX_NODES:
        raise ValueError(f"a drafted tree has 1 to {MAX_NODES} nodes")
    if parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents) if i > 0):
        raise ValueError("node 0 is the root (parent -1) and a node's parent comes before it")


def depths(parents: Sequence[int]) -> List[int]:
    """How many ancestors each node of a host-side tree has."""
    out: List[int] = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def prune(tokens: Sequence[int], parents: Sequence[int], depth: Sequence[int], most: int):
    """(tokens, parents, depth) of the nodes at most ``most`` deep."""
    keep = [i for i, d in enumerate(depth) if d <= most]
    at = {i: k for k, i in enumerate(keep)}
    return ([tokens[i] for i in keep], [-1 if parents[i] < 0 else at[parents[i]] for i in keep],
            [depth[i] for i in keep])


class PromptLookup:
    """Drafts from the text itself: what followed earlier occurrences of the last few ids, the latest first, merged
    into one tree.  An instance is a ``draft`` of ``UtttB200.generate_drafted``."""

    def __init__(self, match: int = 2, depth: int = 8, nodes: int = 16):
        """``match`` ids must agree (fewer at the start of a text); continuations of up to ``depth`` ids; at most
        ``nodes`` drafted ids."""
        if match < 1 or depth < 1 or not 1 <= nodes < MAX_NODES:
            raise ValueError(f"match and depth must be positive and nodes between 1 and {MAX_NODES - 1}")
        self.match, self.depth, self.nodes = match, depth, nodes

    def __call__(self, ids: Sequence[int]) -> Tuple[List[int], List[int]]:
        n = min(self.match, len(ids))
        last = list(ids[-n:])
        tokens: List[int] = []
        parents: List[int] = []
        child = {}
        for at in range(len(ids) - n - 1, -1, -1):
            if len(tokens) >= self.nodes:
                break
            if list(ids[at:at + n]) != last:
                continue
            node = 0
            for tok in ids[at + n:at + n + self.depth]:
                nxt = child.get((node, tok))
                if nxt is None:
                    if len(tokens) >= self.nodes:
                        break
                    tokens.append(int(tok))
                    parents.append(node)
                    nxt = child[(node, tok)] = len(tokens)
                node = nxt
        return tokens, parents


def _int_rows(name: str, t: Optional[torch.Tensor], shape, index: int) -> Optional[int]:
    """Address of a contiguous int32 tensor of this shape on CUDA device ``index`` (None for None)."""
    if t is None:
        return None
    if t.get_device() != index or t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 {tuple(shape)} tensor on cuda:{index}")
    return t.data_ptr()


def tree_attention(qkv: torch.Tensor, parents: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor,
                   k_ring: torch.Tensor, v_ring: torch.Tensor, rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                   n_heads: int, n_nodes: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   k_tree: Optional[torch.Tensor] = None, v_tree: Optional[torch.Tensor] = None,
                   status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Attention of B trees of N nodes (``uttt_attn_tree_status``); returns ``(out, k_tree, v_tree)``.

    ``qkv`` BF16 (B * N, [q | k | v] heads), rows any stride; ``parents`` int32 (B, N); ``pos`` and ``slots``
    int32 (B,): positions cached so far and ring slot of each row; ``k_ring`` / ``v_ring`` BF16
    (slots, n_kv, W, hd) of one layer, only read; ``rope_cos`` / ``rope_sin`` FP32 (positions, hd);
    ``n_nodes`` int32 (B,): nodes of each row (default N).  ``out`` BF16 (B * N, n_heads * hd), rows any stride,
    ``k_tree`` / ``v_tree`` BF16 (B, n_kv, N, hd): taken if given, else new (zeros); what lies behind a row's last
    node is left as it was.  ``status`` int32 (1,): becomes nonzero if a device wait expires (the wait's rows of
    ``out`` are NaN then)."""
    _require_cuda(qkv, parents)
    dev, bf, index = qkv.device, torch.bfloat16, qkv.get_device()
    if parents.dim() != 2 or k_ring.dim() != 4:
        raise ValueError("parents must be (B, N) and the rings (slots, n_kv, W, hd)")
    B, N = parents.shape
    n_slots, n_kv, W, hd = shape = k_ring.shape
    for t in (k_ring, v_ring):
        if t.get_device() != index or t.dtype is not bf or t.shape != shape or not t.is_contiguous() or 0 in shape:
            raise ValueError("the rings must be contiguous BF16 tensors of one shape beside qkv")
    if not 1 <= N <= MAX_NODES:
        raise ValueError(f"a drafted tree has 1 to {MAX_NODES} nodes")
    R, q_dim = B * N, n_heads * hd
    if n_heads < 1 or n_heads % n_kv or qkv.dtype is not bf or qkv.dim() != 2 or qkv.shape[0] != R:
        raise ValueError("qkv must be BF16 (B * N, (n_heads + 2 * n_kv) * hd) rows")
    qkv_ld, step = qkv.stride()
    if step != 1 or qkv.shape[1] < q_dim + 2 * n_kv * hd or qkv_ld >= MAX_LD:
        raise ValueError("qkv must be BF16 (B * N, (n_heads + 2 * n_kv) * hd) rows")
    table = rope_cos.shape
    for t in (rope_cos, rope_sin):
        if t.get_device() != index or t.dtype is not torch.float32 or t.shape != table or not t.is_contiguous():
            raise ValueError("rope_cos and rope_sin must be contiguous FP32 (positions, hd) tables")
    if len(table) != 2 or table[1] != hd or table[0] < 1:
        raise ValueError("rope_cos and rope_sin must be contiguous FP32 (positions, hd) tables")
    if out is None:
        out = torch.zeros(R, q_dim, dtype=bf, device=dev)
    elif out.get_device() != index or out.dtype is not bf or out.shape != (R, q_dim):
        raise ValueError("out must be BF16 (B * N, n_heads * hd) rows")
    out_ld, step = out.stride()
    if (step != 1 or out_ld >= MAX_LD) and R:
        raise ValueError("out must be BF16 (B * N, n_heads * hd) rows")
    kv_shape = (B, n_kv, N, hd)
    k_tree = torch.zeros(kv_shape, dtype=bf, device=dev) if k_tree is None else k_tree
    v_tree = torch.zeros(kv_shape, dtype=bf, device=dev) if v_tree is None else v_tree
    for t in (k_tree, v_tree):
        if t.get_device() != index or t.dtype is not bf or t.shape != kv_shape or not t.is_contiguous():
            raise ValueError("k_tree and v_tree must be contiguous BF16 (B, n_kv, N, hd)")
    rows = (B,)
    args = (_int_rows("parents", parents, (B, N), index), _int_rows("n_nodes", n_nodes, rows, index),
            _int_rows("pos", pos, rows, index), _int_rows("slots", slots, rows, index))
    word = _int_rows("status", status, (1,), index)
    if B == 0:
        return out, k_tree, v_tree
    on, stream = _launch(dev)
    with on:
        st = _lib.load().uttt_attn_tree_status(B, N, n_heads, n_kv, hd, W, n_slots, table[0], qkv.data_ptr(),
                                               qkv_ld if R > 1 else qkv.shape[1], *args, k_ring.data_ptr(),
                                               v_ring.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(),
                                               k_tree.data_ptr(), v_tree.data_ptr(), out.data_ptr(),
                                               out_ld if R > 1 else q_dim, word, 0, stream)
    if st:
        _lib.check(st, "uttt_attn_tree_status")
    return out, k_tree, v_tree


def tree_accept(tokens: torch.Tensor, parents: torch.Tensor, picks: torch.Tensor,
                n_nodes: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The accepted path of each tree (``uttt_tree_accept``): ``(path (B, N), n_path (B,), next (B,))`` int32.

    ``tokens``, ``parents``, ``picks`` int32 (B, N): each node's drafted token and parent, and the model's pick
    after it.  The path is node 0, then from each node on its lowest later child that holds the pick; -1 behind
    its last node, whose pick is ``next``."""
    _require_cuda(tokens)
    if tokens.dim() != 2:
        raise ValueError("tokens must be (B, N)")
    index, shape = tokens.get_device(), tokens.shape
    B, N = shape
    if not 1 <= N <= MAX_NODES:
        raise ValueError(f"a drafted tree has 1 to {MAX_NODES} nodes")
    ptrs = (_int_rows("tokens", tokens, shape, index), _int_rows("parents", parents, shape, index),
            _int_rows("n_nodes", n_nodes, (B,), index), _int_rows("picks", picks, shape, index))
    path = torch.empty_like(tokens)
    n_path = torch.empty(B, dtype=torch.int32, device=tokens.device) if n_nodes is None else torch.empty_like(n_nodes)
    following = torch.empty_like(n_path)
    if B:
        on, stream = _launch(tokens.device)
        with on:
            st = _lib.load().uttt_tree_accept(B, N, *ptrs, path.data_ptr(), n_path.data_ptr(), following.data_ptr(),
                                              stream)
        if st:
            _lib.check(st, "uttt_tree_accept")
    return path, n_path, following
