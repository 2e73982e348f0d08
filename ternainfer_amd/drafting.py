"""Decoding with drafted tokens: several continuations of a text go through the model at once, and the one that it would have written itself stays.

The drafts of a step are a tree: node 0 is the token that is certain (the last one written), every other node continues the node that `parents` names.
A step writes node i's key and value into slot `start + i` of its sequence, attends with `tree_attention`, takes the branch with `tree_accept`, and
puts its rows where the text ends with `cache_move`.  Kernels and their conventions: csrc/draft_tree_kernel.h, csrc/tree_attention_kernel.h.  Every
function takes tensors of one GPU, which need not be the current one, and enqueues on that GPU's current stream; it raises ValueError (TypeError where an
argument is no tensor) for what the kernels do not take, before anything is enqueued.  None has a backward pass, none waits for the device.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib


class DraftTree(NamedTuple):
    """mask int64 [B, T, (T + 63) / 64], bit j of a node's words for itself and each of its ancestors; depth int64 [B, T], 0 for a root.  Padding:
    no bit, depth -1."""
    mask: torch.Tensor
    depth: torch.Tensor


def draft_tree(parents: torch.Tensor) -> DraftTree:
    """Masks and depths of trees: parents int64 [B, T] (T up to 512), of node i a node before it or -1 for a root.  A node with any other parent is padding,
    and what continues it too."""
    return DraftTree(*_lib.native().draft_tree(parents))


def tree_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, start: torch.Tensor, mask: torch.Tensor,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of a tree's nodes q bf16 [B, H, T, D] over the cache bf16 [B, KV, S, D] (any strides of whole 16 bytes; D 64 or 128, S up to 2^25): bf16
    [B * T, H * D].  Sequence b's node i sees the slots 0 .. start[b] - 1 (int64 [B]) and slot start[b] + j of every node j in its mask (`draft_tree`'s,
    or int64 [T, W] for all sequences) -- and nothing of what any other slot holds.  A node without a bit (padding), and a sequence with a negative start, give
    zeros; a node that sees a slot behind the cache, or has a score above what float32 holds,
    gives NaN.  scale: D ** -0.5 by default."""
    return _lib.native().tree_attention(q, cache_k, cache_v, start, mask, scale)


class TreeAccepted(NamedTuple):
    """path int64 [B, T]: the nodes of the branch, then -1; count int64 [B] of them; next int64 [B]: the token behind the last."""
    path: torch.Tensor
    count: torch.Tensor
    next: torch.Tensor


def tree_accept(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor) -> TreeAccepted:
    """The branch that greedy decoding takes, from the nodes' logits [B, T, V] (bfloat16 or float32) and their tokens, int64 [B, T]: from node 0 on the
    first child that carries the token of the node's largest logit (equal ones: the lowest, NaN never; 0 where none is above -inf), while there is one.  Where node 0 is no root
    (parents[b, 0] other than -1) the sequence has no step: count 0, next -1."""
    return TreeAccepted(*_lib.native().tree_accept(logits, tokens, parents))


def cache_move(caches: Sequence[torch.Tensor], start: torch.Tensor, path: torch.Tensor, count: torch.Tensor) -> None:
    """Slot start[b] + path[b, i] -> slot start[b] + i for i < count[b], in place and in every cache of the list: tensors [B, heads, S, D] of any type (bf16 keys and
    values, codes and scales of a `Kv4Cache`), rows contiguous, that share no element.  A path ascends (`tree_accept`'s does); rows outside the cache stay."""
    _lib.native().cache_move(caches if isinstance(caches, (list, tuple)) else list(caches), start, path, count)
