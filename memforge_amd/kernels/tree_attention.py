"""Attention for trees of drafted tokens over the paged cache.

A verify pass of a chain attends causally (``paged_attention_varlen``); where a draft
branches, a node must not see its siblings. Here every node sees its sequence's
context in the pool, itself and its ancestors, all of them in flight: nothing is
written to the pool before a path is accepted (``speculative.accept_tree``). Lengths
and trees are device tensors, and the work is split over the GPU there, so a step
needs no copy to the host and a captured one serves every length up to its
``max_context``."""

from __future__ import annotations

import math
from typing import Optional

import torch

from memforge_amd import _native as nat

TreePlan = nat.TreePlan


def plan_tree(parents: torch.Tensor, cu_nodes: torch.Tensor, context_lens: torch.Tensor, max_nodes: int, num_q_heads: int,
              num_kv_heads: int, head_dim: int, dtype: torch.dtype, max_context: int) -> TreePlan:
    """A step's trees, for every layer's ``paged_attention_tree`` (one launch).

    Rows ``cu_nodes[s] .. cu_nodes[s + 1] - 1`` (int32, B + 1) are sequence s's nodes, at
    most ``max_nodes`` (up to 1024; further rows take no part); ``parents`` (int32 per row)
    their parents' numbers in the tree, each smaller than the node's own, -1 for none; and
    ``context_lens`` (int32, B) the tokens it has in the pool, taken as at most
    ``max_context``. All are read here and not by the attention: a step with other
    lengths or trees has a plan of its own. ``positions`` of the plan (int64 per row) are
    the nodes' positions, context length plus ancestors, as rotary embeddings take them."""
    return nat.tree_plan(parents, cu_nodes, context_lens, max_nodes, max_context, num_q_heads, num_kv_heads, head_dim, dtype)


def paged_attention_tree(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, layer_idx: int,
                         block_tables: torch.Tensor, plan: TreePlan, new_keys: torch.Tensor, new_values: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """Attention of every node of a step's trees, ``(1, heads, rows, head_dim)`` in and out.

    Pools are ``(layers, blocks, slots, kv_heads, head_dim)``; ``block_tables`` int32
    (B, width) on the device, a row for each sequence of the plan, wide enough for its
    ``max_context``; ``new_keys`` / ``new_values`` ``(1, kv_heads, rows, head_dim)`` the
    nodes' own. fp32, fp16 or bf16 throughout, head_dim 32, 64, 128 or 256. Rows that
    belong to no tree are not computed and hold anything. A value that is not finite
    reaches the nodes of its tree that do not see it too, as zero times it does in a
    product."""
    nat.require_device(query, key_pool, new_keys, new_values)
    for name, x in (("query", query), ("new_keys", new_keys), ("new_values", new_values)):
        if x.dim() != 4 or x.shape[0] != 1:
            raise ValueError(f"{name} must be (1, heads, rows, head_dim), got {tuple(x.shape)}")
    if key_pool.dim() != 5 or key_pool.shape != value_pool.shape or key_pool.stride() != value_pool.stride() \
            or key_pool.dtype != value_pool.dtype or key_pool.stride(4) != 1 or value_pool.device != key_pool.device:
        raise ValueError("K and V pools must be (layers, blocks, slots, kv_heads, head_dim) of one shape, layout, dtype and "
                         f"device, got {tuple(key_pool.shape)} in {key_pool.dtype} and {tuple(value_pool.shape)} in "
                         f"{value_pool.dtype}")
    layers, blocks, block_size, kv_heads, dim = key_pool.shape
    if not -layers <= layer_idx < layers:
        raise IndexError(f"layer {layer_idx} of pools of {layers}")
    query, new_keys, new_values = _whole_pieces(query), _whole_pieces(new_keys), _whole_pieces(new_values)
    if new_keys.stride() != new_values.stride():
        new_keys, new_values = new_keys.contiguous(), new_values.contiguous()
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    stride = key_pool.stride()
    at = (layer_idx % layers) * stride[0] * key_pool.element_size()
    nat.tree_attention_at(
        nat._tree_rows("query", query, plan.num_q_heads, plan, 2, 1), nat._tree_rows("out", out, plan.num_q_heads, plan, 2, 1),
        (key_pool.data_ptr() + at, value_pool.data_ptr() + at, stride[1], stride[2], stride[3], block_size, blocks),
        (kv_heads, dim), key_pool.dtype, key_pool.device, block_tables, plan,
        nat._tree_rows("new_keys", new_keys, plan.num_kv_heads, plan, 2, 1),
        nat._tree_rows("new_values", new_values, plan.num_kv_heads, plan, 2, 1)[0],
        float(scale) if scale is not None else 1.0 / math.sqrt(dim))
    return out


def _whole_pieces(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself where its rows and heads begin at whole 16 bytes (as the kernel reads them), else a copy."""
    stride, per = x.stride(), 16 // x.element_size() if x.element_size() < 16 else 1
    if stride[3] == 1 and not (stride[1] % per or stride[2] % per or x.data_ptr() & 15):
        return x
    return x.contiguous()
