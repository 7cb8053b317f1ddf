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
    the nodes' positions, context length plus ancestors, as rotary embeddings take them, and 0
    at rows that belong to no tree."""
    return nat.tree_plan(parents, cu_nodes, context_lens, max_nodes, max_context, num_q_heads, num_kv_heads, head_dim, dtype)


def paged_attention_tree(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, layer_idx: int,
                         block_tables: torch.Tensor, plan: TreePlan, new_keys: torch.Tensor, new_values: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """Attention of every node of a step's trees, ``(1, heads, rows, head_dim)`` in and out.

    Pools are ``(layers, blocks, slots, kv_heads, head_dim)``; ``block_tables`` int32
    (B, width) on the device, a row for each sequence of the plan, wide enough for its
    ``max_context``; ``new_keys`` / ``new_values`` ``(1, kv_heads, rows, head_dim)`` the
    nodes' own. fp32, fp16 or bf16 throughout, head_dim 32, 64, 128 or 256. Rows that
    belong to no tree are not computed and hold anything. An infinity or NaN in a row
    reaches the nodes that see it and no others."""
    nat.require_device(query, key_pool, new_keys, new_values)
    shape, stride = key_pool.shape, key_pool.stride()
    if len(shape) != 5 or shape != value_pool.shape or stride != value_pool.stride() or key_pool.dtype is not value_pool.dtype \
            or stride[4] != 1 or key_pool.device != value_pool.device:
        raise ValueError("K and V pools must be (layers, blocks, slots, kv_heads, head_dim) of one shape, layout, dtype and "
                         f"device, got {tuple(shape)} in {key_pool.dtype} and {tuple(value_pool.shape)} in {value_pool.dtype}")
    layers, blocks, block_size, kv_heads, dim = shape
    nat.check_tree_pool(key_pool, kv_heads, dim, plan)
    if not -layers <= layer_idx < layers:
        raise IndexError(f"layer {layer_idx} of pools of {layers}")
    q, q_rows = _rows("query", query, plan.num_q_heads, plan)
    k, k_rows = _rows("new_keys", new_keys, plan.num_kv_heads, plan)
    v, v_rows = _rows("new_values", new_values, plan.num_kv_heads, plan)
    if k[1:] != v[1:]:
        k, k_rows = _rows("new_keys", new_keys, plan.num_kv_heads, plan, copy=True)
        v, v_rows = _rows("new_values", new_values, plan.num_kv_heads, plan, copy=True)
    out = torch.empty((1, plan.num_q_heads, plan.num_rows, dim), dtype=plan.dtype, device=plan.device)
    at = (layer_idx % layers) * stride[0] * key_pool.element_size()
    nat.tree_attention_at(q, (out.data_ptr(), dim, plan.num_rows * dim),
                          (key_pool.data_ptr() + at, value_pool.data_ptr() + at, stride[1], stride[2], stride[3], block_size,
                           blocks), block_tables, plan, k, v[0], float(scale) if scale is not None else 1.0 / math.sqrt(dim))
    return out


def _rows(name: str, x: torch.Tensor, heads: int, plan: TreePlan, copy: bool = False):
    """((address, row stride, head stride), what has to live until the launch) of ``(1, heads, rows, head_dim)``: of a
    copy where rows or heads do not begin at whole 16 bytes, as the kernel reads them. The stride of an axis of length
    one addresses nothing, may be any number, and is given as 0."""
    if x.shape != (1, heads, plan.num_rows, plan.head_dim) or x.dtype is not plan.dtype or x.device != plan.device:
        raise ValueError(f"{name} must be {(1, heads, plan.num_rows, plan.head_dim)} in {plan.dtype} on {plan.device}, got "
                         f"{tuple(x.shape)} in {x.dtype} on {x.device}")
    _, head, row, last = x.stride()
    at, dim = x.data_ptr(), plan.head_dim
    per = 4 if plan.dtype is torch.float32 else 8
    if copy or last != 1 or (head % per and heads > 1) or (row % per and plan.num_rows > 1) or at & 15:
        x = torch.empty((heads, plan.num_rows, dim), dtype=plan.dtype, device=plan.device).copy_(x[0])
        at, head, row = x.data_ptr(), plan.num_rows * dim, dim
    return (at, row if plan.num_rows > 1 else 0, head if heads > 1 else 0), x
