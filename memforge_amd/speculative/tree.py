"""Which path of a tree of drafted tokens a target accepts.

The target's token is drawn at every node beforehand (``runtime.sampling.sample_tokens``
on the nodes' logits); the accepted path then follows, from the tree's first node,
the drafted child whose token was drawn. Every emitted token is a draw from the
target's own distribution after the tokens before it, whatever was drafted: the
drafts only decide how many come out of one pass. The chain form with draft
probabilities is ``RejectionSampler`` (the reference's
memforge_ml/speculative/rejection_sampler.py:28-83)."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from memforge_amd import _native as nat


@dataclass
class AcceptedPath:
    """Per sequence: ``path`` (int32 (B, max_nodes)) the rows of the accepted nodes, node 0
    first, -1 past the end; ``tokens`` (int64 alike) the tokens the round emits, the
    target's at each of them; ``count`` (int32 (B)) how many."""

    path: torch.Tensor
    tokens: torch.Tensor
    count: torch.Tensor


def accept_tree(tokens: torch.Tensor, targets: torch.Tensor, parents: torch.Tensor, cu_nodes: torch.Tensor,
                max_nodes: int) -> AcceptedPath:
    """The accepted path of every sequence's tree (mf_tree_accept, one launch).

    Rows ``cu_nodes[s] .. cu_nodes[s + 1] - 1`` are sequence s's nodes: row r's token
    ``tokens[r]``, its parent's number in the tree ``parents[r]`` (int32, smaller than
    its own; -1 for none), and the token that the target drew there ``targets[r]``
    (int64). Node 0 is the sequence's newest token; of several children with the drawn
    token the first counts. ``max_nodes``: at least the largest tree's nodes (further
    ones are ignored), at most 1024. ``path`` and ``count`` are what
    ``DeviceBlockTables.extend`` takes to place the accepted rows; a request that it refuses has
    no place for them, and its tokens of this round do not count."""
    return AcceptedPath(*nat.tree_accept(tokens, targets, parents, cu_nodes, max_nodes))
