"""What a plan says of rows that belong to no tree: their position is 0, whatever the memory held before."""

from __future__ import annotations

import random

import pytest
import torch

from memforge_amd.kernels.tree_attention import plan_tree

pytestmark = pytest.mark.gpu


def ints(device, x):
    return torch.tensor(x, dtype=torch.int32).to(device)


def plan(device, parents, cu, ctx, max_nodes, max_context=4000):
    return plan_tree(ints(device, parents), ints(device, cu), ints(device, ctx), max_nodes, 4, 2, 64, torch.bfloat16,
                     max_context=max_context)


@pytest.fixture
def filled(monkeypatch):
    """New memory holds numbers that are no position."""
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: empty(*a, **k).fill_(0x3f3f3f3f))


def positions(parents, cu, ctx, max_nodes):
    want = [0] * len(parents)
    for s, c in enumerate(ctx):
        n = min(cu[s + 1] - cu[s], max_nodes)
        if n <= 0 or cu[s] < 0 or cu[s] + n > len(parents):
            continue
        depth = []
        for i in range(n):
            p = parents[cu[s] + i]
            depth.append(depth[p] + 1 if 0 <= p < i else 0)
            want[cu[s] + i] = c + depth[i]
    return want


@pytest.mark.parametrize("cu,rows,max_nodes", [
    ([0, 3, 5], 9, 4),             # rows behind the trees
    ([0, 3, 9], 9, 4),             # nodes past max_nodes
    ([4, 6, 9], 9, 4),             # rows before them
    ([0, 3, 900], 9, 8),           # a tree that does not lie within the rows
    ([-2, 3, 6], 9, 8),            # nor does this
    ([0, 0, 0], 9, 4), ([9, 9, 9], 9, 4), ([0, 600, 1300], 5000, 512), ([0, 10, 30, 0, 0, 0], 90, 16)])
def test_rows_of_no_tree_have_position_0(device, filled, cu, rows, max_nodes):
    rng = random.Random(rows)
    parents = [rng.randint(-1, 3) for _ in range(rows)]
    ctx = [rng.randint(0, 300) for _ in cu[1:]]
    assert plan(device, parents, cu, ctx, max_nodes).positions.tolist() == positions(parents, cu, ctx, max_nodes)


@pytest.mark.parametrize("rows", [1, 77, 300000])
def test_no_sequences(device, filled, rows):
    assert not plan(device, [0] * rows, [0], [], 4).positions.any()


def test_many_sequences(device, filled):
    rng = random.Random(1)
    cu = [3]
    for _ in range(700):
        cu.append(cu[-1] + rng.choice([0, 1, 5, 9]))
    rows = cu[-1] + 1000
    parents, ctx = [rng.randint(-1, 4) for _ in range(rows)], [rng.randint(0, 300) for _ in cu[1:]]
    assert plan(device, parents, cu, ctx, 6).positions.tolist() == positions(parents, cu, ctx, 6)


def test_replays_whose_trees_shrink(device):
    parents, ctx = [-1] + [0] * 39, [10, 20]
    tensors = ints(device, parents), ints(device, [0, 30, 40]), ints(device, ctx)
    call = lambda: plan_tree(*tensors, 30, 4, 2, 64, torch.bfloat16, max_context=100)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for cu in ([0, 30, 40], [0, 7, 9], [0, 0, 30], [0, 1, 1]):
        tensors[1].copy_(ints(device, cu))
        graph.replay()
        torch.cuda.synchronize()
        assert got.positions.tolist() == positions(parents, cu, ctx, 30)
