"""paged_attention_tree against its definition in 64 bits."""

from __future__ import annotations

import math
import random

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels.tree_attention import paged_attention_tree, plan_tree

pytestmark = pytest.mark.gpu


def ints(device, x):
    return torch.tensor(x, dtype=torch.int32).to(device)


class Trees:
    """One step: contexts in shuffled blocks, trees in flight, and what must come out."""

    def __init__(self, device, dtype, hq, hkv, d, bs, ctx, nodes, seed=0, layers=1, shape="random", spare=0, scale=None):
        gen = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.device, self.dtype, self.hq, self.hkv, self.d, self.bs = device, dtype, hq, hkv, d, bs
        self.ctx, self.nodes, self.spare = list(ctx), list(nodes), spare
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        need = [-(-c // bs) for c in ctx]
        self.blocks = sum(need) + 3
        perm = torch.randperm(self.blocks, generator=gen).tolist()
        self.width = max(max(need, default=0), 1) + 1
        self.tables, at = [], 0
        for n in need:
            self.tables.append(perm[at:at + n])
            at += n
        self.parents = []
        for n in nodes:
            self.parents.append([{"random": rng.randint(max(-1, i - 9), i - 1), "chain": i - 1, "star": 0 if i else -1,
                                  "forest": -1}[shape] if i else -1 for i in range(n)])
        rows = sum(nodes) + spare
        self.rows = rows

        def values(*s):
            return torch.randn(s, generator=gen).to(device, dtype)

        self.k, self.v = values(layers, self.blocks, bs, hkv, d), values(layers, self.blocks, bs, hkv, d)
        self.q = (values(rows, hq, d) * 2).permute(1, 0, 2)[None]
        self.nk, self.nv = values(rows, hkv, d).permute(1, 0, 2)[None], values(rows, hkv, d).permute(1, 0, 2)[None]
        cu = [0]
        for n in nodes:
            cu.append(cu[-1] + n)
        self.cu = cu
        self.cu_t, self.ctx_t = ints(device, cu), ints(device, ctx)
        self.parents_t = ints(device, [p for t in self.parents for p in t] + [0] * spare)
        table = torch.zeros((len(ctx), self.width), dtype=torch.int32)
        for row, t in zip(table, self.tables):
            row[:len(t)] = torch.tensor(t, dtype=torch.int32)
        self.table = table.to(device)

    def plan(self, max_nodes=None, max_context=None):
        return plan_tree(self.parents_t, self.cu_t, self.ctx_t, max_nodes or max(self.nodes), self.hq, self.hkv, self.d,
                         self.dtype, max_context=max(self.ctx) if max_context is None else max_context)

    def run(self, plan=None, layer=0):
        return paged_attention_tree(self.q, self.k, self.v, layer, self.table, plan or self.plan(), self.nk, self.nv,
                                    scale=self.scale)

    def check(self, out, layer=0, most=None, what=""):
        """Every row against 64 bits, within what the roundings can do: half a step of the type at the end, and for each
        weight half a step (16 bits), its score's fp32 sum and the exponential's argument and result."""
        eps = torch.finfo(self.dtype).eps
        group = self.hq // self.hkv
        for s, (c, n) in enumerate(zip(self.ctx, self.nodes)):
            n = min(n, most or n)
            if n == 0:
                continue
            seen = torch.zeros((n, c + n), dtype=torch.bool)
            seen[:, :c] = True
            for i, p in enumerate(self.parents[s][:n]):
                if 0 <= p < i:
                    seen[i, c:] = seen[p, c:]
                seen[i, c + i] = True
            pos = torch.arange(c)
            slots = torch.tensor(self.tables[s] + [0])[pos // self.bs] * self.bs + pos % self.bs
            rows = slice(self.cu[s], self.cu[s] + n)
            for h in range(self.hq):
                g = h // group
                k, v = (torch.cat([pool[layer].flatten(0, 1)[:, g].cpu()[slots], new[0, g, rows].cpu()]).double()
                        for pool, new in ((self.k, self.nk), (self.v, self.nv)))
                q = self.q[0, h, rows].double().cpu()
                t = (q @ k.t() * self.scale).masked_fill(~seen, -math.inf)
                w = torch.softmax(t, -1)
                want = w @ v
                size = w @ v.abs()
                top = (q.abs() @ k.abs().t() * abs(self.scale)).amax(-1, keepdim=True)
                off = top * self.d * 2.0 ** -24 + 2.0 ** -21 + (c + n) * 2.0 ** -24
                tol = eps / 2 * want.abs() + size * (2 * off + (eps / 2 if eps > 1e-6 else 0.0)) * 1.01 + 1e-30
                got = out[0, h, rows].double().cpu()
                bad = (got - want).abs() > tol
                assert not bad.any() and torch.isfinite(got).all(), (
                    what, s, h, float((got - want).abs().max()), float(tol.max()), bad.nonzero()[:3].tolist())


SHAPES = [(15, 5, 64), (9, 3, 64), (40, 8, 128), (8, 8, 32), (6, 1, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("ctx,nodes", [([0], [1]), ([5], [3]), ([33, 0, 700], [8, 8, 8]), ([64, 31, 32], [1, 33, 13]),
                                       ([200, 1500], [64, 20]), ([40, 90], [70, 129])])
def test_against_64_bits(device, dtype, hq, hkv, d, ctx, nodes):
    st = Trees(device, dtype, hq, hkv, d, 16, ctx, nodes, seed=sum(ctx) + d)
    st.check(st.run())


@pytest.mark.parametrize("bs", [1, 3, 8, 16, 48, 64, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_block_sizes(device, dtype, bs):
    st = Trees(device, dtype, 10, 2, 64, bs, [2500, 7, 96], [5, 9, 1], seed=bs)
    st.check(st.run())


@pytest.mark.parametrize("shape", ["chain", "star", "forest", "random"])
def test_kinds_of_trees(device, shape):
    st = Trees(device, torch.bfloat16, 4, 2, 64, 16, [100, 0, 50], [40, 40, 1], seed=2, shape=shape)
    plan = st.plan()
    st.check(st.run(plan))
    depth = []
    for c, tree in zip(st.ctx, st.parents):
        up = []
        for p in tree:
            up.append(0 if p < 0 else up[p] + 1)
        depth += [c + x for x in up]
    assert plan.positions.tolist() == depth


@pytest.mark.parametrize("shape", ["chain", "random"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_largest_trees(device, dtype, shape):
    st = Trees(device, dtype, 6, 2, 32, 16, [70, 0, 33], [1024, 1, 1000], seed=8, shape=shape)
    st.check(st.run())


def test_plans_wider_than_their_trees(device):
    """Trees of up to 1024 nodes are allowed for, few come: most groups of columns are empty."""
    st = Trees(device, torch.bfloat16, 15, 5, 64, 16, [700, 31, 0, 64], [8, 1, 30, 90], seed=9)
    st.check(st.run(st.plan(max_nodes=1024, max_context=st.width * 16)))


@pytest.mark.parametrize("nodes", [1, 4, 17, 48])
def test_one_long_context(device, nodes):
    """Cut over every workgroup, merged from many pieces."""
    st = Trees(device, torch.float16, 10, 2, 128, 16, [30001], [nodes], seed=nodes)
    st.check(st.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_sequences_of_uneven_lengths(device, dtype):
    rng = random.Random(4)
    ctx = [rng.choice([0, 1, rng.randint(0, 300), rng.randint(0, 2000)]) for _ in range(70)]
    nodes = [rng.choice([0, 1, rng.randint(1, 12)]) for _ in range(70)]
    st = Trees(device, dtype, 6, 2, 64, 16, ctx, nodes, seed=4)
    st.check(st.run())


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_scales(device, scale):
    st = Trees(device, torch.bfloat16, 4, 2, 64, 16, [77, 300], [9, 16], seed=8, scale=scale)
    st.check(st.run())


def test_rows_of_no_tree_stay_as_they_were(device):
    st = Trees(device, torch.bfloat16, 4, 2, 64, 16, [77, 30, 10], [9, 16, 12], seed=8, spare=5)
    plan = st.plan(max_nodes=12)  # further nodes take no part
    out = torch.full((st.rows, 4, 64), 7.0, dtype=st.dtype, device=device)
    nat.tree_attention(st.q[0].permute(1, 0, 2), out, nat.PoolView.from_bshd(st.k[0], st.v[0]), st.table, plan,
                       st.nk[0].permute(1, 0, 2), st.nv[0].permute(1, 0, 2), st.scale)
    st.check(out.permute(1, 0, 2)[None], most=12)
    assert (out[9 + 12:9 + 16] == 7).all() and (out[sum(st.nodes):] == 7).all()


def test_unseen_keys_of_any_size(device):
    """Scores of siblings far above the seen ones, and slots behind a context that hold NaN."""
    st = Trees(device, torch.bfloat16, 4, 2, 64, 16, [37, 5], [24, 7], seed=3, shape="star")
    st.nk[0, :, 5] = st.q[0, ::2, 3] * 50
    for pool in (st.k, st.v):
        for t, c in zip(st.tables, st.ctx):
            pool[0, t[-1], (c - 1) % 16 + 1:] = math.nan
    st.check(st.run())


def test_malformed_parents_and_lengths(device):
    """A parent that is not an earlier node is none; a tree outside the rows has no nodes; lengths are bounded."""
    st = Trees(device, torch.bfloat16, 4, 2, 64, 16, [40, 20], [6, 5], seed=1)
    st.parents[0] = [-1, 0, 1, 1, 0, 2]
    bad = [3, 0, 1, 1, 0, 2]
    st.parents_t = ints(device, bad + st.parents[1])
    st.check(st.run())
    st.parents_t = ints(device, [-9, 0, 1, 1, 0, 2] + st.parents[1])
    st.check(st.run())
    wild = plan_tree(st.parents_t, ints(device, [0, 6, 900]), ints(device, [40, 2**31 - 1]), 6, 4, 2, 64, st.dtype, max_context=40)
    out = st.run(wild)
    st.nodes = [6, 0]
    st.check(out)


def test_strides_and_layers(device):
    """Heads-major rows, rows of a fused projection, and a layer of its own."""
    st = Trees(device, torch.bfloat16, 6, 2, 64, 16, [333, 20], [13, 4], seed=6, layers=3)
    plan = st.plan()
    st.check(st.run(plan, layer=2), layer=2)
    packed = torch.cat([x[0].permute(1, 0, 2).flatten(1) for x in (st.q, st.nk, st.nv)], 1)
    q, k, v = packed.split((6 * 64, 2 * 64, 2 * 64), 1)
    st.q, st.nk, st.nv = (x.unflatten(1, (-1, 64)).permute(1, 0, 2)[None] for x in (q, k, v))
    st.check(st.run(plan))
    st.q, st.nk, st.nv = st.q.contiguous(), st.nk.contiguous(), st.nv.clone()
    st.check(st.run(plan))
    odd = torch.zeros((6, st.rows, 65), dtype=st.dtype, device=device)  # rows that are not whole 16 bytes
    odd[:, :, 1:] = st.q[0]
    st.q = odd[None, :, :, 1:]
    st.check(st.run(plan))


def test_captured_steps_follow_lengths_and_trees(device):
    """Two graphs with plans of their own, replayed after lengths, trees and rows changed, between eager calls."""
    cases = [Trees(device, torch.bfloat16, 10, 2, 64, 16, [900, 900], [16, 16], seed=1),
             Trees(device, torch.bfloat16, 10, 2, 64, 16, [5000], [16], seed=2)]
    graphs, outs = [], []
    for st in cases:
        st.run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = st.plan()
            outs.append([st.run(plan), st.run(plan)])
        graphs.append(graph)
    rng = random.Random(3)
    for step in range(4):
        for st, graph, out in zip(cases, graphs, outs):
            st.ctx = [rng.randint(0, c) for c in ([900, 900] if len(st.ctx) == 2 else [5000])]
            st.ctx_t.copy_(ints(device, st.ctx))
            st.parents = [[-1] + [rng.randint(0, i - 1) for i in range(1, n)] for n in st.nodes]
            st.parents_t.copy_(ints(device, [p for t in st.parents for p in t]))
            st.q.copy_(torch.randn(st.q.shape, generator=torch.Generator().manual_seed(step)).to(device, st.dtype))
            graph.replay()
            torch.cuda.synchronize()
            st.check(out[0], what="replay")
            st.check(out[1], what="replay")
            st.check(st.run(), what="eager")


def test_on_another_stream(device):
    st = Trees(device, torch.bfloat16, 10, 2, 128, 16, [4000, 100], [16, 3], seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = st.run()
    main = st.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, main)
    st.check(out)


def test_no_sequences(device):
    plan = plan_tree(ints(device, []), ints(device, [0]), ints(device, []), 4, 4, 2, 64, torch.bfloat16, max_context=0)
    q = torch.empty((1, 4, 0, 64), dtype=torch.bfloat16, device=device)
    kv = torch.empty((1, 2, 0, 64), dtype=torch.bfloat16, device=device)
    pool = torch.zeros((1, 2, 16, 2, 64), dtype=torch.bfloat16, device=device)
    assert paged_attention_tree(q, pool, pool, 0, torch.zeros((0, 1), dtype=torch.int32, device=device), plan, kv, kv).shape == q.shape
