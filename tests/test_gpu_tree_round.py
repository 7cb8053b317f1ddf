"""Whole rounds of speculation over trees on the device: slots, attention, sampling, the accepted path and its keys and
values in the pool. Whatever is drafted, a greedy run must emit what plain decoding in 64 bits emits."""

from __future__ import annotations

import random

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels.tree_attention import paged_attention_tree, plan_tree
from memforge_amd.runtime.device_tables import DeviceBlockTables
from memforge_amd.runtime.sampling import sample_tokens
from memforge_amd.speculative import accept_tree

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, VOCAB, BS, WIDTH, BLOCKS = 2, 4, 2, 32, 400, 8, 24, 90
HIDDEN = 64


class Model:
    """Two attention layers over token and position embeddings; ``nodes`` per sequence in a round."""

    def __init__(self, dtype, device):
        gen = torch.Generator().manual_seed(5)

        def w(*s, scale=1.0):
            return (scale * torch.randn(s, generator=gen, dtype=torch.float64)).to(dtype).to(device)

        self.embed, self.place = w(VOCAB, HIDDEN), w(256, HIDDEN)
        self.q, self.k = w(LAYERS, HIDDEN, HQ * D, scale=0.1), w(LAYERS, HIDDEN, HKV * D, scale=0.1)
        self.v, self.o = w(LAYERS, HIDDEN, HKV * D, scale=0.15), w(LAYERS, HQ * D, HIDDEN, scale=0.1)
        self.head = w(HIDDEN, VOCAB, scale=0.3)

    def forward(self, tokens, positions, attend):
        """Logits of rows; ``attend(layer, q, k, v)`` on (rows, heads, dim)."""
        x = self.embed[tokens] + self.place[positions]
        for i in range(LAYERS):
            q, k, v = (torch.matmul(x, m[i]).unflatten(1, (-1, D)) for m in (self.q, self.k, self.v))
            x = x + torch.matmul(attend(i, q, k, v).flatten(1), self.o[i])
        return torch.matmul(x, self.head)


def plain_decode(prompt, count):
    """Greedy tokens after ``prompt`` in 64 bits, each from a pass over everything before it; and the smallest gap to a
    second choice, which a 32-bit run's error must not reach."""
    model = Model(torch.float64, "cpu")

    def attend(_, q, k, v):
        k, v = (x.repeat_interleave(HQ // HKV, 1) for x in (k, v))
        t = torch.einsum("nhd,mhd->hnm", q, k) * D ** -0.5
        mask = torch.ones(t.shape[-2:], dtype=torch.bool).tril()
        return torch.einsum("hnm,mhd->nhd", torch.softmax(t.masked_fill(~mask, -torch.inf), -1), v)

    tokens, gap = list(prompt), 1e9
    for _ in range(count):
        logits = model.forward(torch.tensor(tokens), torch.arange(len(tokens)), attend)[-1]
        top = logits.topk(2).values
        gap = min(gap, float(top[0] - top[1]))
        tokens.append(int(logits.argmax()))
    return tokens[len(prompt):], gap


class Rounds:
    def __init__(self, device, prompts):
        self.device, self.model = device, Model(torch.float32, device)
        b = len(prompts)
        self.state = DeviceBlockTables.allocate(b, WIDTH, BLOCKS, BS, device)
        self.k, self.v = (torch.full((LAYERS, BLOCKS, BS, HKV, D), torch.nan, device=device) for _ in range(2))
        self.root = torch.tensor([p[-1] for p in prompts], device=device)
        # the prompts but for their last tokens, as chains with no context before them
        lens = [len(p) - 1 for p in prompts]
        self.run(torch.tensor([t for p in prompts for t in p[:-1]], device=device),
                 torch.tensor([i - 1 for n in lens for i in range(n)], dtype=torch.int32, device=device), lens, prompt=True)

    def views(self, i):
        return nat.PoolView.from_bshd(self.k[i], self.v[i])

    def run(self, tokens, parents, nodes, prompt=False):
        """One pass over trees; without ``prompt`` their first nodes are the newest tokens. Emitted tokens and counts."""
        device, state = self.device, self.state
        cu = torch.tensor([0] + torch.tensor(nodes).cumsum(0).tolist(), dtype=torch.int32).to(device) \
            if not isinstance(nodes, torch.Tensor) else nodes
        most = self.most if isinstance(nodes, torch.Tensor) else max(nodes)
        plan = plan_tree(parents, cu, state.lens, most, HQ, HKV, D, torch.float32, max_context=WIDTH * BS)
        new = []

        def attend(i, q, k, v):
            new.append((k, v))
            return paged_attention_tree(q.permute(1, 0, 2)[None], self.k, self.v, i, state.tables, plan,
                                        k.permute(1, 0, 2)[None], v.permute(1, 0, 2)[None])[0].permute(1, 0, 2)

        logits = self.model.forward(tokens, plan.positions, attend)
        rows = tokens.shape[0]
        if prompt:
            slots = state.extend(torch.tensor(nodes, dtype=torch.int32).to(device), rows).slot_mapping
            emitted = None
        else:
            targets, _ = sample_tokens(logits, torch.zeros(rows, device=device), temperature=0.0)
            got = accept_tree(tokens, targets, parents, cu, most)
            slots = state.extend(got.count, rows, rows=got.path).slot_mapping
            self.root.copy_(got.tokens.gather(1, (got.count.long() - 1)[:, None])[:, 0])
            emitted = got
        for i, (k, v) in enumerate(new):
            nat.kv_write(k, v, slots, self.views(i))
        return emitted


PROMPTS = [[7, 100, 3, 250], [9, 9], list(range(30, 49)), [1, 2, 3, 4, 5, 6, 7, 8, 9]]


def drafts(rng, wanted, nodes):
    """A tree whose nodes often continue ``wanted`` (what plain decoding says comes after the root)."""
    parents, tokens, depth = [-1], [0], [0]
    for i in range(1, nodes):
        p = rng.randint(max(0, i - 4), i - 1)
        parents.append(p)
        depth.append(depth[p] + 1)
        right = depth[i] - 1 < len(wanted) and rng.random() < 0.6
        tokens.append(wanted[depth[i] - 1] if right else rng.randrange(VOCAB))
    return parents, tokens


@pytest.mark.parametrize("captured", [False, True])
def test_greedy_rounds_emit_plain_decoding(device, captured):
    total = 24
    want = [plain_decode(p, total + 12) for p in PROMPTS]
    assert min(gap for _, gap in want) > 1e-3  # (a 32-bit run is off by less than 1e-4 here)
    want = [w for w, _ in want]
    rng = random.Random(3)
    run = Rounds(device, PROMPTS)
    sizes = [6, 11, 1, 16]
    run.most = max(sizes)
    cu = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32).to(device)
    parents = torch.full((sum(sizes),), -1, dtype=torch.int32, device=device)
    tokens = torch.zeros(sum(sizes), dtype=torch.int64, device=device)

    def round_():
        tokens[cu[:-1].long()] = run.root
        return run.run(tokens, parents, cu)

    got, graph, out = [[] for _ in PROMPTS], None, None
    longest = 0
    while min(map(len, got)) < total:
        trees = [drafts(rng, w[len(g):], n) for w, g, n in zip(want, got, sizes)]
        parents.copy_(torch.tensor([p for t in trees for p in t[0]], dtype=torch.int32))
        tokens.copy_(torch.tensor([x for t in trees for x in t[1]]))
        if captured and graph is None and longest:  # the first round ran eagerly
            state = [x.clone() for x in (run.root, run.state.tables, run.state.lens, run.state.held, run.state.free_count)]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = round_()
            for x, y in zip((run.root, run.state.tables, run.state.lens, run.state.held, run.state.free_count), state):
                assert torch.equal(x, y)  # capture runs nothing
        if graph is not None:
            graph.replay()
        else:
            out = round_()
        torch.cuda.synchronize()
        for g, row, n in zip(got, out.tokens.tolist(), out.count.tolist()):
            g += row[:n]
            longest = max(longest, n)
    assert longest > 2  # drafts were accepted
    for g, w in zip(got, want):
        n = min(len(g), len(w))
        assert g[:n] == w[:n]
    assert run.state.lens.tolist() == [len(p) - 1 + len(g) for p, g in zip(PROMPTS, got)]
    run.state.truncate(torch.zeros(len(PROMPTS), dtype=torch.int32, device=device))
    assert int(run.state.free_count) == BLOCKS and sorted(run.state.free.tolist()) == list(range(BLOCKS))
