"""Rounds over draft trees that run out of blocks: a refused request emits nothing and keeps its newest token, and goes on
where it was once others have given their blocks back."""

from __future__ import annotations

import random

import torch
import pytest

from memforge_amd import _native as nat
from memforge_amd.kernels.tree_attention import paged_attention_tree, plan_tree
from memforge_amd.runtime.sampling import sample_tokens
from memforge_amd.speculative import accept_tree
from tests import test_gpu_tree_round as base

pytestmark = pytest.mark.gpu


def round_(run, tokens, parents, cu, most):
    """One round; (accepted path, tokens of it that count, refused requests)."""
    state, new = run.state, []
    plan = plan_tree(parents, cu, state.lens, most, base.HQ, base.HKV, base.D, torch.float32, max_context=base.WIDTH * base.BS)

    def attend(i, q, k, v):
        new.append((k, v))
        return paged_attention_tree(q.permute(1, 0, 2)[None], run.k, run.v, i, state.tables, plan, k.permute(1, 0, 2)[None],
                                    v.permute(1, 0, 2)[None])[0].permute(1, 0, 2)

    logits = run.model.forward(tokens, plan.positions, attend)
    rows = tokens.shape[0]
    targets, _ = sample_tokens(logits, torch.zeros(rows, device=run.device), temperature=0.0)
    got = accept_tree(tokens, targets, parents, cu, most)
    before = state.lens.clone()
    grown = state.extend(got.count, rows, rows=got.path)
    emitted = grown.kv_lens - before
    last = got.tokens.gather(1, (emitted.long() - 1).clamp_min(0)[:, None])[:, 0]
    run.root = torch.where(emitted > 0, last, run.root)
    for i, (k, v) in enumerate(new):
        nat.kv_write(k, v, grown.slot_mapping, run.views(i))
    return got, emitted, grown.refused


def test_greedy_rounds_out_of_blocks(device, monkeypatch):
    total, blocks, sizes = 24, 12, [6, 11, 1, 16]
    monkeypatch.setattr(base, "BLOCKS", blocks)
    want = [base.plain_decode(p, total + 12)[0] for p in base.PROMPTS]
    rng, run = random.Random(2), base.Rounds(device, base.PROMPTS)
    n = len(sizes)
    got, done, refused, rounds = [[] for _ in range(n)], [False] * n, 0, 0
    while not all(done):
        rounds += 1
        assert rounds < 100
        trees = [([], []) if done[s] else base.drafts(rng, want[s][len(got[s]):], sizes[s]) for s in range(n)]
        cu = torch.tensor([0] + torch.tensor([len(t[0]) for t in trees]).cumsum(0).tolist(), dtype=torch.int32).to(device)
        parents = torch.tensor([p for t in trees for p in t[0]], dtype=torch.int32).to(device)
        tokens = torch.tensor([x for t in trees for x in t[1]]).to(device)
        live = torch.tensor([s for s in range(n) if not done[s]]).to(device)
        tokens[cu[live].long()] = run.root[live]
        lens = run.state.lens.tolist()
        path, emitted, left_out = round_(run, tokens, parents, cu, max(sizes))
        counts, emitted = path.count.tolist(), emitted.tolist()
        assert all(e in (0, c) for e, c in zip(emitted, counts))
        assert int(left_out) == sum(e < c for e, c in zip(emitted, counts))
        assert run.state.lens.tolist() == [x + e for x, e in zip(lens, emitted)]
        refused += int(left_out)
        ends = [2**31 - 1] * n
        for s in range(n):
            got[s] += path.tokens[s, :emitted[s]].tolist()
            if not done[s] and len(got[s]) >= total:
                done[s], ends[s] = True, 0
        run.state.truncate(torch.tensor(ends, dtype=torch.int32).to(device))
    assert refused > 0
    for g, w in zip(got, want):
        m = min(len(g), len(w))
        assert m >= total and g[:m] == w[:m]
    assert int(run.state.free_count) == blocks and sorted(run.state.free.tolist()) == list(range(blocks))
