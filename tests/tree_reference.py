"""paged_attention_tree's definition in 64 bits, for a step of tests.test_gpu_tree_attention.Trees."""

from __future__ import annotations

import math

import torch


def seen_keys(st, s):
    """(nodes, context + nodes) of sequence s: context, ancestors and itself."""
    c, n = st.ctx[s], st.nodes[s]
    seen = torch.zeros((n, c + n), dtype=torch.bool)
    seen[:, :c] = True
    for i, p in enumerate(st.parents[s]):
        if 0 <= p < i:
            seen[i, c:] = seen[p, c:]
        seen[i, c + i] = True
    return seen


def definition(st, layer=0):
    """Per sequence (its rows, out, sum of weight |v|), (heads, nodes, head_dim) each. A key that a node does not see is no
    part of its sums, whatever its values."""
    got = []
    group = st.hq // st.hkv
    for s, (c, n) in enumerate(zip(st.ctx, st.nodes)):
        if n == 0:
            continue
        seen = seen_keys(st, s)
        pos = torch.arange(c)
        slots = torch.tensor(st.tables[s] + [0])[pos // st.bs] * st.bs + pos % st.bs
        rows = slice(st.cu[s], st.cu[s] + n)
        out, size = (torch.zeros((st.hq, n, st.d), dtype=torch.float64) for _ in range(2))
        for g in range(st.hkv):
            k, v = (torch.cat([pool[layer].flatten(0, 1)[:, g].cpu()[slots], new[0, g, rows].cpu()]).double()
                    for pool, new in ((st.k, st.nk), (st.v, st.nv)))
            q = st.q[0, g * group:(g + 1) * group, rows].double().cpu()
            t = (q @ k.t() * st.scale).masked_fill(~seen, -math.inf)
            w = torch.softmax(t, -1)
            if torch.isfinite(v).all():
                out[g * group:(g + 1) * group], size[g * group:(g + 1) * group] = w @ v, w @ v.abs()
            else:
                for i in range(n):
                    at = seen[i].nonzero()[:, 0]
                    out[g * group:(g + 1) * group, i] = w[:, i, at] @ v[at]
                    size[g * group:(g + 1) * group, i] = w[:, i, at] @ v[at].abs()
        got.append((rows, out, size))
    return got
