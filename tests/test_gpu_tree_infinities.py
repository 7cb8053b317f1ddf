"""Infinities and NaN in rows of a tree: who sees the row gets them, who does not is as near to 64 bits as ever."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_tree_attention import Trees
from tests.tree_reference import definition

pytestmark = pytest.mark.gpu


def check(st, out, exact_kind=True):
    """As Trees.check, at what is finite in 64 bits; elsewhere the same infinity or NaN."""
    eps = torch.finfo(st.dtype).eps
    k_most = max(float(x[torch.isfinite(x)].abs().max()) for x in (st.k, st.nk))
    for rows, want, size in definition(st):
        got = out[0, :, rows].double().cpu()
        fine = torch.isfinite(want)
        assert (torch.isfinite(got) == fine).all()
        if exact_kind:
            assert torch.equal(got[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0))
        # scores of at most top: their sum over head_dim in 32 bits; the exponential's argument; sums over the keys
        top = float(st.q.abs().max()) * k_most * st.d * abs(st.scale)
        off = top * 2.0 ** -24 + 2.0 ** -21 + (max(st.ctx) + max(st.nodes)) * 2.0 ** -24
        tol = eps / 2 * want.abs() + size * (2 * off + (eps / 2 if eps > 1e-6 else 0.0)) * 1.01 + 1e-30
        assert ((got - want).abs()[fine] <= tol[fine]).all()
    return out


def branch(st, s, node):
    """A row of the call, by sequence and node."""
    return st.cu[s] + node


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 32), (15, 5, 64), (10, 2, 128), (6, 1, 256)])
@pytest.mark.parametrize("ctx,nodes", [([0], [3]), ([37, 64], [8, 40]), ([3000, 5], [24, 200]), ([96, 31], [33, 1])])
def test_values_of_a_branch(device, dtype, hq, hkv, d, ctx, nodes):
    st = Trees(device, dtype, hq, hkv, d, 16, ctx, nodes, seed=d + sum(ctx))
    n = nodes[0]
    st.nv[0, :, branch(st, 0, n - 1), 3] = math.inf
    st.nv[0, 0, branch(st, 0, n // 2)] = math.nan
    if len(nodes) > 1:
        st.nv[0, :, branch(st, 1, nodes[1] // 2), d - 1] = -math.inf
        st.nv[0, :, branch(st, 1, nodes[1] - 1), :7] = math.inf
    check(st, st.run())


@pytest.mark.parametrize("dtype", DTYPES)
def test_both_infinities_on_one_path_are_nan(device, dtype):
    st = Trees(device, dtype, 4, 2, 64, 16, [50], [6], seed=3)
    st.parents = [[-1, 0, 0, 1, 2, 4]]
    st.parents_t.copy_(torch.tensor(st.parents[0], dtype=torch.int32))
    st.nv[0, :, 1, 5], st.nv[0, :, 3, 5], st.nv[0, :, 2, 5], st.nv[0, :, 4, 6] = math.inf, -math.inf, -math.inf, math.nan
    out = check(st, st.run())[0, 0].float().cpu()
    assert out[1, 5] == math.inf and out[3, 5].isnan() and out[2, 5] == -math.inf and out[5, 6].isnan() and out[0].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_keys_of_a_branch(device, dtype, value):
    """A key that is not finite: only what sees it is not."""
    st = Trees(device, dtype, 4, 2, 64, 16, [50, 700], [9, 20], seed=4)
    for row in (branch(st, 0, 5), branch(st, 1, 19)):
        st.nk[0, :, row, 7] = value
    got = st.run()
    for x in (st.nk,):  # the nodes that see such a key are left out
        bad = ~torch.isfinite(x[0, 0]).all(-1).cpu()
    clean = st.nk.clone()
    for s in range(2):
        for i, p in enumerate(st.parents[s]):
            at = branch(st, s, i)
            if 0 <= p < i and bad[branch(st, s, p)]:
                bad[at] = True
    st.nk = torch.where(torch.isfinite(clean), clean, torch.zeros_like(clean))
    got[0][:, bad.to(device)] = st.run()[0][:, bad.to(device)]
    check(st, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx", [1, 33, 64, 2500])
def test_the_last_keys_of_a_context(device, dtype, ctx):
    """Every node sees them; rows past the end are no part of it."""
    st = Trees(device, dtype, 4, 2, 64, 16, [ctx], [7], seed=5)
    block, slot = st.tables[0][(ctx - 1) // 16], (ctx - 1) % 16
    st.v[0, block, slot, :, 2] = math.inf
    if slot < 15:
        st.v[0, block, slot + 1:] = math.nan
        st.k[0, block, slot + 1:] = math.nan
    check(st, st.run(), exact_kind=dtype is not torch.float16)


def test_many_wild_rows_of_the_largest_trees(device):
    st = Trees(device, torch.bfloat16, 6, 2, 32, 16, [70, 0], [1024, 1000], seed=8)
    for s in range(2):
        for i in range(500, st.nodes[s], 3):
            st.nv[0, :, branch(st, s, i), i % 32] = (math.inf, -math.inf, math.nan)[i % 7 % 3]
    check(st, st.run())


def test_replays(device):
    st = Trees(device, torch.bfloat16, 10, 2, 128, 16, [900, 33], [16, 5], seed=6)
    st.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = st.run()
    keep = st.nv.clone()
    for value in (math.inf, 1.0, math.nan, -math.inf):
        st.nv.copy_(keep)
        st.nv[0, :, 9] = value
        st.nv[0, :, 18, 3] = value
        graph.replay()
        torch.cuda.synchronize()
        check(st, out)
