"""How near paged_attention_tree comes to 64 bits: the small weights of fp16, and errors in the norm of a head's output."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_tree_attention import Trees
from tests.tree_reference import definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,nodes", [(64, 1), (64, 20), (128, 48), (256, 2)])
@pytest.mark.parametrize("sink", [0, 17000, 31999, "node"])
def test_a_flat_tail_far_below_one_key(device, dtype, d, nodes, sink):
    """One key that holds nearly all the mass and has values 0: what comes out is the tail of 32,000 keys, each 2^-25.6 of
    it, and has to come out: all within half a step, and fp16's within keys * 2^-35 of the sum besides (at most keys
    half steps of 2^-24, where the largest weight is 2^10 or more)."""
    st = Trees(device, dtype, 4, 2, d, 16, [32000], [nodes], seed=1, scale=0.125, shape="star")
    st.q.zero_()
    st.q[..., 0] = 8.0
    for x in (st.k, st.nk):
        x.zero_()
        x[..., 0] = -8.875
    if sink == "node":  # node 0, an ancestor of all
        st.nk[0, :, 0, 0], st.nv[0, :, 0] = 8.875, 0.0
    else:
        block, slot = st.tables[0][sink // 16], sink % 16
        st.k[0, block, slot, :, 0], st.v[0, block, slot] = 8.875, 0.0
    st.v.abs_()
    st.nv.abs_()
    got = st.run()
    (rows, want, size), = definition(st)
    eps = torch.finfo(dtype).eps
    # a weight: half a step; scores exact but for roundings of 26 log2 units to 32 bits, in the product, the sum with the
    # maximum and the exponential (3 * 26 * 2^-24 < 2^-17); sums of 32,020 terms in 32 bits
    rel = (eps / 2 if eps > 1e-6 else 0.0) + 2.0 ** -17 + 32020 * 2.0 ** -24
    tol = eps / 2 * want.abs() + 1.01 * rel * size + 32020 * 2.0 ** -35 * float(st.v.max()) + 2.0 ** -25
    err = (got[0, :, rows].double().cpu() - want).abs()
    assert (err <= tol).all(), (float(err.max()), float(tol.min()), float(want.mean()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_scores_of_millions(device, dtype):
    """Where scores' 32-bit roundings are several log2 units the weights are what they are, but finite: an average of the
    values, all of them the same."""
    st = Trees(device, dtype, 4, 2, 64, 16, [3000], [20], seed=2, scale=1000.0)
    st.q.mul_(64)
    st.k.mul_(32)
    st.v.fill_(1.5)
    st.nv.fill_(1.5)
    assert torch.isclose(st.run().float(), torch.tensor(1.5, device=device), rtol=2.0 ** -7).all()


def norm_error(st, out):
    """The largest error of a head's output (all of its rows) relative to its norm."""
    worst = 0.0
    for rows, want, _ in definition(st):
        err = (out[0, :, rows].double().cpu() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
        worst = max(worst, float(err.max()))
    return worst


def norm_bound(st):
    """Roundings are of either sign and add up as a random walk does. The result and the 16-bit weights: each at most half
    a step, eps / (2 sqrt 3) of the norm in the mean square, so sqrt(2 / 3) < 1 times eps / 2 together. In 32 bits: sums over
    n keys in numerator and denominator, sqrt(n) 2^-24 each, and scores of a few units, 8 * 2^-24."""
    eps = torch.finfo(st.dtype).eps
    n = max(st.ctx) + max(st.nodes)
    return (eps / 2 if eps > 1e-6 else 0.0) + (8 + 2 * math.sqrt(n)) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(15, 5, 64), (40, 8, 128), (8, 8, 32), (6, 1, 256)])
@pytest.mark.parametrize("ctx,nodes", [([33, 0, 700], [8, 8, 8]), ([200, 1500], [64, 20]), ([9001], [3]), ([40, 90], [70, 129])])
def test_errors_in_the_norm(device, dtype, hq, hkv, d, ctx, nodes):
    st = Trees(device, dtype, hq, hkv, d, 16, ctx, nodes, seed=sum(ctx) + d)
    assert norm_error(st, st.run()) <= norm_bound(st)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_errors_in_the_norm_of_a_long_context(device, dtype):
    st = Trees(device, dtype, 4, 1, 128, 16, [30001], [17], seed=3)
    assert norm_error(st, st.run()) <= norm_bound(st)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs,ctx", [(3, 4000), (3, 9100), (7, 9000), (5, 5121), (6, 6144), (48, 50000)])
def test_long_tables_of_odd_blocks(device, dtype, bs, ctx):
    """More than 1,024 blocks of a size that is no power of two."""
    st = Trees(device, dtype, 4, 2, 64, bs, [ctx, 10], [9, 3], seed=bs)
    out = st.run()
    st.check(out)
    assert norm_error(st, out) <= norm_bound(st)
