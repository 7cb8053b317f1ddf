"""paged_attention_tree on rows that do not begin at whole 16 bytes, and on single rows and heads of any stride."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_tree_attention import Trees

pytestmark = pytest.mark.gpu


def misaligned(x):
    flat = torch.empty(x.numel() + 8, dtype=x.dtype, device=x.device)[1:x.numel() + 1]
    return flat.view(x.shape).copy_(x)


def odd_single(x):
    x = x.contiguous()
    return x.as_strided(x.shape, [s if n > 1 else 67 for s, n in zip(x.stride(), x.shape)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,nodes", [(1, 1, 1), (4, 1, 6), (6, 2, 1), (6, 2, 9)])
@pytest.mark.parametrize("lay", [misaligned, odd_single])
def test_layouts(device, dtype, hq, hkv, nodes, lay):
    st = Trees(device, dtype, hq, hkv, 64, 16, [77], [nodes], seed=3)
    st.check(st.run())
    st.q = lay(st.q)
    st.check(st.run())
    st.nk = lay(st.nk)
    st.check(st.run())
    st.nv = lay(st.nv)
    st.check(st.run())


@pytest.mark.parametrize("nodes", [[1], [5, 1, 40]])
def test_trees_without_context_or_tables(device, nodes):
    st = Trees(device, torch.bfloat16, 4, 2, 64, 16, [0] * len(nodes), nodes, seed=3)
    st.table = st.table[:, :0].contiguous()
    st.check(st.run())
