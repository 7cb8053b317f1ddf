"""A pool class of the caller's own (PagedKVPool's arrays and methods, nothing else): every path that takes a pool object
serves it."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels import attention_backend, batched_decode
from memforge_amd.kernels.varlen_attention import paged_attention_varlen_pool
from memforge_amd.runtime import ModelKVSpec, PagedKVPool
from memforge_amd.runtime.graphed_paged_decode import GraphedPagedDecoder
from memforge_amd.runtime.packed_pass import packed_forward
from memforge_amd.runtime.prefix_sharing import copy_blocks
from memforge_amd.runtime.varlen_cache import _slot_bitmap, build_write_index
from tests.tiny_models import tiny_llama


class OwnPool:
    def __init__(self, pool):
        for name in ("spec", "num_blocks", "block_size", "key_pool", "value_pool", "capacity_tokens", "layer_view",
                     "flat_indices", "write_flat", "gather_flat"):
            setattr(self, name, getattr(pool, name))


def test_arrays_alone_say_where_and_in_what_type():
    pool = SimpleNamespace(key_pool=torch.zeros((1, 4, 16, 2, 8), dtype=torch.bfloat16), capacity_tokens=64)
    assert _slot_bitmap(pool).device == pool.key_pool.device
    assert (nat.kv_bits(pool), nat.kv_dtype(pool)) == (16, torch.bfloat16)
    # the arrays' type counts, not the spec's
    pool.spec, pool.block_size = SimpleNamespace(num_kv_heads=2, dtype=torch.float32), 16
    binding = attention_backend._VarlenBinding(pool, [[0, 1]], [0, 0], [3, 4])
    assert binding.meta(4, 32, nat.kv_dtype(pool), "cpu")["plan"].n_narrow > 0


@pytest.mark.gpu
def test_every_path_takes_it(device):
    model = tiny_llama()
    spec = ModelKVSpec.from_config(model.config, torch.float32, str(device))
    pools = [PagedKVPool(spec, 16), PagedKVPool(spec, 16)]
    pools[1] = OwnPool(pools[1])
    prompt, table = list(range(2, 40)), [3, 1, 0, 5]
    outs = []
    for pool in pools:
        got = [packed_forward(model, pool, [prompt], [0], [table], [37]).logits]
        got.append(GraphedPagedDecoder(model, pool, max_batch=2, max_model_len=64).step([7], [38], [table]))
        q = torch.full((1, 4, 2, spec.head_dim), 0.5, device=device)
        got.append(paged_attention_varlen_pool(q, pool, 1, [table], [0, 0], [5, 38]))
        slots = torch.tensor(table, device=device)
        layers, mask, _ = batched_decode.assemble_batch(pool, batched_decode.BatchedDecodeBuffers(spec.num_layers), [slots], [30])
        got += [x.clone() for kv in layers for x in kv] + [mask]
        new = [torch.full((1, 2, 1, spec.head_dim), float(i + 1), device=device) for i in range(spec.num_layers)]
        batched_decode.scatter_new_tokens(pool, [slots], [39], new, new)
        copy_blocks(pool, [(3, 9)])
        got += [pool.key_pool.clone(), pool.value_pool.clone()]
        got.append(build_write_index(pool, [table], [0, 0], [4, 5]))
        cache = SimpleNamespace(position=20, block_table_tensor_cached=lambda: slots.to(torch.int32))
        with attention_backend.paged_attention_context(pool, cache) as binding:
            one = q[:, :, :1]
            got.append(attention_backend.paged_attention_forward(SimpleNamespace(layer_idx=0), one, one[:, :2], one[:, :2])[0])
            assert binding.used == 1
        outs.append(got)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
