"""The 4-bit pool under a model: a step's rows written and attended in every layer, as the packed pass, the
single-sequence cache and the engine run them."""

from __future__ import annotations

import pytest
import torch

from memforge_amd.kernels import attention_backend
from memforge_amd.kernels.batched_decode import BatchedDecodeBuffers, assemble_batch, scatter_new_tokens
from memforge_amd.runtime import ContinuousBatchingEngine, ModelKVSpec, PagedCache, PagedKVPool4, SamplingParams
from memforge_amd.runtime.packed_pass import packed_forward
from tests.scored_reference import attend, check, round4
from tests.tiny_models import StubTokenizer, tiny_capped, tiny_llama

pytestmark = pytest.mark.gpu

PROMPTS = ["a shared beginning of every prompt, and one end", "a shared beginning of every prompt, and another",
           "something else", "x"]


def _pool(model, blocks=40, bs=16):
    return PagedKVPool4(ModelKVSpec.from_config(model.config, model.dtype, "cuda:0"), blocks, bs)


@pytest.mark.parametrize("make,softcap,scale", [(tiny_llama, 0.0, 32 ** -0.5), (tiny_capped, 2.0, 2 ** -0.5)])
def test_every_layer_of_packed_steps(device, monkeypatch, make, softcap, scale):
    """Two prompts prefilled in chunks beside each other, then decoded: each layer's attention output against the
    64-bit definition over the rounded rows that the layer was handed so far."""
    model = make(dtype=torch.float16, **({"head_dim": 32} if make is tiny_llama else {}))
    pool = _pool(model)
    seen = []
    inner = attention_backend._varlen_forward

    def record(module, query, key, value, *args, **kw):
        out = inner(module, query, key, value, *args, **kw)
        seen.append((module.layer_idx, query[0].transpose(0, 1).cpu(), key[0].transpose(0, 1).cpu(),
                     value[0].transpose(0, 1).cpu(), out[0].cpu()))
        return out

    monkeypatch.setattr(attention_backend, "_varlen_forward", record)
    tables = [[3, 9, 1], [20, 7]]
    history = {}
    steps = [([40, 7], [0, 0]), ([1, 20], [40, 7]), ([1, 1], [41, 27])]
    gen = torch.Generator().manual_seed(1)
    for lens, starts in steps:
        tokens = [torch.randint(2, 250, (n,), generator=gen).tolist() for n in lens]
        seen.clear()
        packed_forward(model, pool, tokens, starts, tables, [sum(lens) - 1])
        assert len(seen) == 2
        for layer, q, k, v, out in seen:
            at = 0
            for s, (n, start) in enumerate(zip(lens, starts)):
                hk, hv = history.get((layer, s), (k[:0], v[:0]))
                hk, hv = torch.cat([hk, k[at:at + n]]), torch.cat([hv, v[at:at + n]])
                history[layer, s] = hk, hv
                ref = attend(q[at:at + n], round4(hk, torch.float16), round4(hv, torch.float16), range(start, start + n),
                             scale, softcap)
                check(out[at:at + n], *ref, torch.float16, 32, start + n, softcap, f"layer {layer} sequence {s}")
                at += n
        for layer in range(2):
            k, _ = pool.gather_flat(layer, pool.flat_indices(torch.tensor(tables[0], device=device), 0,
                                                             starts[0] + lens[0]))
            assert torch.equal(k[0].transpose(0, 1).cpu().double(), round4(history[layer, 0][0], torch.float16))


def test_single_sequence_cache(device):
    """PagedCache over a 4-bit pool: what update returns are the rounded rows, and a bound decode attends to them."""
    model = tiny_llama(dtype=torch.bfloat16, head_dim=32)
    pool = _pool(model)
    cache = PagedCache(pool, [5, 2])
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn((1, 2, 19, 32), generator=gen).to(torch.bfloat16).to(device) for _ in range(2))
    cache.layers[0].update(k[:, :, :18], v[:, :, :18])
    got = cache.layers[0].update(k[:, :, 18:], v[:, :, 18:])
    for g, x in zip(got, (k, v)):
        assert torch.equal(g.cpu().double(), round4(x, torch.bfloat16))
    q = torch.randn((1, 4, 1, 32), generator=gen).to(torch.bfloat16).to(device)

    class Layer:
        layer_idx = 0

    with attention_backend.paged_attention_context(pool, cache) as bound:
        out, _ = attention_backend.paged_attention_forward(Layer, q, k[:, :, 18:], v[:, :, 18:], scaling=0.3)
    assert bound.used == 1
    ref = attend(q[0].transpose(0, 1), *(g[0].transpose(0, 1) for g in got), [18], 0.3)
    check(out[0], *ref, torch.bfloat16, 32, 19)


def test_batch_assembly(device):
    model = tiny_llama(dtype=torch.bfloat16, head_dim=32)
    pool = _pool(model)
    gen = torch.Generator().manual_seed(3)
    tables = [torch.tensor([4, 6], device=device), torch.tensor([1], device=device)]
    k, v = (torch.randn((1, 2, 20, 32), generator=gen).to(torch.bfloat16).to(device) for _ in range(2))
    for layer in range(2):
        pool.write_flat(layer, pool.flat_indices(tables[0], 0, 20), k, v)
    new = torch.randn((2, 2, 1, 32), generator=gen).to(torch.bfloat16).to(device)
    scatter_new_tokens(pool, tables, [20, 0], [new, new], [new, new])
    layers, mask, padded = assemble_batch(pool, BatchedDecodeBuffers(2), tables, [21, 1])
    assert mask.sum(1).tolist() == [21, 1]
    for keys, _ in layers:
        assert torch.equal(keys[0, :, padded - 21:padded - 1].cpu().double(), round4(k[0], torch.bfloat16))
        assert torch.equal(keys[:, :, -1:].cpu().double(), round4(new, torch.bfloat16))


def _tokens(model, **kw):
    engine = ContinuousBatchingEngine(model, StubTokenizer(), block_size=16, num_blocks=48, max_num_seqs=4,
                                      max_model_len=256, kv_cache_bits=4, **kw)
    params = SamplingParams(max_new_tokens=12, temperature=0.0, stop_on_eos=False)
    return engine, [r["token_ids"] for r in engine.generate(PROMPTS, params)]


def test_engine(device):
    """Greedy tokens do not depend on how the steps run: captured or eager, with or without shared prefixes (blocks
    copied on write)."""
    model = tiny_llama(dtype=torch.float16, head_dim=32)
    engine, want = _tokens(model, enable_prefix_sharing=False)
    assert all(len(t) == 12 for t in want) and engine.pool.kv_bits == 4
    assert _tokens(model, paged_cuda_graph=True)[1] == want
    shared, got = _tokens(model)
    assert got == want


def test_engine_refuses(device):
    kw = dict(block_size=16, num_blocks=8, max_num_seqs=2, max_model_len=64)
    with pytest.raises(ValueError):
        ContinuousBatchingEngine(tiny_llama(head_dim=32), StubTokenizer(), kv_cache_bits=4, **kw)  # fp32
    model = tiny_llama(dtype=torch.float16, head_dim=32)
    with pytest.raises(ValueError):
        ContinuousBatchingEngine(model, StubTokenizer(), kv_cache_bits=8, **kw)
    with pytest.raises(ValueError):
        ContinuousBatchingEngine(model, StubTokenizer(), kv_cache_bits=4, draft_model=model, lookahead_k=2, **kw)
    with pytest.raises(ValueError):  # head_dim 16
        ContinuousBatchingEngine(tiny_llama(dtype=torch.float16), StubTokenizer(), kv_cache_bits=4, **kw)
