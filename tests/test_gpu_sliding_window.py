"""A model whose second kind of layer attends within a sliding window, through the engine: served up to the window,
refused past it on every route."""

from __future__ import annotations

import pytest
import torch

from memforge_amd.runtime import ContinuousBatchingEngine, ModelKVSpec, PagedKVPool, SamplingParams
from memforge_amd.runtime.graphed_paged_decode import GraphedPagedDecoder
from memforge_amd.runtime.packed_pass import packed_forward
from tests.tiny_models import StubTokenizer, VOCAB_SIZE, hf_greedy, tiny_llama

pytestmark = pytest.mark.gpu

WINDOW = 48
PROMPT = list(range(2, 34))


def windowed(device, seed=0):
    from transformers import Gemma2Config, Gemma2ForCausalLM

    torch.manual_seed(seed)
    config = Gemma2Config(vocab_size=VOCAB_SIZE, hidden_size=64, intermediate_size=128, num_hidden_layers=2,
                          num_attention_heads=4, num_key_value_heads=2, head_dim=32, max_position_embeddings=1024,
                          sliding_window=WINDOW, attn_logit_softcapping=2.0, query_pre_attn_scalar=2,
                          initializer_range=0.3, tie_word_embeddings=False, eos_token_id=1, bos_token_id=0, pad_token_id=0)
    config._attn_implementation = "eager"
    model = Gemma2ForCausalLM(config).to(device=device, dtype=torch.float32)
    model.eval()
    return model


@pytest.mark.parametrize("graph", [False, True])
def test_engine_serves_up_to_the_window(device, graph):
    model = windowed(device)
    params = SamplingParams(max_new_tokens=100, temperature=0.0, stop_on_eos=False)
    with pytest.warns(UserWarning, match="sliding windows of 48"):
        engine = ContinuousBatchingEngine(model, StubTokenizer(), num_blocks=32, max_num_seqs=2, max_model_len=256,
                                          paged_cuda_graph=graph)
    assert engine.max_model_len == WINDOW
    got = engine.generate([PROMPT], params)[0]["token_ids"]
    assert got == hf_greedy(model, PROMPT, WINDOW - len(PROMPT), stop_on_eos=False)
    with pytest.raises(ValueError, match="max_model_len"):
        engine.submit(list(range(2, 2 + WINDOW)), params)


def test_packed_and_captured_steps_refuse_past_the_window(device):
    model = windowed(device)
    pool = PagedKVPool(ModelKVSpec.from_config(model.config, torch.float32, str(device)), 16)
    table = list(range(8))
    packed_forward(model, pool, [list(range(2, 2 + WINDOW - 1))], [0], [table], [0])
    with pytest.raises(ValueError, match="sliding window"):
        packed_forward(model, pool, [[2, 3]], [WINDOW - 1], [table], [0])
    graphed = GraphedPagedDecoder(model, pool, max_batch=1, max_model_len=100)
    first = graphed.step([5], [WINDOW - 1], [table])
    assert torch.equal(first, graphed.step([5], [WINDOW - 1], [table]))
    with pytest.raises(ValueError, match="sliding window"):
        graphed.step([5], [WINDOW], [table])


def test_a_draft_with_a_window_stops_proposing_at_it(device):
    model = tiny_llama()
    params = SamplingParams(max_new_tokens=40, temperature=0.0, stop_on_eos=False)
    engine = ContinuousBatchingEngine(model, StubTokenizer(), num_blocks=32, max_num_seqs=2, max_model_len=256,
                                      draft_model=windowed(device), lookahead_k=3, draft_cuda_graph="batched")
    got = engine.generate([PROMPT], params)[0]["token_ids"]
    assert got == hf_greedy(model, PROMPT, 40, stop_on_eos=False)
    assert engine.total_speculative_rounds > 0
