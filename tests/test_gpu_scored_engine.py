"""A model that caps its attention scores, served through the engine: greedy output equals plain transformers' on every
kind of pass (packed prefill and decode, captured decode, the speculative verify)."""

from __future__ import annotations

import pytest
import torch

from memforge_amd.runtime import ContinuousBatchingEngine, SamplingParams
from tests.tiny_models import StubTokenizer, hf_greedy, tiny_capped

pytestmark = pytest.mark.gpu

PROMPTS = ["a capped prompt", "second prompt, quite a bit longer than the first one was", "x"]


def _generate(model, **kw):
    engine = ContinuousBatchingEngine(model, StubTokenizer(), block_size=16, num_blocks=64, max_num_seqs=4,
                                      max_model_len=256, **kw)
    params = SamplingParams(max_new_tokens=12, temperature=0.0, stop_on_eos=False)
    return engine, [r["token_ids"] for r in engine.generate(PROMPTS, params)]


@pytest.mark.parametrize("graph", [False, True])
def test_engine_matches_transformers(device, graph):
    model = tiny_capped()
    want = [hf_greedy(model, StubTokenizer()(p)["input_ids"], 12, stop_on_eos=False) for p in PROMPTS]
    uncapped = tiny_capped(softcap=None)
    plain = [hf_greedy(uncapped, StubTokenizer()(p)["input_ids"], 12, stop_on_eos=False) for p in PROMPTS]
    assert want != plain, "the cap must matter for this test"
    engine, got = _generate(model, paged_cuda_graph=graph)
    assert got == want


def test_speculative_verify_caps_scores(device):
    model, draft = tiny_capped(), tiny_capped(seed=1)
    want = [hf_greedy(model, StubTokenizer()(p)["input_ids"], 12, stop_on_eos=False) for p in PROMPTS]
    _, got = _generate(model, draft_model=draft, lookahead_k=3)
    assert got == want
