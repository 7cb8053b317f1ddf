"""Layers with a sliding window, without a GPU: the paged kernels attend to whole contexts, so every paged route refuses
a context longer than the window, and the eager one masks it."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from memforge_amd.kernels import attention_backend as backend


def _forward(q_len, keys, window, **kw):
    gen = torch.Generator().manual_seed(q_len + keys)
    q = torch.randn((1, 2, q_len, 8), generator=gen)
    k, v = (torch.randn((1, 1, keys, 8), generator=gen) for _ in range(2))
    out, _ = backend.paged_attention_forward(SimpleNamespace(layer_idx=0), q, k, v, None, None, sliding_window=window, **kw)
    return q, k, v, out


def test_packed_pass_refuses_a_context_past_the_window():
    pool = SimpleNamespace(block_size=16)
    for last, window in ((40, 40), (200, 64)):
        with backend.varlen_attention_context(pool, [list(range(16))] * 2, [0, 0, 1], [last - 1, last, 3]):
            with pytest.raises(ValueError, match="sliding window"):
                _forward(3, 3, window)
    meta = {"kv_lens": torch.tensor([3, 65])}
    for longest in (65, None):  # None: the pass's lengths are on the device alone
        with backend.bind_varlen(backend._VarlenBinding.from_packed(pool, meta, 3, longest=longest)):
            with pytest.raises(ValueError, match="sliding window"):
                _forward(3, 3, 64)


def test_a_window_no_context_reaches_is_not_refused():
    binding = backend._VarlenBinding(None, [], [0, 0], [62, 63])
    binding.check_window(64)
    binding.check_window(None)
    binding.check_window(-1)
    binding.check_window(200)
    assert binding.window == 64  # the shortest named: what a captured step's later contexts are checked against
    with pytest.raises(ValueError):
        backend._VarlenBinding(None, [], [0], [64]).check_window(64)


@pytest.mark.parametrize("q_len", [1, 5])
def test_single_sequence_route(q_len):
    cache = SimpleNamespace(position=30)
    pool = SimpleNamespace(kv_bits=16)
    with backend.paged_attention_context(pool, cache) as binding:
        # a cache that hands on the new keys alone: their context's window cannot be attended to
        with pytest.raises(ValueError, match="sliding window"):
            _forward(q_len, q_len, 16)
        # the whole context: masked in plain torch
        q, k, v, out = _forward(q_len, 30, 16)
        assert binding.used == 0 and binding.fallbacks == 1
    pos = torch.arange(30 - q_len, 30)
    key = torch.arange(30)
    seen = (key <= pos[:, None]) & (key > pos[:, None] - 16)
    score = torch.matmul(q, k.transpose(2, 3)) / 8 ** 0.5
    want = torch.softmax(score.masked_fill(~seen, float("-inf")), -1) @ v
    torch.testing.assert_close(out, want.transpose(1, 2), rtol=1e-5, atol=1e-5)


def test_windows_of_a_config():
    def config(**kw):
        return SimpleNamespace(**kw)

    assert backend.attention_window(config()) is None
    assert backend.attention_window(config(sliding_window=None)) is None
    assert backend.attention_window(config(sliding_window=-1)) is None
    assert backend.attention_window(config(sliding_window=128)) == 128
    assert backend.attention_window(config(sliding_window=128, layer_types=["full_attention"] * 2)) is None
    assert backend.attention_window(config(sliding_window=128, layer_types=["full_attention", "sliding_attention"])) == 128
