"""sample_tokens against its definition in 64 bits: tokens equal, probabilities to a few roundings of 32 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from memforge_amd.runtime.sampling import sample_tokens
from tests.sampling_reference import sample_rows

pytestmark = pytest.mark.gpu

# The share is formed in fp64 from weights exact to 2^-30 and rounded once to fp32 (2^-24 of its value).
SHARE = 2.0 ** -24 + 2.0 ** -28


def check(logits, u, **settings):
    want, share = sample_rows(logits, u, *(settings.get(k, d) for k, d in (("temperature", 1.0), ("top_k", 0),
                                                                         ("top_p", 1.0), ("min_p", 0.0))))
    tokens, probs = sample_tokens(logits, u, **settings)
    assert tokens.dtype == torch.int64 and probs.dtype == torch.float32
    got = tokens.cpu().numpy()
    assert np.array_equal(got, want), [(r, got[r], want[r]) for r in np.flatnonzero(got != want)[:5]]
    np.testing.assert_allclose(probs.double().cpu().numpy(), share, rtol=SHARE, atol=0)
    return tokens


def rows_of(device, rows, vocab, dtype, seed=0, pad=0, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab + pad), generator=gen) * scale
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 8), generator=gen), 3.0 * torch.rand((rows, 8), generator=gen))
    return x.to(device, dtype)[:, :vocab], torch.rand(rows, generator=gen).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab,pad", [(1, 0), (2, 5), (7, 0), (63, 1), (1031, 0), (8191, 2), (32000, 0), (49152, 3),
                                       (130021, 0)])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=1), dict(temperature=0.6, top_k=40, top_p=0.9),
                                      dict(top_p=0.5), dict(min_p=0.1, temperature=1.5),
                                      dict(temperature=0.8, top_k=300, top_p=0.95, min_p=0.01)])
def test_against_64_bits(device, dtype, vocab, pad, settings):
    logits, u = rows_of(device, 9, vocab, dtype, seed=vocab + pad, pad=pad)
    check(logits, u, **settings)


@pytest.mark.parametrize("rows", [1, 2, 17, 64, 65, 130, 257, 300])
def test_settings_of_every_row(device, rows):
    logits, u = rows_of(device, rows, 5000, torch.bfloat16, seed=rows, pad=1)
    gen = torch.Generator().manual_seed(rows)

    def pick(values, dtype=torch.float32):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (rows,), generator=gen)].to(device)

    check(logits, u, temperature=pick([0.0, -1.0, 0.3, 1.0, 2.0]), top_k=pick([0, 1, 5, 200, 9000], torch.int32),
          top_p=pick([1.0, 0.99, 0.7, 0.0, 1.5]), min_p=pick([0.0, 0.05, 0.5, 1.0, 1.5]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 3000, 40001])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=1000, top_p=0.7), dict(min_p=0.5), dict(temperature=0.0)])
@pytest.mark.parametrize("kind", ["equal", "two values", "all banned", "nan", "one left", "infinite", "late peak",
                                  "huge", "signed zeros"])
def test_rows_that_leave_little_or_are_alike(device, dtype, vocab, settings, kind):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((6, vocab), generator=gen)
    if kind == "equal":
        x[:] = 0.25
    elif kind == "two values":
        x = (x > 0.3).float() * 0.5
    elif kind == "all banned":
        x[:] = -math.inf
    elif kind == "nan":
        x[:, ::2] = math.nan
        x[1] = math.nan
    elif kind == "one left":
        at = vocab - 2
        keep = x[:, at].clone()
        x[:] = -math.inf
        x[:, at] = keep
    elif kind == "infinite":
        x[:, ::3] = math.inf
        x[2, 1:] = -math.inf
    elif kind == "late peak":  # far above what the row's first piece holds
        x[:, -1] = 500.0
        x[:3, -2] = 499.5
    elif kind == "huge":
        x = x * 1e30
    else:
        x = torch.where(x > 0, 0.0, -0.0)
    u = torch.tensor([0.0, 0.3, 0.5, 0.75, 0.999, 1.0 - 2.0 ** -24])
    check(x.to(device, dtype), u.to(device), **settings)


@pytest.mark.parametrize("temperature", [1e-3, 0.05, 8.0, 1000.0, 1e30])
@pytest.mark.parametrize("vocab", [700, 20011])
def test_extreme_temperatures(device, temperature, vocab):
    """From all mass on one token to one bin for the whole row."""
    logits, u = rows_of(device, 7, vocab, torch.float32, seed=11)
    check(logits, u, temperature=temperature)
    check(logits, u, temperature=temperature, top_k=333, top_p=0.9)


def test_uniform_numbers_outside_their_range(device):
    logits, _ = rows_of(device, 6, 1000, torch.float32)
    check(logits, torch.tensor([-1.0, 0.0, 1.0, 2.0, math.inf, math.nan]).to(device), top_k=50)


def test_frequencies(device):
    """20000 draws from one row: each token's share within 5 standard deviations."""
    row = torch.tensor([1.0, 3.0, 2.5, -2.0, 0.0, 2.9])
    n = 20000
    tokens, _ = sample_tokens(row.to(device).expand(n, -1).contiguous(),
                              torch.rand(n, generator=torch.Generator().manual_seed(1)).to(device), temperature=0.7)
    p = torch.softmax(row.double() / 0.7, -1).numpy()
    got = np.bincount(tokens.cpu().numpy(), minlength=6) / n
    assert (np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


@pytest.mark.parametrize("rows", [3, 200])
def test_captured_and_on_another_stream(device, rows):
    """A captured call reads new logits at every replay, between eager calls of its own kind."""
    logits, u = rows_of(device, rows, 20000, torch.bfloat16, seed=5)
    check(logits, u, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, probs = sample_tokens(logits, u, top_p=0.9)
    for seed in (6, 7, 8):
        fresh, v = rows_of(device, rows, 20000, torch.bfloat16, seed=seed)
        logits.copy_(fresh)
        u.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = check(logits, u, top_p=0.9)
        assert torch.equal(tokens, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(logits, u, top_k=30)
    torch.cuda.current_stream().wait_stream(side)


def test_same_result_every_time(device):
    logits, u = rows_of(device, 40, 49152, torch.float32, seed=9, scale=0.5)
    first = sample_tokens(logits, u, top_p=0.95)
    for _ in range(5):
        again = sample_tokens(logits, u, top_p=0.95)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("kind", ["normal", "equal"])
def test_largest_vocabulary(device, kind):
    vocab = 1 << 20
    logits, u = rows_of(device, 3, vocab, torch.bfloat16, seed=2, pad=1)
    if kind == "equal":
        logits[:] = 1.0
    check(logits, u)
    check(logits, u, top_k=vocab - 5, top_p=0.999, min_p=1e-6)


def test_expanded_and_distant_rows(device):
    """One row for many draws, and rows further apart than 32 bits hold."""
    logits, u = rows_of(device, 40, 3001, torch.float32, seed=4)
    check(logits[:1].expand(40, -1), u, top_p=0.9)
    far = torch.zeros((3, 1 << 30), dtype=torch.bfloat16, device=device)
    far[:, 7:3008] = logits[:3].to(torch.bfloat16)
    check(far[:, 7:3008], u[:3], top_k=500)


def test_two_streams_at_once(device):
    """Split rows on two streams keep memory of their own."""
    sets = [rows_of(device, 3, 60000, torch.float32, seed=s) for s in (1, 2)]
    want = [sample_tokens(*s, top_p=0.97) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for s, stream, out in zip(sets, streams, got):
            with torch.cuda.stream(stream):
                out.append(sample_tokens(*s, top_p=0.97))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]) for o in outs)


def test_no_rows(device):
    tokens, probs = sample_tokens(torch.empty((0, 10), device=device), torch.empty(0, device=device))
    assert tokens.shape == probs.shape == (0,)
