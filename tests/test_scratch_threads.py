"""Calls of several launches made by host threads at the same time on one stream: the scratch that their launches hand to
each other is each thread's own."""

from __future__ import annotations

import threading

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.runtime.sampling import sample_tokens
from tests.test_round_checks_host import TREE_CALL, _plan

ROWS, VOCAB = 2, 50000  # split over the GPU


def in_threads(n, work):
    """work(i) in n threads at once; their results."""
    got, errors = [None] * n, []
    gate = threading.Barrier(n)

    def run(i):
        try:
            gate.wait(60)
            got[i] = work(i)
        except BaseException as e:  # noqa: BLE001  (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not errors, errors
    assert not any(t.is_alive() for t in threads)
    return got


@pytest.fixture
def launches(monkeypatch):
    """Stands in for the GPU: keeps (entry point, the calling thread, its arguments), and returns to no thread before both
    have launched."""
    calls, gate, lock = [], threading.Barrier(2), threading.Lock()

    def launch(dev, what, fn, *args):
        with lock:
            calls.append((what, threading.get_ident(), args))
        gate.wait(60)

    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "device_cus", lambda _: 256)
    monkeypatch.setattr(nat, "_stream", lambda *_: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(nat, "_launch", launch)
    return calls


def test_sampling_rows_split_in_two_threads(launches):
    logits, uniforms = torch.zeros((ROWS, VOCAB)), torch.zeros(ROWS)
    need = nat.lib().mf_sample_workspace_size(ROWS, VOCAB, 256)
    assert need > 0
    in_threads(2, lambda _: sample_tokens(logits, uniforms) and sample_tokens(logits, uniforms))
    at = {}
    for _, thread, args in launches:
        at.setdefault(thread, set()).add(args[-2])
    (a,), (b,) = at.values()  # each thread's own, and the same at its next call
    assert abs(a - b) >= need


def test_tree_attention_in_two_threads(launches, monkeypatch):
    from memforge_amd.kernels.tree_attention import paged_attention_tree

    gate = nat._launch
    monkeypatch.setattr(nat, "_launch", lambda *_: None)
    plan = _plan()
    monkeypatch.setattr(nat, "_launch", gate)
    in_threads(2, lambda _: [paged_attention_tree(**{**TREE_CALL, "plan": plan}) for _ in range(2)])
    at = {}
    for _, thread, args in launches:
        at.setdefault(thread, set()).add(args[-2])
    (a,), (b,) = at.values()
    assert abs(a - b) >= 4 * plan.partials_floats


@pytest.mark.parametrize("kind", ["partials", "counters", "verify", "bins"])
def test_threads_have_scratch_of_their_own(monkeypatch, kind):
    monkeypatch.setattr(nat, "_stream", lambda *_: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ws, device = nat.Workspace(), torch.device("cpu")
    take = lambda _: (getattr(ws, kind)(16, device), getattr(ws, kind)(16, device))  # noqa: E731
    pairs = [take(0)] + in_threads(2, take)
    assert all(a is b for a, b in pairs)
    assert len({a.data_ptr() for a, _ in pairs}) == 3


@pytest.mark.gpu
def test_threads_on_one_stream(device):
    """Samples of split rows and tree attention from two threads on the default stream: each as when made alone."""
    from tests.test_gpu_tree_attention import Trees

    gen = torch.Generator().manual_seed(4)
    logits = [torch.randn((ROWS, VOCAB), generator=gen).to(device) * 3 for _ in range(2)]
    uniforms = [torch.rand(ROWS, generator=gen).to(device) for _ in range(2)]
    temps = [torch.tensor([1.0, 0.0], device=device), torch.tensor([0.0, 0.7], device=device)]
    trees = [Trees(device, torch.bfloat16, 4, 2, 64, 16, [3000 + i], [8], seed=i) for i in range(2)]
    plans = [t.plan() for t in trees]
    alone = [(sample_tokens(logits[i], uniforms[i], temps[i], top_p=0.9), trees[i].run(plans[i])) for i in range(2)]
    torch.cuda.synchronize()

    def work(i):
        torch.cuda.set_device(device)
        return [(sample_tokens(logits[i], uniforms[i], temps[i], top_p=0.9), trees[i].run(plans[i])) for _ in range(50)]

    for i, runs in enumerate(in_threads(2, work)):
        torch.cuda.synchronize()
        (tokens, shares), out = alone[i]
        for (t, p), o in runs:
            assert torch.equal(t, tokens) and torch.equal(p, shares) and torch.equal(o, out)
