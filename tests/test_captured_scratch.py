"""Scratch memory of calls recorded into a graph: the graph's own, for the fused merge's arrival counters and the rejection
verify as for the partials of a split range."""

from __future__ import annotations

import pytest
import torch

from memforge_amd import _native as nat
from tests.test_gpu_scored import Step


@pytest.mark.parametrize("kind", ["partials", "counters", "verify"])
def test_captured_scratch_is_not_kept(monkeypatch, kind):
    monkeypatch.setattr(nat, "_stream", lambda *_: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    ws, device = nat.Workspace(), torch.device("cpu")
    take = getattr(ws, kind)
    capturing = False
    warm = take(16, device)
    capturing = True
    first, second = take(16, device), take(1 << 21, device)
    spans = [(x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in (warm, first, second)]
    assert all(a[1] <= b[0] or b[1] <= a[0] for i, a in enumerate(spans) for b in spans[:i])
    if kind == "counters":
        assert not first.any() and not second.any()
    capturing = False
    assert take(16, device) is warm
    assert take(1 << 21, device) is not second


@pytest.mark.gpu
def test_fused_merges_of_two_graphs(device, monkeypatch):
    """Two graphs captured on one stream before any eager call has made counters, then replays between eager calls whose
    plans are larger."""
    monkeypatch.setattr(nat, "_WORKSPACE", nat.Workspace())
    steps = [Step(device, torch.bfloat16, 8, 2, 64, 16, [(0, n - 1, 1, 0)] * 2, seed=n) for n in (3000, 5000, 9000)]
    plans = [st.plan() for st in steps]
    assert all(p.n_merges > 0 for p in plans)
    graphs, outs = [], []
    for st, plan in zip(steps[:2], plans):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(st.run(None, plan, fused_merge=True))
        graphs.append(graph)
    for _ in range(3):
        steps[2].verify(steps[2].run(None, plans[2], fused_merge=True))
        for graph, st, out in zip(graphs, steps, outs):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            st.verify(out, what="replay")


@pytest.mark.gpu
def test_verifies_of_two_graphs(device, monkeypatch):
    monkeypatch.setattr(nat, "_WORKSPACE", nat.Workspace())
    gen = torch.Generator().manual_seed(5)

    def inputs(rows, k, vocab):
        draft = torch.softmax(torch.randn((rows, k, vocab), generator=gen), -1)
        args = [torch.randint(0, vocab, (rows, k), generator=gen).to(torch.int32), draft,
                torch.randn((rows, k + 1, vocab), generator=gen), 1.0,
                torch.rand((rows, k), generator=gen), torch.empty((rows, vocab)).exponential_(generator=gen)]
        return [x.to(device) if isinstance(x, torch.Tensor) else x for x in args]

    calls = [inputs(3, 2, 5000), inputs(5, 4, 9000), inputs(64, 8, 20000)]
    want = [nat.spec_verify(*c) for c in calls]
    want = [(w.count.clone(), w.num_accepted.clone()) for w in want]
    torch.cuda.synchronize()
    nat._WORKSPACE._verify.clear()
    graphs, outs = [], []
    for c in calls[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(nat.spec_verify(*c))
        graphs.append(graph)
    for _ in range(3):
        big = nat.spec_verify(*calls[2])
        assert torch.equal(big.count, want[2][0])
        for graph, out, (count, accepted) in zip(graphs, outs, want):
            out.packed.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.count, count) and torch.equal(out.num_accepted, accepted)
