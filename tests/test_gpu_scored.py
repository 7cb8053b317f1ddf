"""Attention with capped, biased and masked scores against the 64-bit definition (tests/scored_reference.py): every
path of the kernels (single-wave and cooperative decode items, items sharing tiles through LDS, items that do not, mixed
launches, other block sizes and padded head_dims, split ranges), in-flight keys, written-in-flight steps, captured
launches, rows that see nothing, and NaN where no row looks."""

from __future__ import annotations

import math

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels.varlen_attention import paged_attention_varlen
from tests.gpu_helpers import pad_tables, random_tables
from tests.scored_reference import attend, check

pytestmark = pytest.mark.gpu


def slopes_of(hq, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32, device=device)


class Step:
    """One packed call: runs are (first key, position of the first row, rows, prefix length), each a sequence with a
    block table of its own unless ``table_of`` names another run's."""

    def __init__(self, device, dtype, hq, hkv, d, bs, runs, seed=0, table_of=None):
        gen = torch.Generator().manual_seed(seed)
        self.runs, self.dtype, self.hq, self.hkv, self.d, self.bs, self.device = runs, dtype, hq, hkv, d, bs, device
        own = [i if table_of is None else table_of[i] for i in range(len(runs))]
        self.kv = [start + n for _, start, n, _ in runs]
        length = [max([self.kv[j] for j in range(len(runs)) if own[j] == i] or [0]) for i in range(len(runs))]
        blocks = sum(-(-n // bs) for n in length) + 3
        tables = random_tables(gen, blocks, length, bs)
        self.tables = [tables[o] for o in own]
        self.kp = torch.randn((blocks, bs, hkv, d), generator=gen).to(dtype).to(device)
        self.vp = torch.randn((blocks, bs, hkv, d), generator=gen).to(dtype).to(device)
        self.rows = sum(n for _, _, n, _ in runs)
        self.q = (2 * torch.randn((self.rows, hq, d), generator=gen)).to(dtype).to(device)
        self.cu = [0]
        for _, _, n, _ in runs:
            self.cu.append(self.cu[-1] + n)
        self.positions = [start + i for _, start, n, _ in runs for i in range(n)]
        self.bt = pad_tables(self.tables, device)
        self.cu_t = torch.tensor(self.cu, dtype=torch.int32, device=device)
        self.kv_t = torch.tensor(self.kv, dtype=torch.int32, device=device)
        self.pos_t = torch.tensor(self.positions, dtype=torch.int64, device=device)
        self.scale = 1.0 / math.sqrt(d)

    def slots(self, i, a, b):
        pos = torch.arange(a, b)
        return torch.tensor(self.tables[i], dtype=torch.int64)[pos // self.bs] * self.bs + pos % self.bs

    def scoring(self, softcap=0.0, slopes=None, masks=True):
        first, prefix = [r[0] for r in self.runs], [r[3] for r in self.runs]

        def dev(x):
            return torch.tensor(x, dtype=torch.int32, device=self.device) if masks and any(x) else None

        return nat.Scoring(softcap, slopes, dev(first), dev(prefix))

    def plan(self, **kw):
        first, prefix = [r[0] for r in self.runs], [r[3] for r in self.runs]
        return nat.plan_attention(self.cu, self.kv, self.hq, self.hkv, self.d, self.dtype, self.device,
                                  first_keys=first if any(first) else None,
                                  prefix_lens=prefix if any(prefix) else None, **kw)

    def run(self, scoring, plan=None, **kw):
        out = torch.full_like(self.q, float("nan"))
        nat.paged_attention(self.q, out, nat.PoolView.from_bshd(self.kp, self.vp), self.bt, self.cu_t, self.kv_t,
                            self.pos_t, plan if plan is not None else self.plan(), self.scale, self.hkv,
                            scoring=scoring, **kw)
        return out

    def verify(self, out, softcap=0.0, slopes=None, what=""):
        flat_k, flat_v = (x.view(-1, self.hkv, self.d).cpu() for x in (self.kp, self.vp))
        for i, (first, start, n, prefix) in enumerate(self.runs):
            at = self.slots(i, 0, self.kv[i])
            ref = attend(self.q[self.cu[i]:self.cu[i + 1]], flat_k[at], flat_v[at], range(start, start + n), self.scale,
                         softcap, slopes, first, prefix)
            check(out[self.cu[i]:self.cu[i + 1]], *ref, self.dtype, self.d, self.kv[i], softcap, f"{what} run {i}")


MODS = [(30.0, False), (0.0, True), (5.0, True)]
DECODES = [(0, 0, 1, 0), (0, 16, 1, 0), (0, 299, 1, 0), (0, 30, 1, 0), (0, 1500, 1, 0)]
PREFILLS = [(0, 0, 37, 0), (0, 45, 80, 0), (0, 0, 1, 0), (0, 250, 33, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,bs", [(15, 5, 64, 16), (8, 1, 128, 16), (4, 4, 32, 16), (6, 2, 16, 16),
                                         (6, 2, 64, 8), (5, 5, 128, 5), (16, 2, 256, 16)])
@pytest.mark.parametrize("softcap,bias", MODS)
def test_against_definition(device, dtype, hq, hkv, d, bs, softcap, bias):
    if dtype == torch.float32 and d == 256:
        pytest.skip("fp32 heads go to 128")
    slopes = slopes_of(hq, device) if bias else None
    for name, runs in (("decode", DECODES), ("prefill", PREFILLS), ("mixed", DECODES + PREFILLS)):
        st = Step(device, dtype, hq, hkv, d, bs, runs, seed=hq * d + bs)
        st.verify(st.run(st.scoring(softcap, slopes)), softcap, slopes, name)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("bs", [16, 32, 7])
def test_documents_and_prefixes(device, dtype, d, bs):
    # one packed prompt of four documents (runs over one table), with and without prefixes; another sequence's decode
    runs = [(0, 0, 45, 20), (45, 45, 1, 0), (46, 46, 130, 100), (176, 176, 60, 236), (0, 99, 1, 0), (64, 99, 1, 0)]
    table_of = [0, 0, 0, 0, 4, 4]
    st = Step(device, dtype, 6, 2, d, bs, runs, seed=3, table_of=table_of)
    for softcap, slopes in ((0.0, None), (20.0, slopes_of(6, device))):
        st.verify(st.run(st.scoring(softcap, slopes)), softcap, slopes, "documents")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing_get_zeros(device, dtype):
    # documents that begin after the row, past the context and past the table
    runs = [(40, 30, 5, 0), (200, 99, 1, 0), (10**6, 20, 1, 0), (0, 50, 1, 0), (38, 30, 20, 0)]
    st = Step(device, dtype, 8, 2, 64, 16, runs, seed=4)
    out = st.run(st.scoring())
    st.verify(out)
    assert (out[:7] == 0).all()


@pytest.mark.parametrize("dtype,bs", [(torch.bfloat16, 16), (torch.float16, 32), (torch.float32, 16), (torch.bfloat16, 8)])
@pytest.mark.parametrize("planned", [True, False])
def test_nan_where_no_row_looks(device, dtype, bs, planned):
    """Keys before a document's first and slots past the context may hold anything; a plan that does not know the
    first keys reads them and masks them."""
    runs = [(70, 70, 90, 0), (70, 200, 1, 0), (333, 600, 1, 0), (5, 40, 1, 0)]
    st = Step(device, dtype, 6, 2, 64, bs, runs, seed=5)
    flat_k, flat_v = (x.view(-1, 2, 64) for x in (st.kp, st.vp))
    used = torch.zeros(flat_k.shape[0], dtype=torch.bool)
    for i, (first, *_) in enumerate(runs):
        used[st.slots(i, first, st.kv[i])] = True
    flat_k[~used.to(device)] = float("nan")
    flat_v[~used.to(device)] = float("inf")
    plan = st.plan() if planned else nat.plan_attention(st.cu, st.kv, 6, 2, 64, dtype, device)
    out = st.run(st.scoring(25.0), plan)
    flat_k[~used.to(device)] = 0
    flat_v[~used.to(device)] = 0
    st.verify(out, 25.0, what="nan")


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.bfloat16, 15, 5, 64), (torch.float16, 8, 1, 128), (torch.float32, 4, 2, 64)])
def test_in_flight_and_written_in_flight(device, dtype, hq, hkv, d):
    """A verify pass (keys from pool_lens on are the new rows) and a step that writes its rows: the same bits as the
    rows written first, and the same pool."""
    runs = [(0, 100, 5, 0), (0, 0, 40, 0), (0, 333, 1, 0), (0, 64, 130, 0)]
    softcap, slopes = 20.0, slopes_of(hq, device)
    st = Step(device, dtype, hq, hkv, d, 16, runs, seed=6)
    gen = torch.Generator().manual_seed(7)
    nk, nv = (torch.randn((st.rows, hkv, d), generator=gen).to(dtype).to(device) for _ in range(2))
    slots = torch.cat([st.slots(i, r[1], st.kv[i]) for i, r in enumerate(runs)]).to(device)
    before = st.kp.clone(), st.vp.clone()
    pool_lens = torch.tensor([r[1] for r in runs], dtype=torch.int32, device=device)
    plan, scoring = st.plan(), st.scoring(softcap, slopes)
    verify = st.run(scoring, plan, pool_lens=pool_lens, new_k_rows=nk, new_v_rows=nv)
    assert torch.equal(st.kp, before[0])
    fused = torch.full_like(st.q, float("nan"))
    nat.paged_attention_kv_write(st.q, fused, nat.PoolView.from_bshd(st.kp, st.vp), st.bt, st.cu_t, st.kv_t, st.pos_t,
                                 plan, st.scale, hkv, nk, nv, slots, scoring=scoring)
    want_k, want_v = before[0].clone().view(-1, hkv, d), before[1].clone().view(-1, hkv, d)
    want_k[slots], want_v[slots] = nk, nv
    assert torch.equal(st.kp.view(-1, hkv, d), want_k) and torch.equal(st.vp.view(-1, hkv, d), want_v)
    st.verify(fused, softcap, slopes, "fused")
    st.verify(verify, softcap, slopes, "verify")


def test_captured_launch_replays_with_new_plans(device):
    """Counts in device memory: a graph captured once serves steps of other lengths, its replays interleaved with
    eager work."""
    hq, hkv, d, dtype = 15, 5, 64, torch.bfloat16
    softcap = 30.0
    lens = [[5, 700, 33], [64, 17, 1200], [1, 1, 1]]
    steps = [Step(device, dtype, hq, hkv, d, 16, [(0, n - 1, 1, 0) for n in ls], seed=8) for ls in lens]
    st = Step(device, dtype, hq, hkv, d, 16, [(0, 1199, 1, 0)] * 3, seed=8)
    plan = nat.CountedPlan(4 * 3 * hkv * 80, 0, 3 * hkv, 3 * hkv * 80 * 16 * (d + 2), device)
    out = torch.full_like(st.q, float("nan"))
    scoring = nat.Scoring(softcap)

    def load(s):
        st.q.copy_(s.q)
        st.pos_t.copy_(s.pos_t)
        st.kv_t.copy_(s.kv_t)
        st.positions = s.positions
        st.kv = s.kv
        st.runs = s.runs
        plan.update(*nat.plan_host(s.cu, s.kv, hq, hkv, d, dtype, device)[:3])

    def launch():
        nat.paged_attention(st.q, out, nat.PoolView.from_bshd(st.kp, st.vp), st.bt, st.cu_t, st.kv_t, st.pos_t, plan,
                            st.scale, hkv, scoring=scoring)

    load(steps[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        launch()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    for s in (steps[1], steps[2], steps[0]):
        load(s)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        st.verify(out, softcap, what="replay")
        eager = st.run(scoring, nat.plan_attention(s.cu, s.kv, hq, hkv, d, dtype, device))
        st.verify(eager, softcap, what="eager")


def test_list_operator(device):
    """Rows in any order, documents named per row, a prefix per sequence; strided queries; a negative scale."""
    gen = torch.Generator().manual_seed(9)
    hq, hkv, d, bs, dtype = 8, 2, 64, 16, torch.bfloat16
    kp = torch.randn((2, 24, bs, hkv, d), generator=gen).to(dtype).to(device)
    vp = torch.randn((2, 24, bs, hkv, d), generator=gen).to(dtype).to(device)
    perm = torch.randperm(24, generator=gen).tolist()
    tables = [perm[:7], perm[7:11]]
    rows = [(0, p, 0 if p < 40 else 40) for p in range(30, 60)] + [(1, 63, 0), (1, 10, 10)]
    order = torch.randperm(len(rows), generator=gen).tolist()
    rows = [rows[i] for i in order]
    q = torch.randn((1, len(rows), hq, d), generator=gen).to(dtype).to(device).transpose(1, 2)
    slopes, prefix = slopes_of(hq, device), [50, 0]
    scale = -0.2
    out = paged_attention_varlen(q, kp, vp, 1, tables, [r[0] for r in rows], [r[1] for r in rows], bs, scale=scale,
                                 softcap=12.0, slopes=slopes, doc_starts=[r[2] for r in rows], prefix_lens=prefix)
    assert out.shape == q.shape and out.dtype == dtype
    for i, (s, pos, first) in enumerate(rows):
        n = max(pos + 1, prefix[s])
        at = torch.tensor(tables[s])[torch.arange(n) // bs] * bs + torch.arange(n) % bs
        k, v = (x[1].view(-1, hkv, d).cpu()[at] for x in (kp, vp))
        ref = attend(q[:, :, i], k, v, [pos], scale, 12.0, slopes, first, prefix[s])
        check(out[:, :, i], *ref, dtype, d, n, 12.0, f"row {i}")


def test_inactive_scoring_is_the_plain_call(device):
    st = Step(device, torch.bfloat16, 6, 2, 64, 16, DECODES + PREFILLS, seed=10)
    plan = st.plan()
    assert torch.equal(st.run(nat.Scoring(), plan), st.run(None, plan))


def test_long_context_offsets(device):
    """A pool past 2^31 elements and a context whose blocks lie at its far end."""
    hq, hkv, d, bs = 8, 8, 128, 16
    blocks = (1 << 31) // (bs * hkv * d) + 64
    kp = torch.zeros((blocks, bs, hkv, d), dtype=torch.bfloat16, device=device)
    vp = torch.zeros_like(kp)
    gen = torch.Generator(device=device).manual_seed(11)
    kp[-64:].normal_(generator=gen)
    vp[-64:].normal_(generator=gen)
    table = list(range(blocks - 1, blocks - 61, -1))
    q = torch.randn((1, hq, 1, d), generator=gen, device=device).to(torch.bfloat16)
    out = paged_attention_varlen(q, kp[None], vp[None], 0, [table], [0], [950], bs, softcap=30.0)
    at = torch.tensor(table, device=device)
    k, v = (x[at].reshape(-1, hkv, d)[:951] for x in (kp, vp))
    check(out[:, :, 0], *attend(q[:, :, 0], k, v, [950], d ** -0.5, 30.0), torch.bfloat16, d, 951, 30.0)


def test_eager_and_block_routes_of_the_backend_cap_scores(device):
    from memforge_amd.kernels.attention_backend import _eager_attention
    from memforge_amd.kernels.block_attention import paged_attention_blockwise

    gen = torch.Generator().manual_seed(12)
    kp, vp = (torch.randn((1, 6, 16, 2, 64), generator=gen).to(device) for _ in range(2))
    q = (3 * torch.randn((1, 4, 1, 64), generator=gen)).to(device)
    k, v = (x[0, [3, 1, 5]].reshape(-1, 2, 64)[:41] for x in (kp, vp))
    out = paged_attention_blockwise(q, kp, vp, 0, torch.tensor([3, 1, 5]), 41, 16, softcap=6.0)
    ref = attend(q[:, :, 0], k, v, [40], 0.125, 6.0)
    check(out[:, :, 0], *ref, torch.float32, 64, 41, 6.0)
    eager = _eager_attention(None, q, k.transpose(0, 1)[None], v.transpose(0, 1)[None], None, None, 6.0)
    assert float((eager[:, 0].cpu().double() - ref[0]).abs().max()) < 1e-4


def test_captured_calls_have_partials_of_their_own(device, monkeypatch):
    """Calls that split ranges, captured into two graphs with ordinary plans: no graph's partials are another's or an
    eager call's, and replays stay right after a larger call has grown the eager workspace."""
    steps = [Step(device, torch.bfloat16, 8, 2, 64, 16, [(0, n - 1, 1, 0)] * 2, seed=n) for n in (3000, 5000, 9000)]
    plans = [st.plan() for st in steps]
    assert all(p.partials_floats > 0 for p in plans)
    at, real = [], nat.Workspace.partials

    def spy(self, floats, dev):
        at.append(real(self, floats, dev))
        return at[-1]

    monkeypatch.setattr(nat.Workspace, "partials", spy)
    graphs, outs = [], []
    for st, plan in zip(steps[:2], plans):
        st.run(st.scoring(20.0), plan)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(st.run(st.scoring(20.0), plan))
        graphs.append(graph)
    spans = [(x.data_ptr(), x.data_ptr() + 4 * x.numel()) for x in (at[2], at[1], at[3])]
    assert all(a[1] <= b[0] or b[1] <= a[0] for i, a in enumerate(spans) for b in spans[:i])
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        steps[2].verify(steps[2].run(steps[2].scoring(20.0), plans[2]), 20.0)
        for st, out in zip(steps, outs):
            st.verify(out, 20.0, what="replay")
            out.zero_()


def test_shapes_are_checked(device):
    st = Step(device, torch.bfloat16, 8, 2, 64, 16, [(0, 40, 1, 0)])
    args = (st.bt, st.cu_t, st.kv_t, st.pos_t, st.plan(), st.scale)
    pool, mods = nat.PoolView.from_bshd(st.kp, st.vp), st.scoring(20.0)
    with pytest.raises(ValueError):
        nat.paged_attention(st.q, torch.empty_like(st.q[:, :4]), pool, *args, 2, scoring=mods)
    with pytest.raises(ValueError):
        nat.paged_attention(st.q, torch.empty_like(st.q), pool, *args, 1, scoring=mods)
    with pytest.raises(ValueError):
        nat.paged_attention(st.q, torch.empty_like(st.q), pool, *args, 2, scoring=mods,
                            partials=torch.empty(1 << 20, dtype=torch.bfloat16, device=device))


@pytest.mark.parametrize("cap", [1e-9, 1e-6, 1e-2, 300.0, 1e5, 1e8, 1e12, 1e20])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_caps_of_any_size(device, dtype, cap):
    """A cap no score comes near leaves the scores to a relative 5.5e-7 (the bound takes 2e-7 of a cap of 4 |t|); one
    far below them keeps 2e-7 of itself."""
    st = Step(device, dtype, 6, 2, 64, 16, DECODES + PREFILLS, seed=11)
    out = st.run(st.scoring(cap))
    flat_k, flat_v = (x.view(-1, 2, 64).cpu() for x in (st.kp, st.vp))
    for i, (_, start, n, _) in enumerate(st.runs):
        at, rows = st.slots(i, 0, st.kv[i]), slice(st.cu[i], st.cu[i + 1])
        ref = attend(st.q[rows], flat_k[at], flat_v[at], range(start, start + n), st.scale, cap)
        check(out[rows], *ref, dtype, 64, st.kv[i], min(cap, 4 * float(ref[2][..., 1].max())), f"cap {cap} run {i}")
