"""The 4-bit pool: rows rounded by the definition bit for bit, gathered back exactly, copied, and attended against the
64-bit definition over the values they stand for, on every path of the kernels."""

from __future__ import annotations

import math

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels.varlen_attention import paged_attention_varlen_pool
from memforge_amd.runtime import ModelKVSpec, PagedKVPool4
from memforge_amd.runtime.graphed_paged_decode import split_plan_capacity
from memforge_amd.runtime.prefix_sharing import copy_blocks
from tests.gpu_helpers import pad_tables, random_tables
from tests.scored_reference import attend, check, round4
from tests.test_gpu_scored import DECODES, PREFILLS, slopes_of

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def make_pool(device, dtype, hkv, d, blocks, bs=16, layers=1):
    return PagedKVPool4(ModelKVSpec(layers, hkv, d, dtype, str(device)), blocks, bs)


def rows_of_all_kinds(gen, n, hkv, d, dtype):
    """Values over the type's whole range, groups of ties, zeros, negative zeros, one dominant element, subnormals."""
    x = torch.randn((n, hkv, d // 32, 32), generator=gen, dtype=torch.float64)
    kind = torch.randint(0, 8, (n, hkv, d // 32, 1), generator=gen)
    big = {torch.float16: (-22, 15), torch.bfloat16: (-124, 127), torch.float32: (-124, 127)}[dtype]
    e = torch.randint(big[0], big[1], (n, hkv, d // 32, 1), generator=gen).double()
    ties = torch.randint(-28, 29, x.shape, generator=gen).double() * 0.25
    x = torch.where(kind == 1, x * torch.exp2(e) / 4, x)
    x = torch.where(kind == 2, ties * torch.exp2(torch.clamp(e, big[0], big[1] - 3)), x)
    x = torch.where(kind == 3, torch.zeros_like(x), x)
    x = torch.where(kind == 4, -torch.zeros_like(x), x)
    x = torch.where((kind == 5) & (torch.arange(32) == 7), x * 100, x)
    x = torch.where(kind == 6, torch.exp2(e) * torch.sign(x) * (1.75 + torch.randint(-1, 2, x.shape, generator=gen) * 2.0**-7) / 2, x)
    return x.view(n, hkv, d).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)


@pytest.mark.parametrize("src", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hkv,d,bs", [(5, 64, 16), (8, 128, 32), (1, 32, 48), (2, 256, 16)])
def test_rows_are_rounded_by_the_definition(device, src, dtype, hkv, d, bs):
    gen = torch.Generator().manual_seed(hkv * d)
    n, blocks = 77, 9
    k, v = (rows_of_all_kinds(gen, n, hkv, d, src) for _ in range(2))
    pool = make_pool(device, dtype, hkv, d, blocks, bs, layers=2)
    slots = torch.randperm(blocks * bs, generator=gen)[:n]
    pool.write_flat(1, slots.to(device), k.to(device).transpose(0, 1)[None], v.to(device).transpose(0, 1)[None])
    got = pool.gather_flat(1, slots.to(device))
    assert (pool.key_codes[0] == 0).all() and (pool.value_scales[0] == 0).all()
    for g, x in zip(got, (k, v)):
        want = round4(x, dtype)
        assert g.dtype == dtype
        assert int((g[0].transpose(0, 1).cpu().double() != want).sum()) == 0


@pytest.mark.parametrize("new", [1, 16, 33, 300])
def test_write_at_any_alignment(device, new):
    """Strided and unaligned rows, runs of consecutive slots and single ones, skipped slots."""
    gen = torch.Generator().manual_seed(new)
    hkv, d, bs, blocks = 3, 64, 16, 30
    pool = make_pool(device, torch.bfloat16, hkv, d, blocks, bs)
    wide = torch.randn((2, hkv, new + 1, d + 3), generator=gen).to(torch.bfloat16).to(device)
    k, v = wide[0, :, 1:, 1:1 + d].permute(1, 0, 2), wide[1, :, 1:, 1:1 + d].permute(1, 0, 2)
    start = 7
    slots = torch.arange(start, start + new)
    skipped = torch.rand(new, generator=gen) < 0.2
    target = torch.where(skipped, torch.tensor([-1, blocks * bs, 1 << 40])[torch.arange(new) % 3], slots)
    pool.write_flat(0, target.to(device), k.permute(1, 0, 2)[None], v.permute(1, 0, 2)[None])
    got = pool.gather_flat(0, torch.arange(blocks * bs, device=device))
    for g, x in zip(got, (k, v)):
        want = torch.zeros((blocks * bs, hkv, d), dtype=torch.float64)
        want[slots[~skipped]] = round4(x.cpu(), torch.bfloat16)[~skipped]
        assert int((g[0].transpose(0, 1).cpu().double() != want).sum()) == 0
    left = torch.full((new, hkv, d), 7.0, device=device)
    nat.kv4_gather(pool.layer_view(0), target.to(device), left, left.clone())
    assert (left.cpu()[skipped] == 7.0).all() and (left.cpu()[~skipped] != 7.0).any()


def test_groups_that_are_not_finite_read_as_nan(device):
    pool = make_pool(device, torch.bfloat16, 1, 64, 2)
    k = torch.ones((2, 1, 64), device=device)
    k[0, 0, 3], k[1, 0, 40] = float("nan"), float("-inf")
    pool.write_flat(0, torch.tensor([3, 20], device=device), k.transpose(0, 1)[None], k.transpose(0, 1)[None])
    for g in pool.gather_flat(0, torch.tensor([3, 20], device=device)):
        bad = torch.isnan(g[0, 0]).view(2, 2, 32)
        assert bad[0, 0].all() and not bad[0, 1].any() and not bad[1, 0].any() and bad[1, 1].all()


def test_no_rows(device):
    pool = make_pool(device, torch.bfloat16, 2, 64, 2)
    none = torch.empty((1, 2, 0, 64), device=device)
    index = torch.empty(0, dtype=torch.int64, device=device)
    pool.write_flat(0, index, none, none)
    assert pool.gather_flat(0, index)[0].shape == (1, 2, 0, 64)


def test_copy_blocks(device):
    gen = torch.Generator().manual_seed(1)
    pool = make_pool(device, torch.float16, 3, 32, 6, layers=2)
    for layer in range(2):
        x = torch.randn((1, 3, 96, 32), generator=gen).to(device)
        pool.write_flat(layer, torch.arange(96, device=device), x, -x)
    before = [pool.gather_flat(layer, torch.arange(96, device=device)) for layer in range(2)]
    copy_blocks(pool, [(1, 4), (0, 5)])
    for layer in range(2):
        for b, a in zip(before[layer], pool.gather_flat(layer, torch.arange(96, device=device))):
            want = b.clone()
            want[:, :, 64:80], want[:, :, 80:] = b[:, :, 16:32], b[:, :, :16]
            assert torch.equal(a, want)


class Step4:
    """test_gpu_scored.Step over a 4-bit pool."""

    def __init__(self, device, dtype, hq, hkv, d, bs, runs, seed=0, table_of=None):
        gen = torch.Generator().manual_seed(seed)
        self.runs, self.dtype, self.hq, self.hkv, self.d, self.bs, self.device = runs, dtype, hq, hkv, d, bs, device
        own = [i if table_of is None else table_of[i] for i in range(len(runs))]
        self.kv = [start + n for _, start, n, _ in runs]
        length = [max([self.kv[j] for j in range(len(runs)) if own[j] == i] or [0]) for i in range(len(runs))]
        blocks = sum(-(-n // bs) for n in length) + 3
        tables = random_tables(gen, blocks, length, bs)
        self.tables = [tables[o] for o in own]
        self.pool = make_pool(device, dtype, hkv, d, blocks, bs)
        self.k, self.v = (torch.randn((blocks * bs, hkv, d), generator=gen).to(dtype) for _ in range(2))
        self.write()
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

    def write(self):
        every = torch.arange(self.k.shape[0], device=self.device)
        self.pool.write_flat(0, every, self.k.to(self.device).transpose(0, 1)[None],
                             self.v.to(self.device).transpose(0, 1)[None])

    def slots(self, i, a, b):
        pos = torch.arange(a, b)
        return torch.tensor(self.tables[i], dtype=torch.int64)[pos // self.bs] * self.bs + pos % self.bs

    def masks(self):
        return [r[0] for r in self.runs], [r[3] for r in self.runs]

    def scoring(self, softcap=0.0, slopes=None):
        return nat.Scoring(softcap, slopes, *(torch.tensor(x, dtype=torch.int32, device=self.device) if any(x) else None
                                              for x in self.masks()))

    def plan(self, **kw):
        first, prefix = self.masks()
        return nat.plan_attention(self.cu, self.kv, self.hq, self.hkv, self.d, self.dtype, self.device,
                                  first_keys=first if any(first) else None,
                                  prefix_lens=prefix if any(prefix) else None, kv_bits=4, **kw)

    def run(self, scoring=None, plan=None):
        out = torch.full_like(self.q, float("nan"))
        nat.paged_attention(self.q, out, self.pool.layer_view(0), self.bt, self.cu_t, self.kv_t, self.pos_t,
                            plan if plan is not None else self.plan(), self.scale, self.hkv, scoring=scoring)
        return out

    def verify(self, out, softcap=0.0, slopes=None, what=""):
        for i, (first, start, n, prefix) in enumerate(self.runs):
            at = self.slots(i, 0, self.kv[i])
            k, v = round4(self.k[at], self.dtype), round4(self.v[at], self.dtype)
            ref = attend(self.q[self.cu[i]:self.cu[i + 1]], k, v, range(start, start + n), self.scale, softcap, slopes,
                         first, prefix)
            check(out[self.cu[i]:self.cu[i + 1]], *ref, self.dtype, self.d, self.kv[i], softcap, f"{what} run {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,bs", [(15, 5, 64, 16), (8, 1, 128, 16), (4, 4, 32, 48), (40, 8, 128, 32),
                                         (16, 2, 256, 16), (6, 2, 64, 128)])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (30.0, False), (5.0, True)])
def test_against_definition(device, dtype, hq, hkv, d, bs, softcap, bias):
    slopes = slopes_of(hq, device) if bias else None
    for name, runs in (("decode", DECODES), ("prefill", PREFILLS), ("mixed", DECODES + PREFILLS)):
        st = Step4(device, dtype, hq, hkv, d, bs, runs, seed=hq * d + bs)
        st.verify(st.run(st.scoring(softcap, slopes)), softcap, slopes, name)


@pytest.mark.parametrize("tiles", [1, 2, 5, 16, 64])
def test_every_partition(device, tiles):
    """Ranges cut anywhere: odd and even numbers of tiles, units with empty quarters, pooled workgroups."""
    runs = [(0, 0, 1, 0), (0, 15, 1, 0), (0, 16, 1, 0), (0, 1000, 1, 0), (0, 531, 9, 0), (0, 40, 25, 0)]
    st = Step4(device, torch.bfloat16, 6, 2, 64, 16, runs, seed=tiles)
    plan = nat.plan_attention(st.cu, st.kv, 6, 2, 64, torch.bfloat16, device, partition_tiles=tiles, kv_bits=4)
    st.verify(st.run(None, plan), what=f"{tiles} tiles")


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 64, 16), (torch.float16, 128, 32), (torch.bfloat16, 256, 16)])
def test_documents_and_prefixes(device, dtype, d, bs):
    runs = [(0, 0, 45, 20), (45, 45, 1, 0), (46, 46, 130, 100), (176, 176, 60, 236), (0, 99, 1, 0), (64, 99, 1, 0)]
    st = Step4(device, dtype, 6, 2, d, bs, runs, seed=3, table_of=[0, 0, 0, 0, 4, 4])
    for softcap, slopes in ((0.0, None), (20.0, slopes_of(6, device))):
        st.verify(st.run(st.scoring(softcap, slopes)), softcap, slopes, "documents")


@pytest.mark.parametrize("d", [64, 256])
def test_rows_that_see_nothing_get_zeros(device, d):
    runs = [(40, 30, 5, 0), (200, 99, 1, 0), (10**6, 20, 1, 0), (0, 50, 1, 0), (38, 30, 20, 0)]
    st = Step4(device, torch.bfloat16, 8, 2, d, 16, runs, seed=4)
    out = st.run(st.scoring())
    st.verify(out)
    assert (out[:7] == 0).all()


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 64, 16), (torch.float16, 128, 32), (torch.bfloat16, 32, 16),
                                        (torch.float16, 256, 16)])
@pytest.mark.parametrize("planned", [True, False])
def test_nan_where_no_row_looks(device, dtype, d, bs, planned):
    runs = [(70, 70, 90, 0), (70, 200, 1, 0), (333, 600, 1, 0), (5, 40, 1, 0)]
    st = Step4(device, dtype, 6, 2, d, bs, runs, seed=5)
    used = torch.zeros(st.k.shape[0], dtype=torch.bool)
    for i, (first, *_) in enumerate(runs):
        used[st.slots(i, first, st.kv[i])] = True
    keep = st.k.clone(), st.v.clone()
    st.k[~used], st.v[~used] = float("nan"), float("inf")
    st.write()
    plan = st.plan() if planned else nat.plan_attention(st.cu, st.kv, 6, 2, d, dtype, device, kv_bits=4)
    out = st.run(st.scoring(25.0), plan)
    st.k, st.v = keep
    st.verify(out, 25.0, what="nan")


@pytest.mark.parametrize("d,hq,hkv", [(64, 15, 5), (128, 8, 8)])
def test_plans_of_a_captured_decode(device, d, hq, hkv):
    """The plans that a captured decode step takes: without merges, with fixed capacities, with split ranges."""
    lens = [4000, 1, 333, 2017]
    st = Step4(device, torch.float16, hq, hkv, d, 16, [(0, n - 1, 1, 0) for n in lens], seed=d)
    args = (st.cu, st.kv, hq, hkv, d, torch.float16)
    for made in (nat.plan_attention_host(*args, num_cus=256, merge_free=True, kv_bits=4),
                 nat.plan_attention_host(*args, partition_tiles=64), nat.plan_attention_host(*args, num_cus=256, kv_bits=4)):
        plan = nat.CountedPlan(*split_plan_capacity(len(lens), hkv, 252, 16, d), device)
        plan.update(*made)
        st.verify(st.run(None, plan), what=f"{made[2].tolist()}")


def test_replays_of_a_captured_step(device):
    """A write and its attention captured once: each replay reads that step's rows, lengths and plan, with eager
    work in between."""
    hq, hkv, d, bs, dtype = 15, 5, 64, 16, torch.bfloat16
    lens = [[5, 700, 33], [64, 17, 1200], [1, 1, 1]]
    st = Step4(device, dtype, hq, hkv, d, bs, [(0, 1199, 1, 0)] * 3, seed=8)
    gen = torch.Generator().manual_seed(9)
    plan = nat.CountedPlan(4 * 3 * hkv * 80, 0, 3 * hkv, 3 * hkv * 80 * 16 * (d + 2), device)
    nk, nv = (torch.empty((3, hkv, d), dtype=dtype, device=device) for _ in range(2))
    slots = torch.zeros(3, dtype=torch.int64, device=device)
    out = torch.empty_like(st.q)
    view = st.pool.layer_view(0)

    def load(ls):
        st.kv, st.runs = ls, [(0, n - 1, 1, 0) for n in ls]
        st.kv_t.copy_(torch.tensor(ls, dtype=torch.int32))
        st.pos_t.copy_(torch.tensor([n - 1 for n in ls]))
        st.q.copy_(torch.randn(st.q.shape, generator=gen).to(dtype))
        at = torch.cat([st.slots(i, n - 1, n) for i, n in enumerate(ls)])
        st.k[at], st.v[at] = (torch.randn((3, hkv, d), generator=gen).to(dtype) for _ in range(2))
        nk.copy_(st.k[at])
        nv.copy_(st.v[at])
        slots.copy_(at)
        plan.update(*nat.plan_host(st.cu, ls, hq, hkv, d, dtype, device, kv_bits=4)[:3])

    def launch():
        nat.kv4_write(nk, nv, slots, view)
        nat.paged_attention(st.q, out, view, st.bt, st.cu_t, st.kv_t, st.pos_t, plan, st.scale, hkv)

    load(lens[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        launch()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    for ls in (lens[1], lens[2], lens[0]):
        load(ls)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        st.verify(out, what="replay")
        st.verify(st.run(None, nat.plan_attention(st.cu, ls, hq, hkv, d, dtype, device, kv_bits=4)), what="eager")


def test_list_operator(device):
    gen = torch.Generator().manual_seed(9)
    hq, hkv, d, bs, dtype = 8, 2, 64, 32, torch.float16
    pool = make_pool(device, dtype, hkv, d, 12, bs, layers=2)
    k, v = (torch.randn((12 * bs, hkv, d), generator=gen) for _ in range(2))
    pool.write_flat(1, torch.arange(12 * bs, device=device), k.to(device).transpose(0, 1)[None],
                    v.to(device).transpose(0, 1)[None])
    perm = torch.randperm(12, generator=gen).tolist()
    tables = [perm[:4], perm[4:7]]
    rows = [(0, p, 0 if p < 40 else 40) for p in range(30, 60)] + [(1, 63, 0), (1, 10, 10)]
    rows = [rows[i] for i in torch.randperm(len(rows), generator=gen).tolist()]
    q = torch.randn((1, len(rows), hq, d), generator=gen).to(device).transpose(1, 2)  # fp32: taken to the pool's type
    slopes, prefix = slopes_of(hq, device), [50, 0]
    out = paged_attention_varlen_pool(q, pool, 1, tables, [r[0] for r in rows], [r[1] for r in rows], scale=-0.2,
                                      softcap=12.0, slopes=slopes, doc_starts=[r[2] for r in rows], prefix_lens=prefix)
    assert out.shape == q.shape and out.dtype == torch.float32
    k, v = round4(k, dtype), round4(v, dtype)
    for i, (s, pos, first) in enumerate(rows):
        n = max(pos + 1, prefix[s])
        at = torch.tensor(tables[s])[torch.arange(n) // bs] * bs + torch.arange(n) % bs
        ref = attend(q[:, :, i].to(dtype), k[at], v[at], [pos], -0.2, 12.0, slopes, first, prefix[s])
        check(out[:, :, i], *ref, dtype, d, n, 12.0, f"row {i}")


def test_far_end_of_a_large_pool(device):
    """More than 2^32 bytes of codes: the offsets of the last blocks pass 32 bits."""
    hkv, d, bs = 8, 256, 16
    blocks = (1 << 32) // (bs * hkv * d // 2) + 64
    pool = make_pool(device, torch.bfloat16, hkv, d, blocks, bs)
    assert pool.key_codes.numel() * 4 > 1 << 32
    gen = torch.Generator().manual_seed(11)
    table = list(range(blocks - 1, blocks - 61, -1))
    n = 951
    at = torch.tensor(table)[torch.arange(n) // bs] * bs + torch.arange(n) % bs
    k, v = (torch.randn((n, hkv, d), generator=gen).to(torch.bfloat16) for _ in range(2))
    pool.write_flat(0, at.to(device), k.to(device).transpose(0, 1)[None], v.to(device).transpose(0, 1)[None])
    got = pool.gather_flat(0, at.to(device))
    assert torch.equal(got[0][0].transpose(0, 1).cpu().double(), round4(k, torch.bfloat16))
    assert torch.equal(got[1][0].transpose(0, 1).cpu().double(), round4(v, torch.bfloat16))
    q = torch.randn((1, hkv, 1, d), generator=gen).to(torch.bfloat16).to(device)
    out = paged_attention_varlen_pool(q, pool, 0, [table], [0], [n - 1])
    ref = attend(q[:, :, 0], round4(k, torch.bfloat16), round4(v, torch.bfloat16), [n - 1], d ** -0.5)
    check(out[:, :, 0], *ref, torch.bfloat16, d, n)


def test_gpu_refusals(device):
    """Calls that the host turns away before anything is launched."""
    pool = make_pool(device, torch.bfloat16, 2, 64, 4)
    rows = torch.zeros((1, 2, 3, 64), device=device)
    with pytest.raises(ValueError):  # heads
        pool.write_flat(0, torch.arange(3, device=device), rows[:, :1], rows[:, :1])
    with pytest.raises(ValueError):  # slots
        pool.write_flat(0, torch.arange(2, device=device), rows, rows)
    with pytest.raises(ValueError):  # a host slot list
        pool.write_flat(0, torch.arange(3), rows, rows)
    st = Step4(device, torch.bfloat16, 4, 2, 64, 16, [(0, 20, 1, 0)])
    with pytest.raises(TypeError):  # a query of another type
        st.q = st.q.half()
        st.run()
    st = Step4(device, torch.bfloat16, 4, 2, 64, 16, [(0, 20, 1, 0)])
    out = torch.empty_like(st.q)
    args = (st.bt, st.cu_t, st.kv_t, st.pos_t, st.plan(), st.scale, 2)
    with pytest.raises(ValueError):  # in-flight keys
        nat.paged_attention(st.q, out, st.pool.layer_view(0), *args, pool_lens=st.kv_t, new_k_rows=st.q, new_v_rows=st.q)
    with pytest.raises(ValueError):
        nat.paged_attention(st.q, out, st.pool.layer_view(0), *args, fused_merge=True)
    full = make_pool(device, torch.float32, 2, 64, 4)
    with pytest.raises(TypeError):  # fp32 pools are for rows only
        nat.paged_attention(st.q.float(), out.float(), full.layer_view(0), *args)
