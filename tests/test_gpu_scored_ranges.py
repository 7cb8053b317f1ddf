"""Scored and 4-bit attention over long ranges, and masks beside in-flight rows: shared prefill ranges past 128 tiles
(several windows of a block table), decode waves of up to 128 tiles, first keys and prefixes on either side of the border
between the pool and the new rows."""

from __future__ import annotations

import pytest
import torch

from memforge_amd import _native as nat
from tests.test_gpu_kv4 import Step4
from tests.test_gpu_scored import Step, slopes_of

pytestmark = pytest.mark.gpu


def plan_of_one_unit(st, kv_bits=16):
    """A plan made for one compute unit, which leaves shared ranges whole."""
    def plan(lens):
        return nat.plan_attention_host(st.cu, lens, st.hq, st.hkv, st.d, st.dtype, num_cus=1, kv_bits=kv_bits)

    firsts = [r[0] for r in st.runs]
    items, merges, counts = nat._plan_from_first_keys(plan, st.cu, st.kv, firsts) if any(firsts) else plan(st.kv)
    dev_items, dev_merges = nat.upload(nat.plan_upload_parts(items, merges), st.device)
    return nat.plan_from_parts(items, merges, counts, dev_items, dev_merges)


LONG = [(0, 2990, 37, 0), (300, 2600, 40, 0), (0, 20, 33, 2500)]


def _longest(plan):
    held = plan.items_host[plan.n_narrow:plan.n_narrow + plan.n_wide]
    return int((held[:, 5] - held[:, 4]).max())


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 64, 16), (torch.float16, 128, 16), (torch.bfloat16, 128, 32),
                                        (torch.float16, 64, 48), (torch.float16, 32, 16)])
@pytest.mark.parametrize("softcap,bias", [(20.0, True), (0.0, False)])
def test_long_shared_ranges(device, dtype, d, bs, softcap, bias):
    runs = [(f, a, n, p) if p == 0 else (f, a + 2500, n, 2540) for f, a, n, p in LONG]
    slopes = slopes_of(8, device) if bias else None
    st = Step(device, dtype, 8, 1, d, bs, runs, seed=d + bs)
    plan = plan_of_one_unit(st)
    assert _longest(plan) > 128
    st.verify(st.run(st.scoring(softcap, slopes), plan), softcap, slopes, "long")


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 64, 16), (torch.float16, 128, 16), (torch.bfloat16, 128, 32),
                                        (torch.float16, 32, 64)])
@pytest.mark.parametrize("softcap,bias", [(20.0, True), (0.0, False)])
def test_long_shared_ranges_of_4_bits(device, dtype, d, bs, softcap, bias):
    runs = [(f, a, n, p) if p == 0 else (f, a + 2500, n, 2540) for f, a, n, p in LONG]
    slopes = slopes_of(8, device) if bias else None
    st = Step4(device, dtype, 8, 1, d, bs, runs, seed=d + bs)
    plan = plan_of_one_unit(st, kv_bits=4)
    assert _longest(plan) > 128
    st.verify(st.run(st.scoring(softcap, slopes), plan), softcap, slopes, "long")


LONG_DECODES = [(0, 2046, 1, 0), (0, 1999, 1, 0), (0, 8190, 1, 0), (0, 7000, 1, 0), (700, 9000, 1, 0), (0, 1100, 1, 0)]


@pytest.mark.parametrize("dtype,d,bs", [(torch.bfloat16, 64, 16), (torch.float16, 128, 16), (torch.bfloat16, 256, 16),
                                        (torch.float16, 128, 32)])
@pytest.mark.parametrize("bits", [4, 16])
def test_waves_of_128_tiles(device, dtype, d, bs, bits):
    slopes = slopes_of(4, device)
    st = (Step4 if bits == 4 else Step)(device, dtype, 4, 2, d, bs, LONG_DECODES, seed=d)
    plan = st.plan(partition_tiles=128)
    held = plan.items_host[:plan.n_narrow]
    assert int((held[:, 5] - held[:, 4]).max()) > 120
    st.verify(st.run(st.scoring(15.0, slopes), plan), 15.0, slopes, "waves")


MASKED_RUNS = [(50, 100, 5, 0), (0, 0, 40, 30), (20, 64, 130, 100), (100, 90, 30, 0), (0, 333, 1, 334), (0, 200, 70, 150),
               (340, 300, 50, 0), (150, 149, 1, 0)]


@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.bfloat16, 15, 5, 64), (torch.float16, 8, 1, 128), (torch.float32, 4, 2, 64),
                                            (torch.bfloat16, 4, 2, 256)])
@pytest.mark.parametrize("softcap,bias", [(20.0, True), (0.0, False)])
def test_masks_beside_new_rows(device, dtype, hq, hkv, d, softcap, bias):
    slopes = slopes_of(hq, device) if bias else None
    st = Step(device, dtype, hq, hkv, d, 16, MASKED_RUNS, seed=6)
    gen = torch.Generator().manual_seed(7)
    nk, nv = (torch.randn((st.rows, hkv, d), generator=gen).to(dtype).to(device) for _ in range(2))
    slots = torch.cat([st.slots(i, r[1], st.kv[i]) for i, r in enumerate(MASKED_RUNS)]).to(device)
    # what no row sees may hold anything: keys before the first one, in the pool and among the new rows
    flat_k, flat_v = (x.view(-1, hkv, d) for x in (st.kp, st.vp))
    for i, (first, start, n, _) in enumerate(MASKED_RUNS):
        hidden = st.slots(i, 0, min(first, start)).to(device)
        flat_k[hidden], flat_v[hidden] = float("nan"), float("nan")
        new_hidden = slice(st.cu[i], st.cu[i] + max(0, min(first, start + n) - start))
        nk[new_hidden], nv[new_hidden] = float("nan"), float("nan")
    pool_lens = torch.tensor([r[1] for r in MASKED_RUNS], dtype=torch.int32, device=device)
    plan, scoring = st.plan(), st.scoring(softcap, slopes)
    verify = st.run(scoring, plan, pool_lens=pool_lens, new_k_rows=nk, new_v_rows=nv)
    fused = torch.full_like(st.q, float("nan"))
    nat.paged_attention_kv_write(st.q, fused, nat.PoolView.from_bshd(st.kp, st.vp), st.bt, st.cu_t, st.kv_t, st.pos_t,
                                 plan, st.scale, hkv, nk, nv, slots, scoring=scoring)
    for x, new in ((flat_k, nk), (flat_v, nv)):
        assert torch.equal(x[slots].nan_to_num(7.0), new.nan_to_num(7.0))
        x.nan_to_num_(0.0)
    st.verify(fused, softcap, slopes, "fused")
    st.verify(verify, softcap, slopes, "verify")
