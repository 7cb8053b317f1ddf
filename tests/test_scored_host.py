"""What scored attention refuses, and its plans, without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels._varlen import run_varlen


@pytest.mark.parametrize("cap", [-1.0, float("inf"), float("nan")])
def test_softcap_must_be_finite_and_positive(cap):
    with pytest.raises(ValueError):
        nat.Scoring(cap)


def test_no_cap_no_tensors_is_inactive():
    assert not nat.Scoring().active and not nat.Scoring(None).active
    assert nat.Scoring(30.0).active and nat.Scoring(slopes=torch.ones(2)).active


@pytest.mark.parametrize("scoring", [
    nat.Scoring(slopes=torch.ones(3)),
    nat.Scoring(slopes=torch.ones(4, dtype=torch.float64)),
    nat.Scoring(slopes=torch.ones(8)[::2]),
    nat.Scoring(first_keys=torch.zeros(2, dtype=torch.int64)),
    nat.Scoring(first_keys=torch.zeros(3, dtype=torch.int32)),
    nat.Scoring(prefix_lens=torch.zeros(1, dtype=torch.int32)),
])
def test_tensors_are_checked(scoring):
    with pytest.raises(TypeError):
        scoring.struct(4, 2, torch.device("cpu"))


def test_tensors_on_another_device_are_refused():
    with pytest.raises(ValueError):
        nat.Scoring(slopes=torch.ones(4)).struct(4, 2, torch.device("cuda", 0))


def test_c_entry_refuses():
    L = nat.lib()
    fn = L.mf_paged_attention_scored

    def call(scoring, sliced_items=4, dtype=2):
        buf = (ctypes.c_int64 * 64)()
        a = (ctypes.addressof(buf) + 15) & ~15
        return fn(ctypes.addressof(scoring) if scoring is not None else None, a, 64, 64, a, 64, 64, dtype, a, a, 1024,
                  64, 64, 16, a, 1, a, a, a, None, None, None, None, 0, 0, None, 0, 0, 1, 1, 64, 0.125,
                  a, sliced_items, 0, None, 0, None, None, 0, None)

    s = nat._ScoringStruct
    assert call(None) == -1
    for cap in (-1.0, float("nan"), float("inf"), 1e-42, 3e38):
        assert call(s(cap, None, None, None)) == -1, cap
    assert call(s(30.0, None, None, None), sliced_items=3) == -1  # not whole workgroups
    assert call(s(30.0, None, None, None), dtype=7) == -1


def _plan(cu, kv, first, hq=8, hkv=2, d=64, cus=256):
    def plan(lens):
        return nat.plan_attention_host(cu, lens, hq, hkv, d, torch.bfloat16, num_cus=cus)

    return nat._plan_from_first_keys(plan, cu, kv, first)


def test_plans_start_at_the_first_key():
    rng = np.random.default_rng(0)
    for _ in range(30):
        n = int(rng.integers(1, 12))
        rows = rng.integers(1, 200, n) if rng.random() < 0.5 else np.ones(n, dtype=int)
        kv = rows + rng.integers(0, 3000, n)
        first = rng.integers(0, 3500, n)
        cu = np.concatenate([[0], np.cumsum(rows)])
        items, merges, counts = _plan(cu.tolist(), kv.tolist(), first.tolist())
        tile = np.minimum(first, kv - 1) // 16
        seen = {}
        for it in items:
            if it[9] == 0 or it[3] == 0:
                continue
            s = it[0]
            assert it[10] == kv[s] and it[9] == rows[s]
            assert tile[s] <= it[4] <= it[5] <= -(-kv[s] // 16)
            seen.setdefault((s, it[1], it[2]), []).append((it[4], it[5]))
        for s in range(n):  # the last key's tile is in some range of every kv head, and so is the first one's
            for h in range(2):
                spans = [x for (a, b, _), v in seen.items() if (a, b) == (s, h) for x in v]
                assert min(a for a, _ in spans) == tile[s] and max(b for _, b in spans) == -(-kv[s] // 16)


def test_a_sequence_whose_keys_are_all_hidden_keeps_a_tile():
    items, _, _ = _plan([0, 1, 4], [40, 33], [40, 10**6])
    live = items[items[:, 9] > 0]
    assert set(live[:, 0].tolist()) == {0, 1}


def test_plan_lengths_are_checked():
    with pytest.raises(ValueError):
        nat.plan_host([0, 1], [5], 2, 1, 64, torch.bfloat16, None, first_keys=[0, 0])
    with pytest.raises(ValueError):
        nat.plan_host([0, 1], [5], 2, 1, 64, torch.bfloat16, None, prefix_lens=[])


def _varlen(**kw):
    pool = nat.PoolView.from_bshd(torch.zeros(4, 16, 1, 64), torch.zeros(4, 16, 1, 64))
    q = torch.zeros(2, 1, 64)
    run_varlen(q, torch.zeros_like(q), pool, [[0, 1]], [0, 0], [3, 4], None, 1, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(softcap=-2.0), ValueError),
    (dict(doc_starts=[0]), ValueError),
    (dict(doc_starts=[0, -1]), ValueError),
    (dict(prefix_lens=[1, 2]), ValueError),
    (dict(prefix_lens=[-1]), ValueError),
    (dict(prefix_lens=[33]), IndexError),  # needs a third block
    (dict(doc_starts=[0, 0], pool_lens=[3]), ValueError),
    (dict(), ValueError),  # tensors that are not on a GPU
])
def test_list_operator_refuses(kw, err):
    with pytest.raises(err):
        _varlen(**kw)


def test_prefix_plans_need_a_device():
    """A plan made for no device may leave out tiles that only a prefix makes visible."""
    with pytest.raises(ValueError):
        nat.plan_host([0, 300, 301], [600, 900], 8, 2, 64, torch.bfloat16, prefix_lens=[600, 0])
    items = nat.plan_host([0, 300, 301], [600, 900], 8, 2, 64, torch.bfloat16, prefix_lens=[600, 0], partition_tiles=8)[0]
    for head in range(2):
        for group in {int(i[2]) for i in items if i[0] == 0 and i[9] > 0}:
            assert max(i[5] for i in items if i[0] == 0 and i[1] == head and i[2] == group) == 38
