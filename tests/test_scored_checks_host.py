"""More that scored attention and the 4-bit pool refuse, without a GPU."""

from __future__ import annotations

import pytest
import torch

from memforge_amd import _native as nat


@pytest.mark.parametrize("cap", [1e-50, 1e39, -1e-50])
def test_caps_that_32_bits_do_not_hold(cap):
    """1e-50 is 0 in 32 bits: no cap at all instead of one that flattens every score."""
    with pytest.raises(ValueError):
        nat.Scoring(cap)


def _tensors():
    return dict(block_tables=torch.zeros((1, 2), dtype=torch.int32), cu_seqlens=torch.tensor([0, 1], dtype=torch.int32),
                kv_lens=torch.tensor([9], dtype=torch.int32), positions=torch.tensor([8]))


def _call(pool, scoring, change):
    """paged_attention on host tensors: with the one check for the GPU taken away, the others are to refuse first."""
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    kw = {**_tensors(), **{k: v for k, v in change.items() if k in _tensors()}}
    rest = {k: v for k, v in change.items() if k not in kw}
    plan = nat.plan_attention([0, 1], [9], 2, 1, 64, torch.bfloat16, rest.pop("plan_device", "cpu"),
                              kv_bits=4 if isinstance(pool, nat.Pool4View) else 16)
    nat.paged_attention(q, torch.zeros_like(q), pool, kw["block_tables"], kw["cu_seqlens"], kw["kv_lens"], kw["positions"],
                        plan, 0.125, 1, scoring=scoring, **rest)


def _pool(bits):
    if bits == 4:
        return nat.Pool4View(torch.zeros((2, 1, 16, 8), dtype=torch.int32), torch.zeros((2, 1, 16, 2), dtype=torch.uint8),
                             torch.zeros((2, 1, 8, 16), dtype=torch.int32), torch.zeros((2, 1, 2, 16), dtype=torch.uint8),
                             torch.bfloat16)
    return nat.PoolView.from_bshd(*(torch.zeros((2, 16, 1, 64), dtype=torch.bfloat16) for _ in range(2)))


ROWS = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
LENS = torch.tensor([8], dtype=torch.int32)


@pytest.mark.parametrize("bits,change", [
    (16, dict(row_map=torch.zeros(1, dtype=torch.int64))),
    (4, dict(row_map=torch.zeros(1, dtype=torch.int64))),
    (16, dict(row_map=torch.zeros(4, dtype=torch.int32)[::2])),
    (16, dict(pool_lens=LENS.long(), new_k_rows=ROWS, new_v_rows=ROWS)),
    (16, dict(pool_lens=LENS.repeat(2), new_k_rows=ROWS, new_v_rows=ROWS)),
    (16, dict(pool_lens=LENS, new_k_rows=ROWS.float(), new_v_rows=ROWS.float())),
    (16, dict(pool_lens=LENS, new_k_rows=ROWS.repeat(1, 2, 1), new_v_rows=ROWS.repeat(1, 2, 1))),
    (16, dict(pool_lens=LENS, new_k_rows=ROWS[0], new_v_rows=ROWS[0])),
    (16, dict(plan_device="meta")),
    (4, dict(plan_device="meta")),
])
def test_index_arrays_and_new_rows_are_checked(monkeypatch, bits, change):
    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "_check4", lambda *_: None)  # its test is for the GPU too
    monkeypatch.setattr(nat, "_launch", lambda *a, **k: pytest.fail("launched"))
    with pytest.raises((ValueError, TypeError)):
        _call(_pool(bits), nat.Scoring(30.0), change)


@pytest.mark.parametrize("bits", [4, 16])
def test_what_is_right_passes_the_checks(monkeypatch, bits):
    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "_check4", lambda *_: None)
    launched = []
    monkeypatch.setattr(nat, "_launch", lambda *a, **k: launched.append(a))
    change = dict(row_map=torch.zeros(1, dtype=torch.int32))
    if bits == 16:
        change.update(pool_lens=LENS, new_k_rows=ROWS, new_v_rows=ROWS)
    _call(_pool(bits), nat.Scoring(30.0), change)
    assert len(launched) == 1


def test_a_4_bit_pool_is_not_written_in_the_attention_launch():
    t = _tensors()
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="4-bit"):
        nat.paged_attention_kv_write(q, q, _pool(4), t["block_tables"], t["cu_seqlens"], t["kv_lens"], t["positions"], None,
                                     0.125, 1, ROWS, ROWS, torch.zeros(1, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("name", ["row_map", "cu_seqlens", "kv_lens", "positions", "block_tables"])
def test_host_index_arrays_are_refused(device, bits, name):
    pool = _pool(bits)
    if bits == 4:
        pool = nat.Pool4View(*(x.to(device) for x in (pool.key_codes, pool.key_scales, pool.value_codes, pool.value_scales)),
                             torch.bfloat16)
    else:
        pool = nat.PoolView.from_bshd(*(torch.zeros((2, 16, 1, 64), dtype=torch.bfloat16, device=device) for _ in range(2)))
    t = {k: v.to(device) for k, v in {**_tensors(), "row_map": torch.zeros(1, dtype=torch.int32)}.items()}
    t[name] = t[name].cpu()
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=device)
    plan = nat.plan_attention([0, 1], [9], 2, 1, 64, torch.bfloat16, device, kv_bits=bits)
    with pytest.raises(ValueError):
        nat.paged_attention(q, torch.zeros_like(q), pool, t["block_tables"], t["cu_seqlens"], t["kv_lens"], t["positions"],
                            plan, 0.125, 1, row_map=t["row_map"], scoring=nat.Scoring(30.0))
