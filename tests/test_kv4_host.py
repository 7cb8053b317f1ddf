"""What the 4-bit pool refuses, without a GPU, and its definition of rounding on known values."""

from __future__ import annotations

import ctypes

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.runtime.kv_pool import ModelKVSpec, PagedKVPool, PagedKVPool4
from tests.scored_reference import round4


def _arrays(n=2, h=3, bs=16, d=64):
    return (torch.zeros((n, h, bs, d // 8), dtype=torch.int32), torch.zeros((n, h, bs, d // 32), dtype=torch.uint8),
            torch.zeros((n, h, d // 8, bs), dtype=torch.int32), torch.zeros((n, h, d // 32, bs), dtype=torch.uint8))


def test_view():
    v = nat.Pool4View(*_arrays(), torch.bfloat16)
    assert (v.num_blocks, v.num_heads, v.block_size, v.head_dim, v.num_slots) == (2, 3, 16, 64, 32)


@pytest.mark.parametrize("change", [
    lambda a: a[:2] + (a[2].transpose(2, 3).contiguous(),) + a[3:],
    lambda a: (a[0].to(torch.int64),) + a[1:],
    lambda a: a[:1] + (a[1][..., :1],) + a[2:],
    lambda a: _arrays(n=3)[:1] + a[1:],
    lambda a: tuple(x[::2] if x.shape[0] > 1 else x for x in _arrays(n=4)),
    lambda a: _arrays(d=96),
    lambda a: _arrays(d=512),
    lambda a: _arrays(bs=8),
    lambda a: _arrays(bs=24),
    lambda a: _arrays(bs=528),
])
def test_view_refuses(change):
    with pytest.raises(ValueError):
        nat.Pool4View(*change(_arrays()), torch.bfloat16)


def test_view_refuses_a_dtype():
    with pytest.raises(TypeError):
        nat.Pool4View(*_arrays(), torch.float64)


def _spec(d=64, dtype=torch.bfloat16, device="cuda"):
    return ModelKVSpec(2, 3, d, dtype, device)


@pytest.mark.parametrize("spec,bs,err", [
    (_spec(device="cpu"), 16, ValueError), (_spec(d=80), 16, ValueError), (_spec(), 20, ValueError),
    (_spec(), 0, ValueError), (_spec(), 1024, ValueError), (_spec(dtype=torch.int8), 16, TypeError)])
def test_pool_refuses(spec, bs, err):
    with pytest.raises(err):
        PagedKVPool4(spec, 4, bs)


def test_sizes():
    # 64 elements: 32 bytes of codes and 2 of scales, K and V, 2 layers, 3 heads
    assert PagedKVPool4._bytes_per_token(_spec()) == 2 * 2 * 3 * 34
    four, full = (c.blocks_for_budget(_spec(), 16, 8.0) for c in (PagedKVPool4, PagedKVPool))
    assert four > 3.7 * full


def _struct(**kw):
    buf = (ctypes.c_int64 * 64)()
    base = (ctypes.addressof(buf) + 15) & ~15
    f = dict(key_codes=base, key_scales=base, value_codes=base, value_scales=base, num_blocks=2, block_size=16,
             num_heads=1, head_dim=64, dtype=2)
    f.update(kw)
    s = nat._Pool4Struct(*(f[n] for n, _ in nat._Pool4Struct._fields_))
    s._buf = buf
    return s, base


BAD = [dict(key_codes=None), dict(value_scales=None), dict(num_blocks=0), dict(block_size=8), dict(block_size=0),
       dict(block_size=-16), dict(block_size=1024), dict(num_heads=0), dict(head_dim=96), dict(head_dim=0), dict(dtype=9),
       dict(key_codes=8), dict(value_scales=2)]


@pytest.mark.parametrize("bad", BAD)
def test_c_entries_refuse_a_pool(bad):
    s, base = _struct(**bad)
    p = ctypes.addressof(s)
    L = nat.lib()
    assert L.mf_kv4_write(base, base, 2, 64, 64, base, 1, p, None) < 0
    assert L.mf_kv4_gather(p, base, 1, base, base, 2, 64, 64, None) < 0
    assert L.mf_paged_attention4(None, base, 64, 64, base, 64, 64, 2, p, base, 1, base, base, base, None, 1, 0.1, base, 4,
                                 0, None, 0, None, None, 0, None) < 0


def test_c_entries_refuse():
    s, base = _struct()
    p = ctypes.addressof(s)
    L = nat.lib()
    assert L.mf_kv4_write(base, base, 5, 64, 64, base, 1, p, None) == -1
    assert L.mf_kv4_write(base, base, 2, 64, 64, base, -1, p, None) == -1
    assert L.mf_kv4_write(None, base, 2, 64, 64, base, 1, p, None) == -1
    assert L.mf_kv4_write(base, base, 2, 64, 64, None, 1, p, None) == -1
    assert L.mf_kv4_write(None, None, 2, 64, 64, None, 0, p, None) == 0
    assert L.mf_kv4_write(base, base, 2, 64, 64, base, 1, None, None) == -1

    def attend(q=base, qs=64, out_s=64, dtype=2, scale=0.1, hq=1, narrow=4, merges=0, mods=None, pool=p):
        return L.mf_paged_attention4(mods, q, qs, 64, base, out_s, 64, dtype, pool, base, 1, base, base, base, None, hq,
                                     scale, base, narrow, 0, None, merges, None, None, 0, None)

    assert attend(narrow=0) == 0
    assert attend(q=None) == -1 and attend(qs=63) == -1 and attend(out_s=3) == -1
    assert attend(dtype=0) == -2 and attend(dtype=1) == -1  # the pool is bf16
    assert attend(scale=float("nan")) == -1 and attend(hq=0) == -1 and attend(narrow=6) == -1
    assert attend(merges=1) == -3
    bad = nat._ScoringStruct(-1.0, None, None, None)
    assert attend(mods=ctypes.addressof(bad)) == -1
    two, _ = _struct(num_heads=2)
    assert attend(hq=3, pool=ctypes.addressof(two)) == -1


def test_rounding_of_known_values():
    x = torch.zeros(1, 1, 64)
    x[0, 0, :8] = torch.tensor([6.0, 5.0, 2.5, 0.25, 0.75, -1.25, -3.5, 7.0])  # scale 1: ties go to the even code
    x[0, 0, 32:36] = torch.tensor([7.0625, 6.0, 1.0, -0.4])  # past 7: scale 2
    got = round4(x, torch.bfloat16)[0, 0]
    assert got[:8].tolist() == [6.0, 4.0, 2.0, 0.0, 1.0, -1.0, -4.0, 6.0]
    assert got[32:36].tolist() == [8.0, 6.0, 1.0, -0.0]
    assert got[8:32].abs().max() == 0
    big = torch.full((1, 1, 32), 65504.0)
    assert round4(big, torch.float16)[0, 0, 0] == 6 * 2.0**13  # the largest fp16 scale
    assert round4(big, torch.bfloat16)[0, 0, 0] == 2.0**16


def test_list_operator_checks_before_the_device():
    class Pool:
        block_size, spec = 16, _spec()

        def layer_view(self, i):
            return nat.Pool4View(*_arrays(), torch.bfloat16)

    from memforge_amd.kernels.varlen_attention import paged_attention_varlen_pool
    with pytest.raises(ValueError):
        paged_attention_varlen_pool(torch.zeros(1, 3, 1, 64), Pool(), 0, [[0]], [0], [3])


def test_plans_for_a_4_bit_pool():
    """Every tile of every (sequence, kv head, column tile) in one item, ranges that a wave's registers hold, whole
    workgroups of wide items, merge records that name their partitions."""
    import numpy as np

    rng = np.random.default_rng(1)
    for _ in range(40):
        n = int(rng.integers(1, 40))
        rows = np.ones(n, dtype=int) if rng.random() < 0.5 else rng.integers(1, 60, n)
        kv = rows + (10 ** rng.uniform(0, 4.7, n)).astype(int)
        hq, hkv, d = ((40, 8, 128), (15, 5, 64), (8, 8, 32), (16, 2, 256))[rng.integers(4)]
        cu = np.concatenate([[0], np.cumsum(rows)])
        items, merges, counts = nat.plan_attention_host(cu, kv, hq, hkv, d, torch.bfloat16, num_cus=256, kv_bits=4)
        narrow = int(counts[0])
        seen, parts = {}, {}
        for i, it in enumerate(items):
            if i < narrow:
                assert it[5] - it[4] <= 128
            if it[9] == 0 or it[3] == 0:
                continue
            for c in range(it[2], it[2] + it[3]):
                seen.setdefault((it[0], it[1], c), set()).update(range(it[4], it[5]))
                if it[6] >= 0:
                    parts.setdefault((it[0], it[1], c), set()).add(it[6] + c - it[2])
        for s in range(n):
            for h in range(hkv):
                for c in range(-(-rows[s] * (hq // hkv) // 16)):
                    got = seen[(s, h, c)]
                    last = kv[s] - rows[s] + min((c * 16 + 15) // (hq // hkv), rows[s] - 1)  # the tile's last position
                    assert got >= set(range(last // 16 + 1))
        for m in merges:
            want = {m[4] + p * m[5] for p in range(m[3])}
            assert parts[(m[0], m[1], m[2])] == want
        wide = items[narrow:].reshape(-1, 4, 12)
        assert (wide[:, :, [0, 1, 4, 5]] == wide[:, :1, [0, 1, 4, 5]]).all()
