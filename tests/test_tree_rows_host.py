"""Rows of tree attention as the C entry point takes them -- whole 16 bytes -- from any layout, without a GPU: a stand-in for
the launch reads what it is pointed at."""

from __future__ import annotations

import ctypes

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.kernels.tree_attention import paged_attention_tree, plan_tree


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def read(at, row, head, rows, heads, dim, dtype):
    """(heads, rows, dim) at an address, with strides in elements."""
    size = dtype.itemsize
    assert at % 16 == 0 and row * size % 16 == 0 and head * size % 16 == 0
    n = (rows - 1) * row + (heads - 1) * head + dim
    flat = torch.frombuffer(bytearray(ctypes.string_at(at, n * size)), dtype=dtype)
    return flat.as_strided((heads, rows, dim), (head, row, 1)).clone()


def misaligned(shape, dtype, gen):
    """Contiguous, two or four bytes past 16."""
    n = torch.Size(shape).numel()
    flat = torch.empty(n + 1 + 64, dtype=dtype)
    flat = flat[-flat.data_ptr() % 64 // dtype.itemsize:][1:n + 1]
    assert flat.data_ptr() % 16
    return flat.copy_(torch.randn(n, generator=gen)).view(shape)


def odd_single(shape, dtype, gen):
    """Aligned; axes of length one have strides that are no whole 16 bytes."""
    x = torch.randn(shape, generator=gen).to(dtype)
    return x.as_strided(shape, [s if n > 1 else 67 for s, n in zip(x.stride(), shape)])


def plain(shape, dtype, gen):
    return torch.randn(shape, generator=gen).to(dtype)


def rows_first(shape, dtype, gen):
    _, heads, rows, dim = shape
    return torch.randn((rows, heads, dim), generator=gen).to(dtype).permute(1, 0, 2)[None]


def spread(shape, dtype, gen):
    return torch.randn((*shape[:3], 2 * shape[3]), generator=gen).to(dtype)[..., ::2]


KINDS = [plain, rows_first, misaligned, odd_single, spread]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,rows", [(1, 1), (1, 5), (2, 1), (2, 5)])
@pytest.mark.parametrize("of_q", KINDS)
@pytest.mark.parametrize("of_k,of_v", [(k, k) for k in KINDS] + [(plain, rows_first), (misaligned, plain), (plain, odd_single)])
def test_layouts(monkeypatch, dtype, heads, rows, of_q, of_k, of_v):
    gen, dim, got = torch.Generator().manual_seed(1), 64, {}

    def launch(dev, what, fn, *a):
        if what == "mf_tree_attention":
            q, k, v = (a[0], a[1], a[2]), (a[16], a[18], a[19]), (a[17], a[18], a[19])
            got.update(q=read(*q, rows, 2 * heads, dim, dtype), k=read(*k, rows, heads, dim, dtype),
                       v=read(*v, rows, heads, dim, dtype))

    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "device_cus", lambda _: 256)
    monkeypatch.setattr(nat, "_launch", launch)
    monkeypatch.setattr(nat._WORKSPACE, "partials", lambda n, dev: torch.empty(n))
    plan = plan_tree(ints(*[-1] * rows), ints(0, rows), ints(9), rows, 2 * heads, heads, dim, dtype, max_context=16)
    pool = torch.zeros((1, 4, 16, heads, dim), dtype=dtype)
    q, k, v = (of((1, n, rows, dim), dtype, gen) for of, n in ((of_q, 2 * heads), (of_k, heads), (of_v, heads)))
    paged_attention_tree(q, pool, pool, 0, torch.zeros((1, 1), dtype=torch.int32), plan, k, v)
    assert torch.equal(got["q"], q[0]) and torch.equal(got["k"], k[0]) and torch.equal(got["v"], v[0])


def test_raw_rows_of_one(monkeypatch):
    """The C binding itself: a single row or kv head may have any stride there."""
    calls = []
    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "device_cus", lambda _: 256)
    monkeypatch.setattr(nat, "_launch", lambda dev, what, fn, *a: calls.append(a))
    monkeypatch.setattr(nat._WORKSPACE, "partials", lambda n, dev: torch.empty(n))
    plan = plan_tree(ints(-1), ints(0, 1), ints(9), 1, 1, 1, 64, torch.bfloat16, max_context=16)
    row = torch.zeros(64, dtype=torch.bfloat16).as_strided((1, 1, 64), (67, 33, 1))
    pool = torch.zeros((4, 16, 1, 64), dtype=torch.bfloat16)
    nat.tree_attention(row, row.clone(), nat.PoolView.from_bshd(pool, pool), torch.zeros((1, 1), dtype=torch.int32), plan, row, row,
                       0.125)
    a = calls[-1]
    assert all(x % 8 == 0 for x in (a[1], a[2], a[4], a[5], a[18], a[19]))


def test_tables_without_columns(monkeypatch):
    """A step of trees that have no context: a null pointer is refused below, so none is handed in."""
    calls = []
    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "device_cus", lambda _: 256)
    monkeypatch.setattr(nat, "_launch", lambda dev, what, fn, *a: calls.append(a))
    monkeypatch.setattr(nat._WORKSPACE, "partials", lambda n, dev: torch.empty(n))
    plan = plan_tree(ints(-1, 0), ints(0, 2), ints(0), 2, 2, 1, 64, torch.bfloat16, max_context=0)
    pool = torch.zeros((1, 4, 16, 1, 64), dtype=torch.bfloat16)
    rows = torch.zeros((1, 2, 2, 64), dtype=torch.bfloat16)
    paged_attention_tree(rows, pool, pool, 0, torch.zeros((1, 0), dtype=torch.int32), plan, rows[:, :1], rows[:, :1])
    assert calls[-1][14] and calls[-1][15] == 0
