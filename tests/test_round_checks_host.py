"""What sampling, device tables and accepted paths refuse, without a GPU: with the one check for the GPU taken away, the
others are to refuse before anything is launched."""

from __future__ import annotations

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.runtime.device_tables import DeviceBlockTables
from memforge_amd.runtime.sampling import sample_tokens
from memforge_amd.speculative import accept_tree


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.fixture
def no_gpu_check(monkeypatch):
    monkeypatch.setattr(nat, "require_device", lambda *_: None)

    def launched(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(nat, "_launch", launched)


LOGITS, U = torch.zeros((3, 10)), torch.zeros(3)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        sample_tokens(LOGITS, U)
    with pytest.raises(ValueError):
        DeviceBlockTables.allocate(2, 3, 4, 16, "cpu").extend(ints(1, 2), 5)
    with pytest.raises(ValueError):
        accept_tree(torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64), ints(-1), ints(0, 1), 1)


@pytest.mark.parametrize("args,settings", [
    ((LOGITS[0], U), {}), ((LOGITS.t(), torch.zeros(10)), {}), ((LOGITS.double(), U), {}), ((LOGITS.int(), U), {}),
    ((LOGITS, U[:2]), {}), ((LOGITS, U.double()), {}), ((LOGITS, U[:, None]), {}), ((torch.zeros((3, 0)), U), {}),
    ((torch.zeros((1, 1)).expand(1, nat.SAMPLE_MAX_VOCAB + 1), U[:1]), {}),
    ((LOGITS, U), dict(temperature=torch.ones(3).double())), ((LOGITS, U), dict(temperature=torch.ones(2))),
    ((LOGITS, U), dict(top_k=torch.ones(3, dtype=torch.int64))), ((LOGITS, U), dict(top_p=torch.ones(6)[::2])),
    ((LOGITS, U), dict(min_p=torch.ones((3, 1)))), ((LOGITS, U), dict(top_p=float("nan"))),
    ((LOGITS, U), dict(temperature=float("nan"))), ((LOGITS, U), dict(min_p=torch.ones(3, device="meta"))),
    ((LOGITS, torch.zeros(3, device="meta")), {})])
def test_sampling_refuses(no_gpu_check, args, settings):
    with pytest.raises((ValueError, TypeError)):
        sample_tokens(*args, **settings)


@pytest.mark.parametrize("change", [
    dict(tables=torch.zeros(6, dtype=torch.int32)), dict(tables=torch.zeros((2, 3), dtype=torch.int64)),
    dict(tables=torch.zeros((2, 6), dtype=torch.int32)[:, ::2]), dict(lens=ints(0)), dict(lens=torch.zeros(2)),
    dict(held=ints(0, 0, 0)), dict(free=torch.zeros(4)), dict(free_count=ints(1, 2)),
    dict(free_count=torch.ones(1, dtype=torch.int64)), dict(held=torch.zeros(2, dtype=torch.int32, device="meta"))])
def test_tables_refuse_their_state(no_gpu_check, change):
    state = DeviceBlockTables.allocate(2, 3, 4, 16, "cpu")
    for k, v in change.items():
        setattr(state, k, v)
    with pytest.raises((ValueError, TypeError)):
        state.extend(ints(1, 2), 5)
    with pytest.raises((ValueError, TypeError)):
        state.truncate(ints(1, 2))


@pytest.mark.parametrize("new,rows,most", [
    (ints(1), None, 5), (torch.tensor([1, 2]), None, 5), (ints(1, 2), None, -1), (ints(1, 2), ints(0, 1), 5),
    (ints(1, 2), torch.zeros((3, 2), dtype=torch.int32), 5), (ints(1, 2), torch.zeros((2, 2), dtype=torch.int64), 5),
    (ints(1, 2), torch.zeros((2, 4), dtype=torch.int32)[:, ::2], 5)])
def test_tables_refuse_a_call(no_gpu_check, new, rows, most):
    with pytest.raises((ValueError, TypeError)):
        DeviceBlockTables.allocate(2, 3, 4, 16, "cpu").extend(new, most, rows)


def test_tables_entry_points_check_sizes():
    """The C entry points by themselves, no pointer read."""
    L, p = nat.lib(), 4096
    extend = [p, 3, 3, p, p, p, 4, p, p, 2, 16, 5, None, 0, 0, p, p, p, p, p, p, None]
    for at, bad in ((1, 2), (2, -1), (3, None), (6, -1), (7, None), (9, -1), (9, 4097), (10, 0), (11, -1), (15, None),
                    (17, None), (18, None), (19, None), (20, None)):
        args = list(extend)
        args[at] = bad
        assert L.mf_tables_extend(*args) == -1, (at, bad)
    truncate = [p, 3, 3, p, p, p, 4, p, p, 2, 16, p, None]
    for at, bad in ((1, 2), (2, -1), (4, None), (5, None), (8, None), (9, 4097), (10, 0), (11, None)):
        args = list(truncate)
        args[at] = bad
        assert L.mf_tables_truncate(*args) == -1, (at, bad)
    assert L.mf_tables_truncate(*truncate[:9], 0, *truncate[10:]) == 0  # nothing to do


@pytest.mark.parametrize("change", [
    dict(tokens=ints(1, 2, 3)), dict(targets=torch.zeros(2, dtype=torch.int64)), dict(parents=torch.zeros(3)),
    dict(parents=torch.zeros(3, dtype=torch.int64)), dict(cu_nodes=torch.tensor([0, 3])), dict(max_nodes=0),
    dict(max_nodes=1025), dict(cu_nodes=ints()), dict(targets=torch.zeros(3, dtype=torch.int64, device="meta"))])
def test_accept_refuses(no_gpu_check, change):
    call = dict(tokens=torch.zeros(3, dtype=torch.int64), targets=torch.zeros(3, dtype=torch.int64),
                parents=ints(-1, 0, 0), cu_nodes=ints(0, 3), max_nodes=3)
    with pytest.raises((ValueError, TypeError)):
        accept_tree(**{**call, **change})


def test_sample_and_accept_entry_points_check_sizes():
    L, p = nat.lib(), 4096
    sample = [p, 0, 10, 2, 10, p, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, 256, None, 0, None]
    for at, bad in ((0, None), (1, 3), (2, -1), (3, -1), (4, 0), (4, nat.SAMPLE_MAX_VOCAB + 1), (5, None), (14, None),
                    (16, 0), (17, 4)):
        args = list(sample)
        args[at] = bad
        assert L.mf_sample(*args) == -1, (at, bad)
    need = L.mf_sample_workspace_size(2, 100000, 256)
    assert need > 0 and L.mf_sample_workspace_size(2, 10, 256) == 0 and L.mf_sample_workspace_size(5000, 100000, 256) == 0
    big = [*sample[:2], 100000, 2, 100000, *sample[5:]]
    assert L.mf_sample(*big) == -3 and L.mf_sample(*big[:17], p, need - 1, None) == -3
    accept = [p, p, p, p, 2, 6, 4, p, p, p, None]
    for at, bad in ((0, None), (3, None), (4, -1), (5, -1), (6, 0), (6, 1025), (7, None), (9, None)):
        args = list(accept)
        args[at] = bad
        assert L.mf_tree_accept(*args) == -1, (at, bad)


# ------------------------------------------------------------------------- trees

def _plan(**change):
    from memforge_amd.kernels.tree_attention import plan_tree

    call = dict(parents=ints(-1, 0, 0), cu_nodes=ints(0, 2, 3), context_lens=ints(5, 9), max_nodes=2, num_q_heads=4,
                num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, max_context=16)
    return plan_tree(**{**call, **change})


@pytest.mark.parametrize("change", [
    dict(parents=torch.tensor([-1, 0, 0])), dict(parents=torch.zeros(3)), dict(cu_nodes=ints(0, 3)),
    dict(cu_nodes=torch.tensor([0, 2, 3])), dict(context_lens=ints(5)), dict(context_lens=torch.tensor([5, 9])),
    dict(max_nodes=0), dict(max_nodes=1025), dict(max_context=-1), dict(max_context=(1 << 30) + 1), dict(num_kv_heads=0),
    dict(num_q_heads=5), dict(num_q_heads=0), dict(head_dim=80), dict(head_dim=16), dict(dtype=torch.float64),
    dict(dtype=torch.int32), dict(context_lens=torch.zeros(2, dtype=torch.int32, device="meta"))])
def test_tree_plans_refuse(no_gpu_check, monkeypatch, change):
    monkeypatch.setattr(nat, "device_cus", lambda _: 256)
    with pytest.raises((ValueError, TypeError)):
        _plan(**change)


def test_tree_plan_needs_the_gpu():
    with pytest.raises(ValueError):
        _plan()


TREE_CALL = dict(query=torch.zeros((1, 4, 3, 64), dtype=torch.bfloat16),
                 key_pool=torch.zeros((1, 4, 16, 2, 64), dtype=torch.bfloat16),
                 value_pool=torch.zeros((1, 4, 16, 2, 64), dtype=torch.bfloat16), layer_idx=0,
                 block_tables=torch.zeros((2, 1), dtype=torch.int32),
                 new_keys=torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16),
                 new_values=torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16))


@pytest.mark.parametrize("change", [
    dict(query=TREE_CALL["query"][0]), dict(query=TREE_CALL["query"][:, :3]), dict(query=TREE_CALL["query"][:, :, :2]),
    dict(query=TREE_CALL["query"].float()), dict(query=TREE_CALL["query"].repeat(2, 1, 1, 1)),
    dict(new_keys=TREE_CALL["new_keys"][:, :1]), dict(new_values=TREE_CALL["new_values"].half()),
    dict(new_keys=TREE_CALL["new_keys"][..., :32]), dict(block_tables=torch.zeros((1, 1), dtype=torch.int32)),
    dict(block_tables=torch.zeros((2, 0), dtype=torch.int32)), dict(block_tables=torch.zeros((2, 1))),
    dict(block_tables=torch.zeros(2, dtype=torch.int32)), dict(block_tables=torch.zeros((2, 2), dtype=torch.int32)[:, ::2]),
    dict(key_pool=TREE_CALL["key_pool"].float(), value_pool=TREE_CALL["value_pool"].float()),
    dict(key_pool=TREE_CALL["key_pool"].float()), dict(key_pool=TREE_CALL["key_pool"][:, :, :, :1]),
    dict(key_pool=TREE_CALL["key_pool"][:, :, :8], value_pool=TREE_CALL["value_pool"][:, :, :8]),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(new_keys=TREE_CALL["new_keys"].to("meta"))])
def test_tree_attention_refuses(no_gpu_check, monkeypatch, change):
    from memforge_amd.kernels.tree_attention import paged_attention_tree

    monkeypatch.setattr(nat, "device_cus", lambda _: 256)
    monkeypatch.setattr(nat._WORKSPACE, "partials", lambda n, dev: torch.empty(n))
    launches = []
    monkeypatch.setattr(nat, "_launch", lambda dev, what, *_: launches.append(what))
    plan = _plan()
    paged_attention_tree(**{**TREE_CALL, "plan": plan})
    assert launches == ["mf_tree_plan", "mf_tree_attention"]
    with pytest.raises((ValueError, TypeError)):
        paged_attention_tree(**{**TREE_CALL, "plan": plan, **change})
    assert len(launches) == 2


def test_tree_entry_points_check_sizes():
    import ctypes

    L, p = nat.lib(), 4096
    out = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(out)
    shape = [2, 3, 2, 4, 2, 64, 2, 256]
    assert L.mf_tree_plan_sizes(*shape, at, at + 8) == 0 and out[0] > 0 and out[1] > 0
    words, floats = out[0], out[1]
    for i, bad, status in ((0, -1, -1), (0, 4097, -1), (1, -1, -1), (2, 0, -1), (2, 1025, -1), (3, 3, -1), (4, 0, -1),
                           (5, 80, -2), (5, 0, -1), (6, 3, -1), (7, 0, -1), (7, 5000, -1)):
        args = list(shape)
        args[i] = bad
        assert L.mf_tree_plan_sizes(*args, at, at + 8) == status, (i, bad)
    plan = [p, p, p, 2, 3, 2, 16, 4, 2, 64, 2, 256, p, words, p, None]
    for i, bad, status in ((0, None, -1), (1, None, -1), (2, None, -1), (6, -1, -1), (12, None, -1), (12, p + 4, -1),
                           (13, words - 1, -3), (14, None, -1), (9, 48, -2)):
        args = list(plan)
        args[i] = bad
        assert L.mf_tree_plan(*args) == status, (i, bad)
    call = [p, 256, 64, p, 256, 64, 2, p, p, 2048, 128, 64, 16, 4, p, 1, p, p, 128, 64, 2, 3, 2, 4, 2, 64, 0.125, 256, p, words,
            p, floats, None]
    for i, bad, status in ((0, None, -1), (0, p + 2, -1), (1, 257, -1), (3, p + 8, -1), (5, 65, -1), (9, 2049, -1),
                           (10, 100, -1), (12, 0, -1), (13, 0, -1), (14, None, -1), (15, -1, -1), (16, None, -1),
                           (18, 4, -1), (25, 48, -2), (26, float("nan"), -1), (26, float("inf"), -1), (28, None, -1),
                           (29, words - 1, -3), (30, None, -1), (31, floats - 1, -3)):
        args = list(call)
        args[i] = bad
        assert L.mf_tree_attention(*args) == status, (i, bad)
