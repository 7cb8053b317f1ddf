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
    sample = [p, 0, 10, 2, 10, p, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, None]
    for at, bad in ((0, None), (1, 3), (2, -1), (3, -1), (4, 0), (4, nat.SAMPLE_MAX_VOCAB + 1), (5, None), (14, None)):
        args = list(sample)
        args[at] = bad
        assert L.mf_sample(*args) == -1, (at, bad)
    accept = [p, p, p, p, 2, 6, 4, p, p, p, None]
    for at, bad in ((0, None), (3, None), (4, -1), (5, -1), (6, 0), (6, 1025), (7, None), (9, None)):
        args = list(accept)
        args[at] = bad
        assert L.mf_tree_accept(*args) == -1, (at, bad)
