"""DeviceBlockTables.extend with rows given by number, of which there are none."""

from __future__ import annotations

import pytest
import torch

from memforge_amd import _native as nat
from memforge_amd.runtime.device_tables import DeviceBlockTables


def test_no_columns_is_not_no_rows(monkeypatch):
    calls = []
    monkeypatch.setattr(nat, "require_device", lambda *_: None)
    monkeypatch.setattr(nat, "_stream", lambda *_: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(nat, "_launch", lambda dev, what, fn, *a: calls.append(a))
    state = DeviceBlockTables.allocate(2, 3, 4, 16, "cpu")
    new = torch.tensor([1, 2], dtype=torch.int32)
    state.extend(new, 5)
    state.extend(new, 5, rows=torch.zeros((2, 0), dtype=torch.int32))
    assert calls[0][12:15] == (None, 0, 0)
    assert calls[1][12] and calls[1][13:15] == (0, 0)


@pytest.mark.gpu
def test_requests_that_need_rows_are_refused(device):
    state = DeviceBlockTables.allocate(3, 3, 9, 16, device)
    got = state.extend(torch.tensor([2, 0, 1], dtype=torch.int32).to(device), 4,
                       rows=torch.zeros((3, 0), dtype=torch.int32, device=device))
    assert int(got.refused) == 2 and got.kv_lens.tolist() == [0, 0, 0] and got.slot_mapping.tolist() == [-1] * 4
    assert int(state.free_count) == 9 and state.held.tolist() == [0, 0, 0]
