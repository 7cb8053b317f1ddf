"""Calls at the edges of scored attention: caps of any size beside slots that no row sees, rows at negative positions."""

from __future__ import annotations

import pytest
import torch

from memforge_amd import _native as nat
from tests.scored_reference import attend, check
from tests.test_gpu_kv4 import Step4
from tests.test_gpu_scored import DECODES, PREFILLS, Step, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [float("nan"), float("inf"), 1e4])
@pytest.mark.parametrize("cap", [300.0, 1e4, 1e6, 1e12])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128)])
def test_caps_beside_slots_no_row_sees(device, dtype, d, cap, hidden):
    """What a score becomes does not hang on what the slots past the context hold. No score comes near a cap of 300 or
    more here, so each is within a relative 5.5e-7 (the polynomials' error and their roundings), which the bound counts as
    2e-7 of a cap of 4 |t|."""
    st = Step(device, dtype, 6, 2, d, 16, DECODES + PREFILLS, seed=11)
    flat_k, flat_v = (x.view(-1, 2, d) for x in (st.kp, st.vp))
    used = torch.zeros(flat_k.shape[0], dtype=torch.bool)
    for i in range(len(st.runs)):
        used[st.slots(i, 0, st.kv[i])] = True
    flat_k[~used.to(device)] = hidden
    flat_v[~used.to(device)] = hidden
    out = st.run(st.scoring(cap))
    cpu_k, cpu_v = flat_k.cpu(), flat_v.cpu()
    for i, (_, start, n, _) in enumerate(st.runs):
        at, rows = st.slots(i, 0, st.kv[i]), slice(st.cu[i], st.cu[i + 1])
        ref = attend(st.q[rows], cpu_k[at], cpu_v[at], range(start, start + n), st.scale, cap)
        check(out[rows], *ref, dtype, d, st.kv[i], min(cap, 4 * float(ref[2][..., 1].max())), f"cap {cap} run {i}")


@pytest.mark.parametrize("hidden", [float("nan"), 1e4])
@pytest.mark.parametrize("bits,dtype,d,bs", [(16, torch.bfloat16, 64, 16), (16, torch.float16, 128, 16), (16, torch.bfloat16, 128, 32),
                                             (16, torch.float32, 64, 16), (16, torch.float16, 256, 16), (4, torch.bfloat16, 64, 16),
                                             (4, torch.float16, 128, 32), (4, torch.bfloat16, 256, 16)])
def test_hidden_slots_change_no_bit(device, bits, dtype, d, bs, hidden):
    """The same call over the same keys, other values in the slots that no row sees: the same bits."""
    runs = DECODES + [(0, 0, 37, 0), (21, 45, 80, 0), (70, 200, 1, 0), (333, 600, 1, 0), (130, 250, 33, 0), (5, 40, 1, 0)]
    st = (Step4 if bits == 4 else Step)(device, dtype, 6, 2, d, bs, runs, seed=12)
    k, v = (st.k, st.v) if bits == 4 else (x.view(-1, 2, d) for x in (st.kp, st.vp))
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for i, (first, *_) in enumerate(runs):
        used[st.slots(i, first, st.kv[i])] = True
    outs = []
    for fill in (0.0, hidden):
        k[~used.to(k.device)], v[~used.to(v.device)] = fill, fill
        if bits == 4:
            st.write()
        outs.append([st.run(st.scoring(cap, slopes_of(6, device))) for cap in (30.0, 1e6)])
    for a, b in zip(*outs):
        assert torch.isfinite(a).all() and torch.equal(a, b)


NEGATIVE_RUNS = [(0, 200, 1, 0), (0, 0, 40, 0), (0, 2000, 1, 0), (0, 900, 60, 0), (0, 2100, 3, 0)]


def _at_negative_positions(st, device):
    """Every third row of each run, and all of the first one's, lie at position -1."""
    for i in range(len(st.runs)):
        for r in range(st.cu[i], st.cu[i + 1]):
            if i == 0 or (r - st.cu[i]) % 3 == 1:
                st.positions[r] = -1
    st.pos_t = torch.tensor(st.positions, dtype=torch.int64, device=device)


@pytest.mark.parametrize("dtype,d,bits", [(torch.bfloat16, 64, 16), (torch.float16, 128, 16), (torch.float32, 64, 16),
                                          (torch.bfloat16, 256, 16), (torch.bfloat16, 64, 4), (torch.float16, 256, 4)])
@pytest.mark.parametrize("tiles", [0, 8])
def test_rows_at_negative_positions_get_zeros(device, dtype, d, bits, tiles):
    st = (Step4 if bits == 4 else Step)(device, dtype, 6, 2, d, 16, NEGATIVE_RUNS, seed=13)
    _at_negative_positions(st, device)
    plan = st.plan(partition_tiles=tiles)
    if tiles:
        assert plan.n_merges > 0
    # partials of an earlier call must not be taken for this one's
    nat._WORKSPACE.partials(max(plan.partials_floats, 1), device).fill_(float("nan"))
    out = st.run(st.scoring(30.0), plan).cpu().double()
    seen = torch.tensor(st.positions) >= 0
    assert (out[~seen] == 0).all()
    assert torch.isfinite(out[seen]).all()
    if bits == 16:
        for i in range(len(st.runs)):
            rows = slice(st.cu[i], st.cu[i + 1])
            at = st.slots(i, 0, st.kv[i])
            k, v = (x.view(-1, 2, d).cpu()[at] for x in (st.kp, st.vp))
            check(out[rows], *attend(st.q[rows], k, v, st.positions[rows], st.scale, 30.0), dtype, d, st.kv[i], 30.0, f"run {i}")
