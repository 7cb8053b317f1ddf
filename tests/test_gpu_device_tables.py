"""DeviceBlockTables and accept_tree against plain loops on the host: whole numbers, all of them equal."""

from __future__ import annotations

import random

import pytest
import torch

from memforge_amd.runtime.device_tables import DeviceBlockTables
from memforge_amd.speculative import accept_tree

pytestmark = pytest.mark.gpu


class HostTables:
    def __init__(self, state: DeviceBlockTables):
        self.tables = state.tables.tolist()
        self.lens, self.held = state.lens.tolist(), state.held.tolist()
        self.free, self.bs = state.free.tolist(), state.block_size
        self.stack = self.free[:int(state.free_count)]
        self.width = state.tables.shape[1]

    def extend(self, new, max_rows, rows=None):
        slots, positions = [-1] * max_rows, [0] * max_rows
        cu, asked, refused = [0], 0, 0
        count = len(self.stack)
        for s, n in enumerate(new):
            n = max(n, 0)
            cu.append(cu[-1] + n)
            need = -(-(self.lens[s] + n) // self.bs)
            grow = max(need - self.held[s], 0)
            ok = need <= self.width and cu[-1] <= max_rows and (rows is None or n <= len(rows[s]))
            if ok:
                asked += grow
                ok = grow == 0 or asked <= count
            if ok:
                for j in range(grow):
                    self.tables[s][self.held[s] + j] = self.stack.pop()
                self.held[s] += grow
            refused += not ok
            for i in range(n):
                r = cu[s] + i if rows is None else rows[s][i] if i < len(rows[s]) else -1
                p = self.lens[s] + i
                if rows is None and r < max_rows:
                    positions[r] = p
                if ok and 0 <= r < max_rows:
                    positions[r] = p
                    slots[r] = self.tables[s][p // self.bs] * self.bs + p % self.bs
            if ok:
                self.lens[s] += n
        return slots, positions, cu, list(self.lens), [refused]

    def truncate(self, lengths):
        back = []
        for s, n in enumerate(lengths):
            self.lens[s] = min(max(n, 0), self.lens[s])
            keep = -(-self.lens[s] // self.bs)
            for j in range(keep, self.held[s]):
                back.append(self.tables[s][j])
                self.tables[s][j] = 0
            self.held[s] = min(self.held[s], keep)
        self.stack += back[::-1]

    def check(self, state: DeviceBlockTables):
        assert state.tables.tolist() == self.tables
        assert state.lens.tolist() == self.lens and state.held.tolist() == self.held
        assert int(state.free_count) == len(self.stack)
        assert state.free[:len(self.stack)].tolist() == self.stack


def ints(device, x):
    return torch.tensor(x, dtype=torch.int32).to(device)


def same(got, want):
    for name, x, y in zip(("slot_mapping", "positions", "cu_seqlens", "kv_lens", "refused"),
                          (got.slot_mapping, got.positions, got.cu_seqlens, got.kv_lens, got.refused), want):
        assert x.tolist() == y, name


@pytest.mark.parametrize("requests,blocks,width,bs,most", [
    (1, 4, 4, 16, 40), (3, 40, 12, 16, 30), (8, 60, 9, 1, 6), (17, 90, 30, 5, 60), (300, 700, 8, 32, 90),
    (257, 100, 4, 16, 20), (4096, 9000, 3, 8, 10), (40, 5000, 300, 7, 900)])
def test_rounds_of_growth_and_return(device, requests, blocks, width, bs, most):
    """Random rounds, some of which ask for more blocks, wider tables or more rows than there are."""
    rng = random.Random(requests)
    state = DeviceBlockTables.allocate(requests, width, blocks, bs, device)
    host = HostTables(state)
    for step in range(8):
        new = [rng.choice([0, 1, rng.randint(-3, most), rng.randint(0, most)]) for _ in range(requests)]
        total = sum(max(n, 0) for n in new)
        max_rows = rng.choice([total, total + 9, max(0, total - rng.randint(0, most))])
        same(state.extend(ints(device, new), max_rows), host.extend(new, max_rows))
        host.check(state)
        left = [rng.choice([0, n, n - rng.randint(0, most), n + 5]) for n in host.lens]
        state.truncate(ints(device, left))
        host.truncate(left)
        host.check(state)


def test_cut_back_restores_the_stack(device):
    state = DeviceBlockTables.allocate(9, 20, 150, 16, device)
    state.extend(ints(device, [5, 0, 70, 16, 17, 1, 33, 200, 8]), 400)
    before = [x.clone() for x in (state.tables, state.lens, state.held, state.free, state.free_count)]
    state.extend(ints(device, [17, 3, 64, 1, 0, 90, 16, 100, 9]), 400)
    state.truncate(before[1])
    for x, y in zip(before, (state.tables, state.lens, state.held, state.free, state.free_count)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("requests", [1, 5, 70])
def test_rows_given_by_number(device, requests):
    """The accepted rows of trees: every other row gets no slot."""
    rng = random.Random(requests)
    state = DeviceBlockTables.allocate(requests, 10, 8 * requests, 16, device)
    host = HostTables(state)
    total, most = 12 * requests + 3, 7
    for step in range(5):
        order = rng.sample(range(total), most * requests)
        rows = [order[s * most:(s + 1) * most] for s in range(requests)]
        new = [rng.randint(0, most + (step == 3)) for _ in range(requests)]
        for s in range(requests):
            for j in range(new[s], most):
                rows[s][j] = -1
        if requests > 1:
            rows[1][0] = rng.choice([-1, total, total + 5])
        same(state.extend(ints(device, new), total, ints(device, rows)), host.extend(new, total, rows))
        host.check(state)


def test_no_requests_and_no_rows(device):
    state = DeviceBlockTables.allocate(0, 4, 9, 16, device)
    got = state.extend(ints(device, []), 3)
    assert got.slot_mapping.tolist() == [-1] * 3 and got.cu_seqlens.tolist() == [0] and got.refused.tolist() == [0]
    state.truncate(ints(device, []))
    state = DeviceBlockTables.allocate(2, 0, 0, 16, device)
    got = state.extend(ints(device, [0, 3]), 0)
    assert got.kv_lens.tolist() == [0, 0] and got.refused.tolist() == [1]


def test_lengths_at_the_end_of_31_bits(device):
    """A length that 32 bits do not hold is refused; the one just below is not."""
    most = 2**31 - 1
    state = DeviceBlockTables(torch.zeros((2, 40), dtype=torch.int32, device=device), ints(device, [most - 3, most - 3]),
                              ints(device, [32, 32]), ints(device, [0]), ints(device, [0]), 1 << 26)
    got = state.extend(ints(device, [3, 4]), 10)
    assert got.kv_lens.tolist() == [most, most - 3] and got.refused.tolist() == [1]
    assert got.positions[:3].tolist() == [most - 3, most - 2, most - 1]


def test_largest_lengths(device):
    """Token counts whose sum passes 32 bits are refused, the requests before them served."""
    state = DeviceBlockTables.allocate(4, 6, 12, 16, device)
    got = state.extend(ints(device, [20, 2**31 - 1, 2**31 - 1, 5]), 64)
    assert got.refused.tolist() == [3] and got.kv_lens.tolist() == [20, 0, 0, 0]
    assert got.cu_seqlens.tolist() == [0, 20, 2**31 - 1, 2**31 - 1, 2**31 - 1]
    assert (got.slot_mapping[20:] == -1).all() and (got.slot_mapping[:20] >= 0).all()
    assert int(state.free_count) == 10


def test_captured_rounds(device):
    """Two graphs of the same state, replayed in turn between eager calls."""
    state = DeviceBlockTables.allocate(6, 40, 200, 16, device)
    new, left = ints(device, [9, 17, 0, 1, 30, 16]), ints(device, [0] * 6)
    state.extend(new, 80)
    state.truncate(left)  # warm
    host = HostTables(state)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(state.extend(new, 80))
        graphs.append(graph)
    for step in range(4):
        new.copy_(ints(device, [step, 3 * step, 1, 7, 16, 2]))
        want = host.extend(new.tolist(), 80)
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        same(outs[step % 2], want)
        host.check(state)
        left.copy_(ints(device, [n - 2 for n in host.lens]))
        state.truncate(left)
        host.truncate(left.tolist())
        same(state.extend(new, 90), host.extend(new.tolist(), 90))
        host.check(state)


# ----------------------------------------------------------------- accepted paths

def host_accept(tokens, targets, parents, cu, most):
    paths, out, counts = [], [], []
    for a, b in zip(cu[:-1], cu[1:]):
        n = min(b - a, most)
        path = []
        at = 0 if n > 0 else None
        while at is not None:
            path.append(a + at)
            at = next((i for i in range(at + 1, n) if parents[a + i] == at and tokens[a + i] == targets[path[-1]]), None)
        counts.append(len(path))
        out.append([targets[r] for r in path] + [-1] * (most - len(path)))
        paths.append(path + [-1] * (most - len(path)))
    return paths, out, counts


@pytest.mark.parametrize("nodes,most", [([1], 1), ([0, 4, 1, 0], 4), ([16] * 9, 16), ([64, 3, 65, 100], 100),
                                        ([1024, 5], 1024), ([30] * 300, 30), ([20, 20], 7)])
@pytest.mark.parametrize("vocab", [2, 5, 1 << 40])
def test_accepted_paths(device, nodes, most, vocab):
    rng = random.Random(sum(nodes) + vocab)
    cu, parents = [0], []
    for n in nodes:
        parents += [rng.choice([-1, i - 1, rng.randint(-1, i - 1), rng.randint(i, i + 9), -7]) if i else -1 for i in range(n)]
        cu.append(cu[-1] + n)
    tokens = [rng.randrange(vocab) for _ in parents]
    targets = [rng.randrange(vocab) for _ in parents]
    if vocab > 5:  # chains that go on for long
        for a, b in zip(cu[:-1], cu[1:]):
            for r in range(a + 1, b):
                if 0 <= parents[r] < r - a and rng.random() < 0.9:
                    tokens[r] = targets[a + parents[r]]
    got = accept_tree(torch.tensor(tokens).to(device), torch.tensor(targets).to(device), ints(device, parents),
                      ints(device, cu), most)
    want = host_accept(tokens, targets, parents, cu, most)
    assert got.path.tolist() == want[0] and got.tokens.tolist() == want[1] and got.count.tolist() == want[2]


def test_rows_out_of_bounds_are_no_tree(device):
    n = 6
    got = accept_tree(torch.zeros(n, dtype=torch.int64).to(device), torch.zeros(n, dtype=torch.int64).to(device),
                      ints(device, [-1, 0, 1, -1, 0, 1]), ints(device, [0, 3, -5, 9, 5]), 4)
    assert got.count.tolist() == [3, 0, 0, 0]
    assert got.path[0].tolist() == [0, 1, 2, -1] and (got.path[1:] == -1).all() and (got.tokens[1:] == -1).all()
