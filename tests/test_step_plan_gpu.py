"""A step's block tables and slot maps built on the GPU (``kv_cache.release_blocks``, ``kv_cache.assign_slots``)
against the request-by-request oracle: every output, equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle
from simpler_amd import kv_cache

pytestmark = pytest.mark.gpu


class State:
    """A pool, its free list and the rows of some requests, on the host."""

    def __init__(self, lens, block, width, pool, seed=0):
        rng = np.random.default_rng(seed)
        self.lens, self.block, self.rng = np.array(lens, np.int64).reshape(-1), block, rng
        perm = rng.permutation(pool)
        self.table = np.full((len(self.lens), width), -1)
        at = 0
        for b, n in enumerate(self.lens):
            k = -(-int(min(max(n, 0), width * block)) // block)
            self.table[b, :k] = perm[at:at + k]
            at += k
        self.free = np.full(pool, -1)
        self.free[:pool - at] = perm[at:]
        self.count = pool - at


def i32(a, device):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=device)


def check_assign(s: State, new, num_tokens, device, refused=None):
    table, free = i32(s.table, device), i32(s.free, device)
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    want = kv4_oracle.assign_slots(np.asarray(new), s.lens, s.table, s.free, s.count, s.block, num_tokens)
    for _ in range(2):  # the same call again: the same results
        got = kv_cache.assign_slots(i32(new, device), i32(s.lens, device), table, free, i32([s.count], device), s.block,
                                    num_tokens, errors)
        for name, g, w in zip(("slots", "positions", "requests", "starts", "lens", "granted"), got, want):
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
        assert got.free_count.item() == want[6]
        np.testing.assert_array_equal(table.cpu().numpy(), want[7])
        np.testing.assert_array_equal(free.cpu().numpy(), s.free)
    if refused is not None:
        assert errors.item() == 2 * refused
    return want


def test_decode_step(device):
    s = State([15, 16, 17, 1, 160, 0], 16, 12, 40)
    check_assign(s, [1, 1, 1, 1, 1, 0], 5, device, refused=0)


@pytest.mark.parametrize("block", [1, 5, 16, 128, 1000])
@pytest.mark.parametrize("batch", [1, 2, 63, 511, 513, 1500, 4096])
def test_random_steps(batch, block, device):
    rng = np.random.default_rng(batch * 7 + block)
    lens, new = rng.integers(0, 60, batch), rng.integers(0, 3, batch) * rng.integers(0, 40, batch)
    width = -(-130 // block)
    need = int((-(-(lens + new) // block)).sum())
    for pool in (need + 3, need - need // 5):  # enough blocks, and too few for the last requests
        s = State(lens, block, width, max(pool, int((-(-lens // block)).sum())), seed=batch)
        for tokens in (int(new.sum()), int(new.sum()) + 9, int(new.sum()) * 2 // 3):
            check_assign(s, new, tokens, device)


def test_requests_that_are_refused(device):
    s = State([10, 30, 5, 64, 2, 7], 16, 4, 14, seed=1)
    s.lens[2] = -3
    # past the table row; a negative length; exactly the row; a negative count; more than any pool
    check_assign(s, [1, 40, 1, 0, -2, 57], 100, device, refused=3)
    check_assign(s, [1, 2**31 - 1, 0, 0, 2**31 - 1, 57], 100, device)
    # a request that does not fit the free list; later ones that need no block still go
    s = State([15, 15, 14, 15], 16, 9, 6, seed=2)
    assert s.count == 2
    want = check_assign(s, [1, 50, 2, 1], 60, device, refused=1)
    assert want[5].tolist() == [1, 0, 2, 1]
    # one that needs a block after it does not: it would pass the refused one
    want = check_assign(s, [2, 50, 2, 2], 60, device, refused=2)
    assert want[5].tolist() == [2, 0, 2, 0]


def test_lengths_and_slots_at_the_end_of_32_bits(device):
    """A table row that holds more tokens than a length counts; a block id whose slot passes 2^31 - 1."""
    s = State([3, 3], 4096, 2**19 + 8, 16, seed=5)
    s.lens[0] = 2**31 - 11
    s.table[0, -16:] = 0
    want = check_assign(s, [10, 2], 30, device, refused=0)
    assert want[4][0] == 2**31 - 1
    assert check_assign(s, [11, 2], 30, device, refused=1)[5].tolist() == [0, 2]
    s = State([1, 1], 16, 4, 8, seed=6)
    s.table[0, 0] = 2**27
    assert check_assign(s, [3, 3], 6, device, refused=0)[0][0] == 2**31 - 1
    # prompts whose sum passes 32 bits: those after it have no place
    s = State([0] * 6, 16, 4, 8, seed=7)
    check_assign(s, [2**31 - 1, 5, 2**31 - 1, 2**31 - 1, 3, 0], 40, device)


def test_free_count_outside_the_list(device):
    s = State([3, 3], 4, 5, 8, seed=3)
    for count, clamped in ((-5, 0), (1000, 8)):
        got = kv_cache.assign_slots(i32([2, 2], device), i32(s.lens, device), i32(s.table, device), i32(s.free, device),
                                    i32([count], device), 4, 4)
        want = kv4_oracle.assign_slots(np.array([2, 2]), s.lens, s.table, s.free, clamped, 4, 4)
        np.testing.assert_array_equal(got.slot_mapping.cpu().numpy(), want[0])
        assert got.free_count.item() == want[6]


def test_long_prompts_and_wide_rows(device):
    """A million tokens over 40,000 table entries each."""
    s = State([0, 12345, 0], 16, 40000, 70000, seed=4)
    check_assign(s, [500000, 100001, 400000], 1000001, device, refused=0)


def test_no_requests_and_no_tokens(device):
    s = State([], 16, 4, 8)
    check_assign(s, [], 0, device, refused=0)
    check_assign(s, [], 5, device, refused=0)
    check_assign(State([5, 40], 16, 4, 8), [0, 0], 0, device, refused=0)
    released = kv_cache.release_blocks(i32([], device), i32([], device), i32(s.table, device), i32(s.free, device),
                                       i32([3], device), 16)
    assert released.free_count.item() == 3 and released.context_lens.numel() == 0


@pytest.mark.parametrize("batch", [1, 5, 64, 700, 4096])
def test_release(batch, device):
    rng = np.random.default_rng(batch)
    for block, share in ((16, 0.3), (7, 1.0), (128, 0.0)):
        lens = rng.integers(0, 300, batch)
        s = State(lens, block, -(-300 // block), int((-(-lens // block)).sum()) + 11, seed=batch)
        ended = rng.random(batch) < share
        free, errors = i32(s.free, device), torch.zeros(1, dtype=torch.int32, device=device)
        want = kv4_oracle.release_blocks(ended, s.lens, s.table, s.free, s.count, block)
        for _ in range(2):
            got = kv_cache.release_blocks(i32(ended * 3, device), i32(s.lens, device), i32(s.table, device), free,
                                          i32([s.count], device), block, errors)
            np.testing.assert_array_equal(got.context_lens.cpu().numpy(), want[0])
            np.testing.assert_array_equal(free.cpu().numpy(), want[1])
            assert got.free_count.item() == want[2] and errors.item() == 0


def test_release_of_bad_lengths_and_into_a_full_list(device):
    s = State([40, 64, 10], 16, 4, 8, seed=5)
    lens = np.array([-4, 1000, 10])
    free, errors = i32(np.full(6, -1), device), torch.zeros(1, dtype=torch.int32, device=device)
    got = kv_cache.release_blocks(i32([1, 1, 1], device), i32(lens, device), i32(s.table, device), free,
                                  i32([3], device), 16, errors)
    # nothing of the first, four of the second, of which three fit
    assert errors.item() == 3 and got.free_count.item() == 6
    assert free.cpu().tolist() == [-1] * 3 + s.table[1, :3].tolist()
    assert got.context_lens.cpu().tolist() == [0, 0, 0]


def test_many_steps_of_a_server(device):
    """Requests come, decode and end over 60 steps: no block is held twice or lost, and the oracle agrees."""
    rng = np.random.default_rng(6)
    block, width, pool, batch = 16, 8, 90, 24
    s = State([0] * batch, block, width, pool, seed=7)
    table, free = i32(s.table, device), i32(s.free, device)
    lens, count = i32(s.lens, device), i32([s.count], device)
    host_lens, host_table, host_free, host_count = s.lens, s.table, s.free, s.count
    for _ in range(60):
        ended = (host_lens > 0) & (rng.random(batch) < 0.15)
        new = np.where(ended, 0, np.where(host_lens > 0, 1, rng.integers(0, 50, batch)))
        freed = kv_cache.release_blocks(i32(ended, device), lens, table, free, count, block)
        step = kv_cache.assign_slots(i32(new, device), freed.context_lens, table, free, freed.free_count, block, 400)
        lens, count = step.context_lens, step.free_count
        host_lens, host_free, host_count = kv4_oracle.release_blocks(ended, host_lens, host_table, host_free, host_count,
                                                                     block)
        want = kv4_oracle.assign_slots(new, host_lens, host_table, host_free, host_count, block, 400)
        np.testing.assert_array_equal(step.slot_mapping.cpu().numpy(), want[0])
        host_lens, host_count, host_table = want[4], want[6], want[7]
        np.testing.assert_array_equal(lens.cpu().numpy(), host_lens)
        assert count.item() == host_count
        used = [int(x) for b in range(batch) for x in host_table[b, :-(-int(host_lens[b]) // block)]]
        assert sorted(used + host_free[:host_count].tolist()) == list(range(pool))


def test_captured_graph(device):
    """A captured step, replayed with other lengths, with the state carried over by copies inside the graph."""
    s = State([5, 31, 0, 16], 16, 6, 24, seed=8)
    table, free, count = i32(s.table, device), i32(s.free, device), i32([s.count], device)
    lens, new, ended = i32(s.lens, device), i32([1, 1, 20, 1], device), i32([0, 0, 0, 0], device)
    stream = torch.cuda.Stream(device)
    state = [t.clone() for t in (table, free, count, lens)]
    with torch.cuda.stream(stream):
        def step():
            freed = kv_cache.release_blocks(ended, lens, table, free, count, 16)
            r = kv_cache.assign_slots(new, freed.context_lens, table, free, freed.free_count, 16, 30)
            lens.copy_(r.context_lens)
            count.copy_(r.free_count)
            return r
        step()
        for t, saved in zip((table, free, count, lens), state):
            t.copy_(saved)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            result = step()
    for t, saved in zip((table, free, count, lens), state):
        t.copy_(saved)
    host = (s.lens, s.table, s.free, s.count)
    for step_new, step_ended in (([1, 1, 20, 1], [0] * 4), ([0, 1, 1, 1], [1, 0, 0, 0]), ([25, 1, 0, 1], [0, 0, 1, 0]),
                                 ([1, 1, 1, 1], [0] * 4)):
        new.copy_(i32(step_new, device))
        ended.copy_(i32(step_ended, device))
        torch.cuda.synchronize(device)
        graph.replay()
        torch.cuda.synchronize(device)
        a = kv4_oracle.release_blocks(np.array(step_ended), host[0], host[1], host[2], host[3], 16)
        w = kv4_oracle.assign_slots(np.array(step_new), a[0], host[1], a[1], a[2], 16, 30)
        np.testing.assert_array_equal(result.slot_mapping.cpu().numpy(), w[0])
        np.testing.assert_array_equal(table.cpu().numpy(), w[7])
        host = (w[4], w[7], a[1], w[6])
        assert count.item() == host[3]
