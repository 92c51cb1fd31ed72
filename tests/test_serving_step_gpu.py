"""A server's steps over 4-bit caches as they would be used: tables, prelude, append and attention together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle
from simpler_amd import kv_cache
from simpler_amd import paged_attention as pa
from simpler_amd.workloads import rope_tables
from tests.int4_cases import REL, rel_l2

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HEADS, HKV, DIM, GROUP, BLOCK, WIDTH, POOL, BATCH = 8, 2, 128, 64, 16, 8, 40, 5
SECTIONS = (16, 24, 24)


class Server:
    def __init__(self, device):
        i32 = lambda *s, v=0: torch.full(s, v, dtype=torch.int32, device=device)  # noqa: E731
        self.device = device
        self.pools = kv_cache.alloc_kv4_pools(POOL, BLOCK, HKV, DIM, GROUP, device=device)
        for t in self.pools:
            t.view(torch.uint8).fill_(0xFF)  # NaN scales wherever nothing was written
        self.table, self.lens, self.count = i32(BATCH, WIDTH, v=-1), i32(BATCH), i32(1, v=POOL)
        self.free = torch.arange(POOL, dtype=torch.int32, device=device)
        self.cos, self.sin = (t.to(device) for t in rope_tables(WIDTH * BLOCK, DIM))
        self.qw, self.kw = torch.ones(DIM, device=device), torch.ones(DIM, device=device)
        self.errors = i32(1)

    def prelude(self, qkv, step):
        """q, k and v rows at the step's positions (text: every axis alike)."""
        q, k, v = qkv.split([HEADS * DIM, HKV * DIM, HKV * DIM], 1)
        rows = torch.empty((2, qkv.shape[0], HKV, DIM), dtype=BF16, device=self.device)
        q = kv_cache.qk_norm_mrope_append(q, k, v, step.positions.expand(3, -1).contiguous(), SECTIONS, self.cos, self.sin,
                                          None, rows[0], rows[1], HEADS, q_norm_weight=self.qw, k_norm_weight=self.kw,
                                          error_count=self.errors)
        return q, rows[0], rows[1]

    def tables(self, ended, new, num_tokens):
        freed = kv_cache.release_blocks(ended, self.lens, self.table, self.free, self.count, BLOCK, self.errors)
        step = kv_cache.assign_slots(new, freed.context_lens, self.table, self.free, freed.free_count, BLOCK, num_tokens,
                                     self.errors)
        self.lens.copy_(step.context_lens)
        self.count.copy_(step.free_count)
        return step

    def reference(self, q):
        k = kv4_oracle.pages_to_rows(self.pools[0].cpu().numpy(), self.pools[2].cpu().numpy(), False)
        v = kv4_oracle.pages_to_rows(self.pools[1].cpu().numpy(), self.pools[3].cpu().numpy(), True)
        return kv4_oracle.attention(q.float().cpu().numpy()[:, None], k, v, self.table.cpu().numpy(),
                                    self.lens.cpu().numpy(), DIM**-0.5)[:, 0]


def test_prompts_then_decodes(device):
    s, gen = Server(device), torch.Generator("cuda").manual_seed(1)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    written = [np.zeros((0, HKV, DIM))] * BATCH  # what each request's cache stands for
    steps = [([0] * 5, [30, 1, 0, 47, 16]), ([0] * 5, [1, 1, 0, 1, 1]), ([0, 0, 0, 1, 0], [1, 1, 60, 0, 1]),
             ([0] * 5, [1, 1, 1, 33, 1]), ([1, 0, 0, 0, 0], [0, 1, 1, 1, 1]), ([0] * 5, [5, 1, 1, 1, 1])]
    for ended, new in steps:
        total = sum(new)
        step = s.tables(i32(ended), i32(new), total + 3)  # three places of padding
        assert step.granted.cpu().tolist() == new
        qkv = torch.randn((total + 3, (HEADS + 2 * HKV) * DIM), generator=gen, device=device).to(BF16)
        q, k, v = s.prelude(qkv, step)
        kv_cache.kv4_append(k, v, step.slot_mapping, *s.pools, error_count=s.errors)
        codes = kv4_oracle.dequantise(*kv4_oracle.quantise(k.float().cpu().numpy(), GROUP))
        for b in range(BATCH):
            at = step.starts.cpu().tolist()
            before = written[b][:0] if ended[b] else written[b]
            written[b] = np.concatenate([before, codes[at[b]:at[b + 1]]])
        # the decode of each request's last token over everything it has
        last = (step.starts[1:] - 1).clamp(min=0).long()
        out = pa.paged_attention_decode(q[last], s.pools[0], s.pools[1], s.table, s.lens, out_dtype=torch.float32,
                                        k_scale=s.pools[2], v_scale=s.pools[3])
        pa.check_errors(device)
        assert rel_l2(out.cpu().numpy(), s.reference(q[last])) <= REL[torch.float32]
        # and each request's keys, read back from wherever they lie
        lens = s.lens.cpu().tolist()
        for b in range(BATCH):
            assert lens[b] == len(written[b])
            pos = torch.arange(lens[b], device=device)
            slots = (s.table[b, pos // BLOCK] * BLOCK + pos % BLOCK).to(torch.int32)
            got = kv_cache.kv4_gather(slots, *s.pools, dtype=torch.float32)[0].cpu().numpy()
            np.testing.assert_allclose(got, written[b], rtol=2.0**-23, atol=0)
    assert s.errors.item() == 0


def test_decode_step_as_one_graph(device):
    """Tables, prelude and the append-and-decode of a step captured once and replayed, against the same calls made eagerly."""
    eager, graphed = Server(device), Server(device)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    gen = torch.Generator("cuda").manual_seed(2)
    none, start = i32([0] * BATCH), i32([20, 33, 16, 1, 47])
    prompt = torch.randn((117, (HEADS + 2 * HKV) * DIM), generator=gen, device=device).to(BF16)
    for s in (eager, graphed):
        step = s.tables(none, start, 117)
        _, k, v = s.prelude(prompt, step)
        kv_cache.kv4_append(k, v, step.slot_mapping, *s.pools)

    def decode(s, qkv, ones, out):
        step = s.tables(none, ones, BATCH)
        q, k, v = s.prelude(qkv, step)
        return pa.paged_attention_decode_append(q, s.pools[0], s.pools[1], s.table, s.lens, k, v, out,
                                                k_scale=s.pools[2], v_scale=s.pools[3])

    ones, qkv = i32([1] * BATCH), torch.zeros((BATCH, (HEADS + 2 * HKV) * DIM), dtype=BF16, device=device)
    out = torch.empty((BATCH, HEADS, DIM), dtype=torch.float32, device=device)
    state = (graphed.table, graphed.free, graphed.lens, graphed.count, *graphed.pools)
    saved = [t.clone() for t in state]
    stream = torch.cuda.Stream(device)
    torch.cuda.synchronize(device)
    with torch.cuda.stream(stream):
        decode(graphed, qkv, ones, out)  # sizes the workspace
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            decode(graphed, qkv, ones, out)
    torch.cuda.synchronize(device)
    for t, was in zip(state, saved):
        t.copy_(was)
    for i in range(20):
        new = torch.randn(qkv.shape, generator=gen, device=device).to(BF16)
        qkv.copy_(new)
        want = decode(eager, new, ones, torch.empty_like(out))
        torch.cuda.synchronize(device)
        graph.replay()
        torch.cuda.synchronize(device)
        assert torch.equal(out, want), i
        assert torch.equal(graphed.table, eager.table) and torch.equal(graphed.lens, eager.lens)
    for a, b in zip(graphed.pools, eager.pools):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    q = torch.randn((BATCH, HEADS, DIM), generator=gen, device=device).to(BF16)
    got = pa.paged_attention_decode(q, graphed.pools[0], graphed.pools[1], graphed.table, graphed.lens,
                                    k_scale=graphed.pools[2], v_scale=graphed.pools[3])
    assert rel_l2(got.cpu().numpy(), graphed.reference(q)) <= REL[torch.float32]
    assert eager.errors.item() == graphed.errors.item() == 0
