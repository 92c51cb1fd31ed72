"""The prelude with rotary positions of several axes (``kv_cache.qk_norm_mrope_append``) on the GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle
from simpler_amd import kv_cache
from simpler_amd.workloads import rope_tables

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


class Case:
    def __init__(self, tokens, heads, hkv, dim, sections, *, interleaved=False, proj=FP32, dtype=BF16, norm=True, seed=0,
                 block=16, device=None):
        gen = torch.Generator().manual_seed(seed)
        self.sections, self.interleaved, self.heads, self.dim, self.hkv, self.dtype = (
            sections, interleaved, heads, dim, hkv, dtype)
        qkv = torch.randn((tokens, (heads + 2 * hkv) * dim), generator=gen).to(proj)
        self.q, self.k, self.v = qkv.to(device).split([heads * dim, hkv * dim, hkv * dim], 1)
        self.pos = torch.randint(0, 300, (len(sections), tokens), generator=gen, dtype=torch.int32)
        self.cos, self.sin = rope_tables(300, dim)
        self.inv = 0.5 + torch.rand(tokens, generator=gen) if norm else None
        self.qw = 1 + 0.1 * torch.randn(dim, generator=gen) if norm else None
        self.kw = 1 + 0.1 * torch.randn(dim, generator=gen) if norm else None
        n = (tokens + block - 1) // block + 1
        self.slots = torch.randperm(n * block, generator=gen)[:tokens].to(torch.int32)
        self.caches = [torch.full((n, block, hkv, dim), 7.0, dtype=dtype, device=device) for _ in range(2)]
        self.device, self.tokens, self.block = device, tokens, block

    def run(self, **kw):
        d = lambda t: None if t is None else t.to(self.device)  # noqa: E731
        args = dict(q_proj=self.q, k_proj=self.k, v_proj=self.v, positions=d(self.pos), sections=self.sections,
                    rope_cos=d(self.cos), rope_sin=d(self.sin), slot_mapping=d(self.slots), key_cache=self.caches[0],
                    value_cache=self.caches[1], num_heads=self.heads, interleaved=self.interleaved, inv_rms=d(self.inv),
                    q_norm_weight=d(self.qw), k_norm_weight=d(self.kw))
        return kv_cache.qk_norm_mrope_append(**(args | kw))

    def want(self):
        f = lambda t: t.float().cpu().numpy().reshape(self.tokens, -1, self.dim)  # noqa: E731
        n = lambda t: None if t is None else t.numpy()  # noqa: E731
        turn = lambda x, w: kv4_oracle.mrope(f(x), self.pos.numpy(), self.sections, self.cos.numpy(), self.sin.numpy(),  # noqa: E731
                                             self.interleaved, n(self.inv), n(w))
        v = f(self.v).astype(np.float64) * (1 if self.inv is None else self.inv.numpy().astype(np.float64)[:, None, None])
        return turn(self.q, self.qw), turn(self.k, self.kw), v

    def rows(self):
        at = self.slots.long().to(self.device)
        return [c[at // self.block, at % self.block] for c in self.caches]


def close(got, want, dtype):
    """Half a step of the output type at the value, and fp32's rounding (products, norm: 2^-20 of the row's largest)."""
    got, want = got.double().cpu().numpy(), np.asarray(want)
    bound = np.abs(want) * torch.finfo(dtype).eps / 2 * 1.01 + np.abs(want).max(-1, keepdims=True) * 2.0**-20
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)


SECTIONS = {64: [[32], [12, 10, 10], [16, 16], [8, 8, 8, 8], [0, 20, 12]], 128: [[64], [16, 24, 24], [40, 24], [16, 16, 16, 16]],
            256: [[128], [44, 42, 42], [100, 28]], 80: [[40], [14, 13, 13]], 6: [[3], [1, 1, 1]], 130: [[65], [33, 32]],
            1024: [[512], [200, 156, 156]]}


@pytest.mark.parametrize("dim", sorted(SECTIONS))
@pytest.mark.parametrize("proj", [FP32, BF16, FP16])
def test_sections(dim, proj, device):
    for i, sections in enumerate(SECTIONS[dim]):
        for dtype in (BF16, FP16):
            for norm in (True, False):
                c = Case(5, 6, 2, dim, sections, proj=proj, dtype=dtype, norm=norm, seed=i, device=device)
                q = c.run()
                wq, wk, wv = c.want()
                k, v = c.rows()
                close(q, wq, dtype)
                close(k, wk, dtype)
                close(v, wv, dtype)
                assert sum((t != 7.0).any(-1).sum().item() for t in c.caches) == 2 * 5 * 2  # no other row


@pytest.mark.parametrize("dim,sections", [(64, [12, 10, 10]), (128, [24, 20, 20]), (256, [44, 42, 42]), (128, [32, 32]),
                                          (80, [14, 13, 13]), (128, [40, 8, 8, 8]), (128, [64])])
def test_interleaved(dim, sections, device):
    c = Case(9, 5, 1, dim, sections, interleaved=True, device=device)
    q = c.run()
    wq, wk, wv = c.want()
    close(q, wq, BF16)
    close(c.rows()[0], wk, BF16)
    close(c.rows()[1], wv, BF16)


@pytest.mark.parametrize("tokens,heads,hkv,dim", [(1, 1, 1, 128), (3, 7, 1, 64), (257, 28, 4, 128), (4100, 5, 5, 64),
                                                 (1500, 16, 2, 256), (70, 1, 3, 128)])
def test_tokens_and_heads(tokens, heads, hkv, dim, device):
    """Few tokens (a set of heads per wave) to many (all of a token's heads in one)."""
    half = dim // 2
    c = Case(tokens, heads, hkv, dim, [half - 2 * (half // 3), half // 3, half // 3], proj=BF16, seed=tokens, device=device)
    q = c.run()
    wq, wk, wv = c.want()
    close(q, wq, BF16)
    close(c.rows()[0], wk, BF16)
    close(c.rows()[1], wv, BF16)


def test_one_axis_is_the_plain_prelude(device):
    c = Case(33, 8, 2, 128, [64], seed=3, device=device)
    q = c.run()
    mine = [t.clone() for t in c.caches]
    for t in c.caches:
        t.fill_(7.0)
    d = lambda t: t.contiguous().to(device)  # noqa: E731
    q2 = kv_cache.qk_norm_rope_append(d(c.q), d(c.k), d(c.v), d(c.inv), d(c.qw), d(c.kw), d(c.cos), d(c.sin),
                                      d(c.pos[0] + 1), d(c.slots), *c.caches, num_heads=8)
    # the norm's sum runs in another order: a step of bf16 at most, rarely
    for a, b in zip((q, *mine), (q2, *c.caches)):
        assert ((a.float() - b.float()).abs() <= b.float().abs() * 2.0**-7).all()
        assert (a != b).float().mean() < 1e-3


def test_rows_instead_of_caches(device):
    c = Case(40, 6, 2, 64, [12, 10, 10], dtype=FP16, seed=4, device=device)
    q = c.run()
    rows = torch.full((40, 3, 2, 64), 9.0, dtype=FP16, device=device)
    q2 = c.run(slot_mapping=None, key_cache=rows[:, 0], value_cache=rows[:, 2])
    assert torch.equal(q, q2) and (rows[:, 1] == 9).all()
    assert torch.equal(rows[:, 0], c.rows()[0]) and torch.equal(rows[:, 2], c.rows()[1])


def test_some_of_the_steps_before_the_turn(device):
    """inv_rms and each norm weight on its own."""
    for drop in ("inv", "qw", "kw"):
        c = Case(12, 4, 2, 128, [16, 24, 24], seed=5, device=device)
        setattr(c, drop, None)
        q = c.run()
        wq, wk, wv = c.want()
        close(q, wq, BF16)
        close(c.rows()[0], wk, BF16)
        close(c.rows()[1], wv, BF16)


@pytest.mark.parametrize("dim", [128, 80])
def test_padding_and_positions_outside_the_tables(dim, device):
    half = dim // 2
    c = Case(8, 4, 2, dim, [half - 20, 20, 0], seed=6, device=device)
    c.pos[0, 1] = -1  # padding, whatever the rest says
    c.pos[1, 1] = 10**6
    c.pos[0, 2] = 300
    c.pos[1, 3] = -7
    c.pos[2, 4] = 10**6  # an axis without pairs
    c.slots[5] = -1
    c.slots[6] = 10**6
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    q = c.run(error_count=errors)
    assert errors.item() == 3
    good = [0, 4, 5, 6, 7]
    assert (q[[1, 2, 3]] == 0).all() and (q[good].abs().amax(-1) > 0).all()
    written = (c.caches[0] != 7.0).any(-1).any(-1).flatten().nonzero().flatten().tolist()
    assert written == sorted(c.slots[[0, 4, 7]].tolist())
    saved = c.pos.clone()
    c.pos = c.pos.clamp(0, 299)
    wq = c.want()[0]
    close(q[good], wq[good], BF16)
    c.pos = saved


def test_nan_and_infinity_stay_in_their_head(device):
    c = Case(6, 4, 2, 128, [16, 24, 24], proj=FP32, seed=7, device=device)
    want = c.run().clone()
    c.q[2, 130] = float("nan")
    c.q[4, 3 * 128 + 5] = float("inf")
    got = c.run()
    touched = torch.zeros((6, 4), dtype=torch.bool)
    touched[2, 1] = touched[4, 3] = True
    assert torch.isnan(got[2, 1]).all() and not torch.isfinite(got[4, 3]).all()
    assert torch.equal(got[~touched.to(device)], want[~touched.to(device)])


def test_unaligned_projections_take_the_other_form(device):
    c = Case(7, 4, 2, 128, [16, 24, 24], seed=8, device=device)
    want = c.run()
    k, v = [t.clone() for t in c.rows()]
    wide = torch.zeros((7, 4 * 128 + 3), device=device)
    wide[:, 1:513] = c.q
    c.q = wide[:, 1:513]
    got = c.run()
    assert ((got.float() - want.float()).abs() <= want.float().abs() * 2.0**-7).all()
    assert ((c.rows()[0].float() - k.float()).abs() <= k.float().abs() * 2.0**-7).all()
    assert torch.equal(c.rows()[1], v)


def test_no_tokens(device):
    c = Case(4, 4, 2, 64, [12, 10, 10], device=device)
    none = lambda t: t[:0].contiguous()  # noqa: E731
    q = c.run(q_proj=none(c.q), k_proj=none(c.k), v_proj=none(c.v), positions=c.pos[:, :0].contiguous().to(device),
              slot_mapping=none(c.slots).to(device), inv_rms=none(c.inv).to(device))
    assert q.shape == (0, 4, 64)
