"""The append into 4-bit caches and the read back, on the GPU: the format's definition, bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv4_oracle
from simpler_amd import kv_cache, workloads

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
FORMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 64), (256, 128)]


def empty_pools(n, bs, hkv, dim, group, device, fill=0xA5):
    pools = kv_cache.alloc_kv4_pools(n, bs, hkv, dim, group, device=device)
    for t in pools:
        t.view(torch.uint8).fill_(fill)
    return pools


def expected_pools(pools, key, value, slots, group):
    """The pools (host copies) after the oracle's append."""
    out = [t.cpu().clone() for t in pools]
    n, hkv, bs, row = out[0].shape
    for which, rows in ((0, key), (1, value)):
        codes, s, z = kv4_oracle.quantise(rows.float().numpy(), group)
        index = kv4_oracle.nibble_index(bs, 2 * row, which == 1)
        flat = out[which].numpy().reshape(n, hkv, -1)
        nib = np.stack([flat & 15, flat >> 4], -1).reshape(n, hkv, -1)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < n * bs:
                nib[slot // bs][:, index[slot % bs]] = codes[t]
                out[2 + which].numpy()[slot // bs, :, :, slot % bs, 0] = s[t]
                out[2 + which].numpy()[slot // bs, :, :, slot % bs, 1] = z[t]
        out[which] = torch.from_numpy((nib[..., ::2] | (nib[..., 1::2] << 4)).reshape(n, hkv, bs, row))
    return out


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def rows(shape, dtype, seed, device):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).mul(3).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim,group", FORMS)
def test_append_writes_the_defined_bits_and_gather_reads_them(dim, group, dtype, device):
    for tokens, hkv, bs, n in ((1, 1, 16, 2), (37, 3, 16, 5), (70, 2, 64, 3), (5, 1, 128, 1)):
        key, value = rows((tokens, hkv, dim), dtype, tokens, device), rows((tokens, hkv, dim), dtype, tokens + 1, device)
        slots = torch.randperm(n * bs, generator=torch.Generator().manual_seed(dim))[:tokens].to(torch.int32)
        if tokens > 4:
            slots[2], slots[4] = -1, -100  # padding
        pools = empty_pools(n, bs, hkv, dim, group, device)
        want = expected_pools(pools, key, value, slots, group)
        kv_cache.kv4_append(key.to(device), value.to(device), slots.to(device), *pools)
        for got, w in zip(pools, want):
            assert same(got, w)
        # the values that they stand for, rounded once; zeros for padding
        for which, r in ((0, key), (1, value)):
            exact = torch.from_numpy(kv4_oracle.dequantise(*kv4_oracle.quantise(r.float().numpy(), group)))
            exact[slots < 0] = 0
            for out in (BF16, FP16, FP32):
                got = kv_cache.kv4_gather(slots.to(device), *pools, dtype=out)[which].cpu()
                # c s is exact in fp32 and one addition rounds; the 16-bit types round that again
                eps = 2.0**-24 if out is FP32 else 2.0**-24 + torch.finfo(out).eps / 2
                tiny = 2.0**-25 if out is FP16 else 0.0
                assert ((got.double() - exact).abs() <= exact.abs() * eps * 1.001 + tiny).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_ties_and_values_next_to_them(dtype, device):
    """Groups whose elements lie on, or one step of their type beside, the halves between two codes."""
    gen = torch.Generator().manual_seed(3)
    step = torch.tensor([0.25, 0.0078125, 3.0, 1.40625, 0.1875, 7.0])
    base = torch.tensor([0.0, -1.5, 100.0, -37.25, 0.3125, -8.0])
    x = torch.zeros((400, 1, 64))
    for t in range(400):
        s, b = step[t % 6], base[(t // 6) % 6]
        halves = torch.randint(0, 31, (64,), generator=gen) / 2
        halves[0], halves[1] = 0, 15
        x[t, 0] = b + s * halves
    x = x.to(dtype)
    bits = x.view(torch.int16)
    nudge = torch.randint(-1, 2, x.shape, generator=gen).to(torch.int16)
    nudge[..., :2] = 0
    x = (bits + torch.where(x != 0, nudge, 0)).view(dtype)
    slots = torch.arange(400, dtype=torch.int32)
    pools = empty_pools(4, 128, 1, 64, 64, device)
    want = expected_pools(pools, x, x, slots, 64)
    kv_cache.kv4_append(x.to(device), x.to(device), slots.to(device), *pools)
    for got, w in zip(pools, want):
        assert same(got, w)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_extreme_values(dtype, device):
    big = float(torch.finfo(dtype).max)
    x = torch.randn((12, 2, 64), generator=torch.Generator().manual_seed(4))
    x[0] = 0
    x[1] = -2.5
    x[2, :, 5] = float("nan")
    x[3, :, 40] = float("inf")
    x[4, 0, :32] = -float("inf")
    x[5, :, 0], x[5, :, 1] = big, -big
    x[6] *= 1e-7
    x[7] *= 1e-4
    x[8] = x[8] * 1e-30 + 5
    x[9] = big
    x[10, :, ::2] = 0
    x[11] *= -0.0
    x = x.to(dtype)
    slots = torch.arange(12, dtype=torch.int32)
    pools = empty_pools(1, 16, 2, 64, 32, device)
    want = expected_pools(pools, x, x, slots, 32)
    kv_cache.kv4_append(x.to(device), x.to(device), slots.to(device), *pools)
    for got, w in zip(pools[:2], want[:2]):
        assert same(got, w)
    for got, w in zip(pools[2:], want[2:]):
        np.testing.assert_array_equal(got.cpu()[:, :, :, :12].float().numpy(), w[:, :, :, :12].float().numpy())
    key, _ = kv_cache.kv4_gather(slots.to(device), *pools, dtype=FP32)
    key = key.cpu()
    assert torch.isnan(key[2, :, :32]).all() and torch.isfinite(key[2, :, 32:]).all()
    assert torch.isnan(key[3, :, 32:]).all() and torch.isnan(key[4, 0, :32]).all() and torch.isfinite(key[4, 1]).all()


def test_slots_past_the_pool_are_counted(device):
    key = rows((6, 2, 128), BF16, 5, device).to(device)
    slots = torch.tensor([0, 32, -1, 31, 1 << 30, 33], dtype=torch.int32)
    pools = empty_pools(2, 16, 2, 128, 64, device)
    want = expected_pools(pools, key.cpu(), key.cpu(), slots, 64)
    errors = torch.zeros(1, dtype=torch.int32, device=device)
    kv_cache.kv4_append(key, key, slots.to(device), *pools, error_count=errors)
    assert errors.item() == 3
    for got, w in zip(pools, want):
        assert same(got, w)
    k, v = kv_cache.kv4_gather(slots.to(device), *pools, error_count=errors)
    assert errors.item() == 6
    for t in (1, 2, 4, 5):
        assert (k[t] == 0).all() and (v[t] == 0).all()
    assert (k[0] != 0).any() and (v[3] != 0).any()


def test_parts_of_wider_tensors_and_pools(device):
    """Rows out of a fused projection, pages out of wider pools; the bytes between stay as they were."""
    qkv = rows((50, 5, 2, 128), BF16, 6, device).to(device)
    key, value = qkv[:, 3], qkv[:, 4]
    both = torch.full((9, 2, 2, 16, 64), 0x5A, dtype=torch.uint8, device=device)
    scales = [torch.zeros((4, 2, 2, 16, 2), dtype=FP16, device=device) for _ in range(2)]
    slots = torch.arange(7, 57, dtype=torch.int32, device=device)
    kc, vc = both[1:9:2, 0], both[1:9:2, 1]
    kv_cache.kv4_append(key, value, slots, kc, vc, *scales)
    plain = empty_pools(4, 16, 2, 128, 64, device, fill=0)
    kv_cache.kv4_append(key.contiguous(), value.contiguous(), slots, *plain)
    got = kv_cache.kv4_gather(slots, kc, vc, *scales)
    want = kv_cache.kv4_gather(slots, *plain)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (both[0::2] == 0x5A).all() and (kc[0, :, :7] == 0x5A).all()
    wide = torch.full((50, 3, 2, 128), 7.0, dtype=FP32, device=device)
    kv_cache.kv4_gather(slots, kc, vc, *scales, key=wide[:, 0], value=wide[:, 2])
    assert (wide[:, 1] == 7).all() and torch.equal(wide[:, 0].bfloat16(), want[0])


def test_large_prompt_and_one_row_of_a_large_pool(device):
    """20,001 tokens over shuffled blocks; then a slot whose page lies past 2^32 bytes."""
    tokens, hkv, dim, bs = 20001, 4, 128, 64
    key = torch.randn((tokens, hkv, dim), generator=torch.Generator("cuda").manual_seed(1), device=device).to(BF16)
    n = (tokens + bs - 1) // bs
    order = torch.randperm(n, generator=torch.Generator("cuda").manual_seed(2), device=device)
    pos = torch.arange(tokens, device=device)
    slots = (order[pos // bs] * bs + pos % bs).to(torch.int32)
    pools = empty_pools(n, bs, hkv, dim, 64, device)
    kv_cache.kv4_append(key, key, slots, *pools)
    got = kv_cache.kv4_gather(slots, *pools, dtype=FP32)
    codes, s, z = workloads.quantize_kv4(key.cpu(), 64)
    want = workloads.dequantize_kv4(codes, s, z)
    for g in got:
        assert ((g.cpu().double() - want).abs() <= want.abs() * 2.0**-23).all()
    del pools, got
    blocks = (1 << 32) // (hkv * bs * dim // 2) + 5
    pools = kv_cache.alloc_kv4_pools(blocks, bs, hkv, dim, 64, device=device)
    far = torch.tensor([blocks * bs - 1, 3], dtype=torch.int32, device=device)
    kv_cache.kv4_append(key[:2], key[1:3], far, *pools)
    got = kv_cache.kv4_gather(far, *pools, dtype=FP32)
    assert ((got[0].cpu().double() - want[:2]).abs() <= want[:2].abs() * 2.0**-23).all()
    assert ((got[1].cpu().double() - want[1:3]).abs() <= want[1:3].abs() * 2.0**-23).all()


def test_nothing_to_do(device):
    pools = empty_pools(2, 16, 2, 128, 64, device)
    none = torch.empty((0, 2, 128), dtype=BF16, device=device)
    kv_cache.kv4_append(none, none, torch.empty(0, dtype=torch.int32, device=device), *pools)
    k, v = kv_cache.kv4_gather(torch.empty(0, dtype=torch.int32, device=device), *pools)
    assert k.shape == v.shape == (0, 2, 128)
