"""CPU oracle for the 4-bit caches, the step's tables and the several-axis prelude — TEST INFRASTRUCTURE ONLY.

Nothing in the product path (``simpler_amd``) may import this module. Plain
numpy in 64 bits, written from the definitions in ``include/simpler_hip/
kv_cache.h`` and ``step_plan.h``; the reference has no counterpart of them but for
the prelude (``simpler_setup/goldens/qwen3_14b_decode.py:99-103,207-226``), whose
one-axis case ``oracle/kv_oracle.py`` states.

Pinning: ``tests/test_kv4_oracle.py`` (closed forms: a group of evenly spaced
values is reproduced exactly, a constant one too, an element is off by at most
half a step; every nibble of a page holds one element; attention over one token
is its V row; one axis is the plain RoPE; a step's slots against positions
derived one by one).
"""

from __future__ import annotations

import numpy as np

F16_MAX = 65504.0


def quantise(rows: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """fp32 rows ``[..., D]`` (values of a 16-bit type) -> codes (uint8), scale and zero (fp16 values)."""
    x = rows.astype(np.float32).reshape(*rows.shape[:-1], -1, group)
    lo, hi = x.min(-1), x.max(-1)
    bad = ~np.isfinite(x).all(-1)
    with np.errstate(all="ignore"):
        z = np.clip(lo, -F16_MAX, F16_MAX).astype(np.float16)
        s = np.minimum((hi - lo) / np.float32(15), np.float32(F16_MAX)).astype(np.float16)
        z[bad] = s[bad] = np.nan
        s64 = s.astype(np.float64)[..., None]
        q = (x.astype(np.float64) - z.astype(np.float64)[..., None]) / np.where(s64 > 0, s64, 1.0)
    codes = np.where(s64 > 0, np.clip(np.rint(np.nan_to_num(q)), 0, 15), 0)
    return codes.astype(np.uint8).reshape(rows.shape), s, z


def dequantise(codes: np.ndarray, s: np.ndarray, z: np.ndarray) -> np.ndarray:
    """fp64 values of codes ``[..., D]`` with scale and zero ``[..., D / group]``."""
    c = codes.astype(np.float64).reshape(*s.shape, -1)
    return (c * s.astype(np.float64)[..., None] + z.astype(np.float64)[..., None]).reshape(codes.shape)


def nibble_index(block: int, dim: int, value: bool) -> np.ndarray:
    """``[block, dim]``: which nibble of a K or V page holds element (row, dim)."""
    out = np.empty((block, dim), np.int64)
    for t in range(block):
        for d in range(dim):
            if not value:
                j, a, i = d // 32, d % 32 // 8, d % 8
                word = t * dim // 8 + dim // 32 * a + j
            else:
                h, u, lane, v = d // 64, d % 64 // 32, d % 32 // 2, d % 2
                g, b, r = t // 4, t % 4 // 2, t % 2
                word, i = g * dim // 2 + dim // 32 * lane + h + dim // 64 * b, 4 * r + 2 * u + v
            out[t, d] = 8 * word + i
    return out


def pages_to_rows(pages: np.ndarray, scales: np.ndarray, value: bool) -> np.ndarray:
    """Pages ``[n, kv_heads, block, D/2]`` and scales ``[n, kv_heads, groups, block, 2]`` ->
    fp64 rows ``[n, kv_heads, block, D]``."""
    n, hkv, block, row = pages.shape
    flat = pages.reshape(n, hkv, -1)
    nibbles = np.stack([flat & 15, flat >> 4], -1).reshape(n, hkv, -1)
    codes = nibbles[:, :, nibble_index(block, 2 * row, value)]
    return dequantise(codes, scales[..., 0].swapaxes(2, 3), scales[..., 1].swapaxes(2, 3))


def attention(query: np.ndarray, k_rows: np.ndarray, v_rows: np.ndarray, block_table: np.ndarray,
              context_lens: np.ndarray, scale: float, causal: bool = False) -> np.ndarray:
    """fp64 attention of ``query [B, q_len, Hq, D]`` over paged rows ``[n, kv_heads, block, D]``.
    A block outside the pool is skipped; a row that sees nothing is 0."""
    batch, q_len, hq, dim = query.shape
    n, hkv, block, _ = k_rows.shape
    group = hq // hkv
    out = np.zeros(query.shape, np.float64)
    for b in range(batch):
        length = min(max(int(context_lens[b]), 0), block_table.shape[1] * block)
        pos = np.arange(length)
        ids = block_table[b, pos // block]
        inside = (ids >= 0) & (ids < n)
        pos, ids = pos[inside], ids[inside]
        for h in range(hq):
            k, v = k_rows[ids, h // group, pos % block], v_rows[ids, h // group, pos % block]
            for i in range(q_len):
                see = pos < (length - (q_len - 1 - i) if causal else length)
                if see.any():
                    x = k[see] @ query[b, i, h].astype(np.float64) * scale
                    p = np.exp(x - x.max())
                    out[b, i, h] = (p / p.sum()) @ v[see]
    return out


def release_blocks(ended, lens, table, free, count, block):
    """New lengths, free list and count after the ended requests' blocks went back."""
    lens, free = lens.copy(), free.copy()
    width = table.shape[1]
    for b in range(len(lens)):
        if ended[b]:
            n = -(-min(max(int(lens[b]), 0), width * block) // block)
            for j in range(n):
                if count < len(free):
                    free[count] = table[b, j]
                    count += 1
            lens[b] = 0
    return lens, free, count


def assign_slots(new, lens, table, free, count, block, num_tokens):
    """Slots, positions, requests, starts, lengths, granted, count and table of a step, request by request."""
    table, lens = table.copy(), lens.astype(np.int64)
    width = table.shape[1]
    slots, pos, req = (np.full(num_tokens, -1, np.int64) for _ in range(3))
    starts, granted, out_lens = [0], [], []
    asked, left, at = 0, count, 0
    for b in range(len(lens)):
        n, have = int(new[b]), int(lens[b])
        end = at + max(n, 0)
        ok = n >= 0 and have >= 0 and have + n <= min(width * block, 2**31 - 1) and end <= num_tokens
        had = -(-have // block)
        need = -(-(have + n) // block) - had if ok else 0
        if ok and need:
            asked += need
            ok = asked <= count
        if ok:
            for j in range(need):
                table[b, had + j] = free[count - 1 - (asked - need + j)]
            left -= need
            for i in range(n):
                p = have + i
                phys = int(table[b, p // block])
                slots[at + i] = min(phys * block + p % block, 2**31 - 1) if phys >= 0 else -1
                pos[at + i], req[at + i] = p, b
        granted.append(n if ok else 0)
        out_lens.append(have + n if ok else have)
        at = end
        starts.append(min(at, 2**31 - 1))
    return slots, pos, req, np.array(starts), np.array(out_lens), np.array(granted), left, table


def mrope(x: np.ndarray, positions: np.ndarray, sections, cos: np.ndarray, sin: np.ndarray, interleaved: bool,
          inv_rms: np.ndarray | None = None, weight: np.ndarray | None = None, eps: float = 1e-6) -> np.ndarray:
    """fp64 ``[T, heads, D]``: optional RMS norm, then the several-axis turn of each pair."""
    x = x.astype(np.float64)
    half, n = x.shape[-1] // 2, len(sections)
    if inv_rms is not None:
        x = x * inv_rms.astype(np.float64)[:, None, None]
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    out = np.empty_like(x)
    for i in range(half):
        if interleaved:
            a = i % n if i < n * sections[i % n] else 0
        else:
            a = int(np.searchsorted(np.cumsum(sections), i, side="right"))
        p = positions[a]
        lo, hi = x[:, :, i], x[:, :, i + half]
        out[:, :, i] = lo * cos[p, i, None].astype(np.float64) - hi * sin[p, i, None].astype(np.float64)
        out[:, :, i + half] = (hi * cos[p, i + half, None].astype(np.float64)
                               + lo * sin[p, i + half, None].astype(np.float64))
    return out
