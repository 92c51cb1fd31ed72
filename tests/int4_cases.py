"""Cases of the 4-bit cache tests: pools filled from seeded rows, and their fp64 reference."""

from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np
import torch

from oracle import kv4_oracle
from simpler_amd import workloads

# Largest rel-L2 error of a decode over 4-bit caches by its output type. The
# output's own rounding is at most 2^-9 (bf16) and 2^-12 (fp16) in its 2-norm's
# half steps; p s is rounded to 2^-12 of terms that cancel (codes on both sides
# of a group's middle), a few times the result; fp32: exp2 of arguments to about
# 32 at 2^-24 each, and fp32 sums.
REL = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-9, torch.float32: 2.0**-17}


@dataclass
class Int4Case:
    query: torch.Tensor
    key_rows: torch.Tensor  # 16-bit rows [n, kv_heads, block, D] that were quantised
    value_rows: torch.Tensor
    key_cache: torch.Tensor
    value_cache: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    block_table: torch.Tensor
    context_lens: torch.Tensor
    scale: float
    causal: bool

    def device_args(self, device):
        names = ("query", "key_cache", "value_cache", "block_table", "context_lens")
        return [getattr(self, n).to(device) for n in names], {
            "k_scale": self.k_scale.to(device), "v_scale": self.v_scale.to(device), "scale": self.scale,
            "causal": self.causal}

    def reference(self) -> np.ndarray:
        """fp64 output, shaped as the query."""
        k = kv4_oracle.pages_to_rows(self.key_cache.numpy(), self.k_scale.numpy(), False)
        v = kv4_oracle.pages_to_rows(self.value_cache.numpy(), self.v_scale.numpy(), True)
        q = self.query.float().numpy()
        q4 = q if q.ndim == 4 else q[:, None]
        return kv4_oracle.attention(q4, k, v, self.block_table.numpy(), self.context_lens.numpy(), self.scale,
                                    self.causal).reshape(q.shape)


def quantised_pool(rows: torch.Tensor, group: int, value: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Pages and scales of 16-bit rows ``[n, kv_heads, block, D]``."""
    codes, s, z = workloads.quantize_kv4(rows, group)
    return workloads.pack_kv4_pages(codes, value), torch.stack([s, z], -1).transpose(2, 3).contiguous()


def make_int4_case(lens, *, heads=8, kv_heads=2, dim=128, group=64, block=32, q_len=1, causal=None, dtype=torch.bfloat16,
                   seed=0, extra_width=1, pool_extra=1, magnitude=1.0, scale=None) -> Int4Case:
    gen = torch.Generator("cpu").manual_seed(seed)
    per = [(n + block - 1) // block for n in lens]
    pool = sum(per) + pool_extra
    shape = (pool, kv_heads, block, dim)
    level = torch.randn((kv_heads, 1, dim), generator=gen)  # keys have channels of their own level
    k = (torch.randn(shape, generator=gen) + level).mul(magnitude).to(dtype)
    v = torch.randn(shape, generator=gen).to(dtype)
    perm = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.zeros((len(lens), max(per) + extra_width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = perm[at:at + n]
        at += n
    qshape = (len(lens), q_len, heads, dim) if q_len > 1 else (len(lens), heads, dim)
    (kc, ks), (vc, vs) = quantised_pool(k, group, False), quantised_pool(v, group, True)
    return Int4Case(torch.randn(qshape, generator=gen).mul(magnitude).to(dtype), k, v, kc, vc, ks, vs, table,
                    torch.tensor(lens, dtype=torch.int32), 1.0 / math.sqrt(dim) if scale is None else scale,
                    q_len > 1 if causal is None else causal)


def rel_l2(got: np.ndarray, ref: np.ndarray) -> float:
    norm = float(np.linalg.norm(ref))
    off = float(np.linalg.norm(got.astype(np.float64) - ref))
    return off / norm if norm else off
