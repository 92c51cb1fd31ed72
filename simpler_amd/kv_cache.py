"""KV-cache append and the fused Qwen3 decode prelude on the HIP backend.

The step before paged-attention decode in simpler's Qwen3 decode layer
(``simpler_setup/goldens/qwen3_14b_decode.py``): the current token's K/V are
written into the paged BSND pool at ``slot_mapping`` (``:106-115,261-269``), and
the prelude that produces them and the query — per-head RMS norm with a
weight, half-split RoPE at position ``seq_len − 1``, bf16 rounding
(``:207-226``) — runs fused with that write. Both are kernels in
``libsimpler_hip.so`` (``include/simpler_hip/kv_cache.h``); torch supplies device
memory and the stream only, and there is no fallback.

Around them, also kernels of the library: caches of 4 bits per value
(``alloc_kv4_pools``, ``kv4_append``, ``kv4_gather``; attended to by
``paged_attention.paged_attention_decode``), the prelude with rotary positions
of several axes (``qk_norm_mrope_append``), and a step's block tables and slot
maps built on the device from the requests' lengths (``release_blocks``,
``assign_slots``; ``include/simpler_hip/step_plan.h``).
"""

from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from . import _lib
from .paged_attention import _OUT_DTYPES, PagedAttentionError, _current_device, _current_stream, _raw_stream

EPS = 1e-6  # the golden's eps (qwen3_14b_decode.py:46)

V_SKEW_BYTES = 256  # V pool's distance from K's end, past a multiple of 512 bytes


def alloc_kv_pools(num_blocks: int, block_size: int, kv_heads: int, head_dim: int,
                   dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                   head_dim_v: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V pools, ``[num_blocks, block_size, kv_heads, head_dim(_v)]`` each, in one device allocation.

    V starts ``V_SKEW_BYTES`` past K's end rounded up to 512 bytes, so the two
    pools sit an odd multiple of 256 bytes apart. Pools a multiple of 512
    bytes apart (two separate allocations, or one ``[2, ...]`` tensor) put each
    kv head's K row and V row on the same address bits 8-9; a decode worker
    streams both of its head's rows at once, and those pairs then contend for
    the same HBM channels. Measured on one MI355X, main decode kernel, the
    same inputs in both layouts (bit-identical outputs):

    ========================  ==========  ==========
    config                    apart 0     apart 256
    ========================  ==========  ==========
    Qwen3-8B GQA, B=32        105.8 µs    101.5 µs
    GQA, B=8, L=32768         162.2 µs    158.5 µs
    verify, B=16, q_len=8     129.8 µs    128.0 µs
    ========================  ==========  ==========

    The kernels take any pool addresses; this only places them. Returns the
    two views; the allocation lives as long as either does.
    """
    dv = head_dim if head_dim_v is None else head_dim_v
    esz = torch.empty((), dtype=dtype).element_size()
    k_elems = num_blocks * block_size * kv_heads * head_dim
    v_elems = num_blocks * block_size * kv_heads * dv
    v_start = ((k_elems * esz + 511) // 512 * 512 + V_SKEW_BYTES) // esz
    buf = torch.empty(v_start + v_elems, dtype=dtype, device=device)
    k = buf[:k_elems].view(num_blocks, block_size, kv_heads, head_dim)
    v = buf[v_start:v_start + v_elems].view(num_blocks, block_size, kv_heads, dv)
    return k, v


def _dev(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{name} must be a device (cuda/HIP) tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _cache_strides(cache: torch.Tensor, name: str) -> tuple[int, int, int]:
    if cache.dim() != 4 or cache.stride(-1) != 1:
        raise ValueError(f"{name} must be [num_blocks, block_size, kv_heads, head_dim] with unit head-dim stride")
    return cache.stride()[:3]


def kv_append(key: torch.Tensor, value: torch.Tensor | None, slot_mapping: torch.Tensor, key_cache: torch.Tensor,
              value_cache: torch.Tensor | None, error_count: torch.Tensor | None = None,
              stream: int | None = None) -> None:
    """Write ``key[t]`` (and ``value[t]``), ``[kv_heads, D]`` bf16, at ``slot_mapping[t]`` of the caches.

    ``slot = physical_block · block_size + offset``; negative slots are skipped;
    slots past the pool are skipped and counted in ``error_count`` (an int32
    device tensor of one element) when given. ``value``/``value_cache`` may be
    ``None`` for a K-only (MLA latent) cache.
    """
    a = append_args(key, value, slot_mapping, key_cache, value_cache, error_count)
    launch_append(a, key.device if stream is None else None, stream)


def launch_append(a: _lib.KvAppendArgs, device: torch.device | None = None, stream: int | None = None) -> None:
    """Enqueue a prepared append (``append_args``) on ``stream`` (default: torch's current stream)."""
    if stream is None:
        stream = (_current_stream(device) if device is not None
                  else torch.cuda.current_stream(device).cuda_stream)
    rc = _lib.lib().simpler_hip_kv_append(ctypes.byref(a), stream)
    if rc != 0:
        raise PagedAttentionError(rc, "simpler_hip_kv_append")


# SimplerHipKvAppendArgs as _lib.KvAppendArgs lays it out
_APPEND = struct.Struct("@6P10q6i")
assert _APPEND.size == ctypes.sizeof(_lib.KvAppendArgs)


def _plain_append(key, value, slot_mapping, key_cache, value_cache, error_count) -> _lib.KvAppendArgs | None:
    """``append_args`` where the tensors are as its checks want them, in one pass; None leaves the call to the checks."""
    try:
        bf16 = torch.bfloat16
        tokens, hkv, dk = key.shape
        nblk, bs, chkv, cdk = key_cache.shape
        kt, kh, k1 = key.stride()
        cb, ct, ch, c1 = key_cache.stride()
        if not (key.dtype is bf16 and key_cache.dtype is bf16 and slot_mapping.dtype is torch.int32 and key.is_cuda
                and key_cache.is_cuda and slot_mapping.is_cuda and k1 == 1 and c1 == 1 and chkv == hkv and cdk == dk
                and slot_mapping.shape == (tokens,) and slot_mapping.is_contiguous()):
            return None
        vp = vcp = vt = vh = vb = vct = vch = dv = 0
        if value is not None:
            vn, vhkv, dv = value.shape
            vt, vh, v1 = value.stride()
            vb, vct, vch, vc1 = value_cache.stride()
            if not (value.dtype is bf16 and value_cache.dtype is bf16 and value.is_cuda and value_cache.is_cuda
                    and v1 == 1 and vc1 == 1 and vn == tokens and vhkv == hkv
                    and value_cache.shape == (nblk, bs, hkv, dv)):
                return None
            vp, vcp = value.data_ptr(), value_cache.data_ptr()
        elif value_cache is not None:
            return None
        err = 0
        if error_count is not None:
            if error_count.dtype is not torch.int32 or not error_count.is_cuda:
                return None
            err = error_count.data_ptr()
        return _lib.KvAppendArgs.from_buffer_copy(_APPEND.pack(
            key.data_ptr(), vp, slot_mapping.data_ptr(), key_cache.data_ptr(), vcp, err, kt, kh, vt, vh, cb, ct, ch,
            vb, vct, vch, tokens, hkv, dk, dv, bs, nblk))
    except (AttributeError, TypeError, ValueError, struct.error):
        return None


def append_args(key: torch.Tensor, value: torch.Tensor | None, slot_mapping: torch.Tensor, key_cache: torch.Tensor,
                value_cache: torch.Tensor | None, error_count: torch.Tensor | None = None) -> _lib.KvAppendArgs:
    """Validate the tensors of an append and fill the C ``SimplerHipKvAppendArgs``."""
    a = _plain_append(key, value, slot_mapping, key_cache, value_cache, error_count)
    if a is not None:
        return a
    _dev(key, "key", torch.bfloat16)
    _dev(slot_mapping, "slot_mapping", torch.int32)
    _dev(key_cache, "key_cache", torch.bfloat16)
    if (value is None) != (value_cache is None):
        raise ValueError("value and value_cache go together")
    if key.dim() != 3 or key.stride(-1) != 1:
        raise ValueError("key must be [num_tokens, kv_heads, head_dim] with unit head-dim stride")
    if not slot_mapping.is_contiguous() or slot_mapping.shape != (key.shape[0],):
        raise ValueError("slot_mapping must be a contiguous [num_tokens] tensor")
    a = _lib.KvAppendArgs()
    a.key, a.slot_mapping, a.key_cache = key.data_ptr(), slot_mapping.data_ptr(), key_cache.data_ptr()
    a.key_token_stride, a.key_head_stride = key.stride()[:2]
    a.k_block_stride, a.k_token_stride, a.k_head_stride = _cache_strides(key_cache, "key_cache")
    nblk, bs, hkv, dk = key_cache.shape
    if key.shape[1:] != (hkv, dk):
        raise ValueError(f"key rows {tuple(key.shape[1:])} do not match the cache ({hkv}, {dk})")
    a.num_tokens, a.num_kv_heads, a.head_dim_k, a.block_size, a.num_blocks = key.shape[0], hkv, dk, bs, nblk
    if value is not None:
        _dev(value, "value", torch.bfloat16)
        _dev(value_cache, "value_cache", torch.bfloat16)
        if value.dim() != 3 or value.stride(-1) != 1 or value.shape[:2] != key.shape[:2]:
            raise ValueError("value must be [num_tokens, kv_heads, head_dim_v] with unit head-dim stride")
        a.value, a.value_cache = value.data_ptr(), value_cache.data_ptr()
        a.value_token_stride, a.value_head_stride = value.stride()[:2]
        a.v_block_stride, a.v_token_stride, a.v_head_stride = _cache_strides(value_cache, "value_cache")
        if value_cache.shape[:3] != key_cache.shape[:3] or value_cache.shape[3] != value.shape[2]:
            raise ValueError("value_cache shape does not match key_cache/value")
        a.head_dim_v = value.shape[2]
    if error_count is not None:
        _dev(error_count, "error_count", torch.int32)
        a.error_count = error_count.data_ptr()
    return a


def qk_norm_rope_append(q_proj: torch.Tensor, k_proj: torch.Tensor, v_proj: torch.Tensor, inv_rms: torch.Tensor,
                        q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, rope_cos: torch.Tensor,
                        rope_sin: torch.Tensor, seq_lens: torch.Tensor, slot_mapping: torch.Tensor,
                        key_cache: torch.Tensor, value_cache: torch.Tensor, num_heads: int,
                        q_out: torch.Tensor | None = None, eps: float = EPS,
                        error_count: torch.Tensor | None = None, stream: int | None = None) -> torch.Tensor:
    """The decode prelude fused with the cache write; returns ``q_out`` ``[B, Hq, D]`` bf16.

    ``q_proj [B, Hq·D]``, ``k_proj``/``v_proj [B, Hkv·D]``, ``inv_rms [B]``,
    ``*_norm_weight [D]``, ``rope_cos``/``rope_sin [max_position, D]`` — all fp32
    and contiguous; ``seq_lens``, ``slot_mapping [B]`` int32.
    """
    if q_out is None:
        q_out = torch.empty((q_proj.shape[0], num_heads, key_cache.shape[3]), dtype=torch.bfloat16,
                            device=q_proj.device)
    a = prelude_args(q_proj, k_proj, v_proj, inv_rms, q_norm_weight, k_norm_weight, rope_cos, rope_sin, seq_lens,
                     slot_mapping, key_cache, value_cache, num_heads, q_out, eps, error_count)
    launch_prelude(a, q_proj.device if stream is None else None, stream)
    return q_out


def launch_prelude(a: _lib.QkNormRopeAppendArgs, device: torch.device | None = None,
                   stream: int | None = None) -> None:
    """Enqueue a prepared prelude (``prelude_args``) on ``stream`` (default: torch's current stream)."""
    if stream is None:
        stream = (_current_stream(device) if device is not None
                  else torch.cuda.current_stream(device).cuda_stream)
    rc = _lib.lib().simpler_hip_qk_norm_rope_append(ctypes.byref(a), stream)
    if rc != 0:
        raise PagedAttentionError(rc, "simpler_hip_qk_norm_rope_append")


def prelude_args(q_proj: torch.Tensor, k_proj: torch.Tensor, v_proj: torch.Tensor, inv_rms: torch.Tensor,
                 q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, rope_cos: torch.Tensor,
                 rope_sin: torch.Tensor, seq_lens: torch.Tensor, slot_mapping: torch.Tensor,
                 key_cache: torch.Tensor, value_cache: torch.Tensor, num_heads: int, q_out: torch.Tensor,
                 eps: float = EPS, error_count: torch.Tensor | None = None) -> _lib.QkNormRopeAppendArgs:
    """Validate the tensors of a prelude call and fill the C ``SimplerHipQkNormRopeAppendArgs``."""
    for t, n in ((q_proj, "q_proj"), (k_proj, "k_proj"), (v_proj, "v_proj"), (inv_rms, "inv_rms"),
                 (q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight"), (rope_cos, "rope_cos"),
                 (rope_sin, "rope_sin")):
        _dev(t, n, torch.float32)
        if not t.is_contiguous():
            raise ValueError(f"{n} must be contiguous")
    for t, n in ((seq_lens, "seq_lens"), (slot_mapping, "slot_mapping")):
        _dev(t, n, torch.int32)
        if not t.is_contiguous():
            raise ValueError(f"{n} must be contiguous")
    _dev(key_cache, "key_cache", torch.bfloat16)
    _dev(value_cache, "value_cache", torch.bfloat16)
    nblk, bs, hkv, d = key_cache.shape
    b = q_proj.shape[0]
    if q_proj.shape != (b, num_heads * d) or k_proj.shape != (b, hkv * d) or v_proj.shape != (b, hkv * d):
        raise ValueError("projection shapes do not match num_heads/kv_heads/head_dim of the cache")
    if inv_rms.numel() != b or seq_lens.shape != (b,) or slot_mapping.shape != (b,):
        raise ValueError("inv_rms/seq_lens/slot_mapping must have one entry per sequence")
    if q_norm_weight.numel() != d or k_norm_weight.numel() != d:
        raise ValueError("norm weights must have head_dim entries")
    if rope_cos.dim() != 2 or rope_cos.shape[1] != d or rope_sin.shape != rope_cos.shape:
        raise ValueError("rope tables must be [max_position, head_dim]")
    if value_cache.shape != key_cache.shape:
        raise ValueError("value_cache must match key_cache")
    _dev(q_out, "q_out", torch.bfloat16)
    if not q_out.is_contiguous() or q_out.shape != (b, num_heads, d):
        raise ValueError("q_out must be a contiguous [B, Hq, D] tensor")
    a = _lib.QkNormRopeAppendArgs()
    a.q_proj, a.k_proj, a.v_proj, a.inv_rms = (t.data_ptr() for t in (q_proj, k_proj, v_proj, inv_rms))
    a.q_norm_weight, a.k_norm_weight = q_norm_weight.data_ptr(), k_norm_weight.data_ptr()
    a.rope_cos, a.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    a.seq_lens, a.slot_mapping, a.q_out = seq_lens.data_ptr(), slot_mapping.data_ptr(), q_out.data_ptr()
    a.key_cache, a.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    a.k_block_stride, a.k_token_stride, a.k_head_stride = _cache_strides(key_cache, "key_cache")
    a.v_block_stride, a.v_token_stride, a.v_head_stride = _cache_strides(value_cache, "value_cache")
    a.batch, a.num_heads, a.num_kv_heads, a.head_dim = b, num_heads, hkv, d
    a.block_size, a.num_blocks, a.max_position = bs, nblk, rope_cos.shape[0]
    a.eps = float(eps)
    if error_count is not None:
        _dev(error_count, "error_count", torch.int32)
        a.error_count = error_count.data_ptr()
    return a


def _launch(name: str, packed: bytes, at: int, stream: int | None) -> None:
    """Run the C entry ``name`` on packed args and ``stream`` (default: torch's current one of device ``at``), with
    that device current."""
    fn = getattr(_lib.lib(), name)
    if stream is None:
        stream = _current_stream(torch.device("cuda", at)) if _raw_stream is None else _raw_stream(at)
    if at == _current_device():
        rc = fn(packed, stream)
    else:
        with torch.cuda.device(at):
            rc = fn(packed, stream)
    if rc != 0:
        raise PagedAttentionError(rc, name)


# ---------------------------------------------------------------------------
# Caches of 4 bits per value
# ---------------------------------------------------------------------------


class Kv4Pools(NamedTuple):
    """4-bit K and V pages and their scales, in the order in which ``kv4_append`` and the decode take them."""

    key_cache: torch.Tensor  # uint8 [num_blocks, kv_heads, block_size, head_dim / 2]
    value_cache: torch.Tensor
    k_scale: torch.Tensor  # fp16 [num_blocks, kv_heads, head_dim / group_size, block_size, 2]: scale, zero
    v_scale: torch.Tensor


def alloc_kv4_pools(num_blocks: int, block_size: int, kv_heads: int, head_dim: int, group_size: int = 64,
                    device: torch.device | str = "cuda") -> Kv4Pools:
    """Pools for a cache of 4 bits per value, uninitialised.

    A value is held as a 4-bit code c with a scale s and a zero z, both fp16,
    per token, kv head and group of ``group_size`` dims, and stands for
    ``c * s + z``: ``head_dim / 2 + 4 * head_dim / group_size`` bytes per row.
    The order of the codes within a page is the decode kernel's own
    (``include/simpler_hip/kv_cache.h``): write rows with ``kv4_append``, read them
    with ``kv4_gather``, and move whole pages (``[block]``) as they are.
    head_dim 64, 128 or 256; group_size 32, 64 or 128, at most four groups per
    row; block_size 16, 32, 64 or 128.
    """
    if head_dim not in (64, 128, 256) or group_size not in (32, 64, 128) or not group_size <= head_dim <= 4 * group_size:
        raise ValueError(f"4-bit caches: head_dim 64, 128 or 256 in one, two or four groups of 32, 64 or 128, "
                         f"got {head_dim} and {group_size}")
    if block_size not in (16, 32, 64, 128):
        raise ValueError(f"4-bit caches: block_size 16, 32, 64 or 128, got {block_size}")
    pages = (num_blocks, kv_heads, block_size, head_dim // 2)
    scales = (num_blocks, kv_heads, head_dim // group_size, block_size, 2)
    return Kv4Pools(torch.empty(pages, dtype=torch.uint8, device=device),
                    torch.empty(pages, dtype=torch.uint8, device=device),
                    torch.empty(scales, dtype=torch.float16, device=device),
                    torch.empty(scales, dtype=torch.float16, device=device))


def _one_device(first: torch.Tensor, *others: torch.Tensor) -> bool:
    at = first.get_device()
    for t in others:
        if t.get_device() != at:
            return False
    return True


# SimplerHipKv4Args as _lib.Kv4Args lays it out
_KV4 = struct.Struct("@8P8q8i")
assert _KV4.size == ctypes.sizeof(_lib.Kv4Args)
_HALVES = (torch.bfloat16, torch.float16)
_ROWS = (*_HALVES, torch.float32)


def _kv4_args(key, value, slot_mapping, key_cache, value_cache, k_scale, v_scale, error_count, dtypes) -> bytes:
    """Check the tensors of a 4-bit append or gather (rows of one of ``dtypes``) and pack the C args, in one pass
    over the tensors' attributes (a small append takes the device less time than its checks the host)."""
    rt, shape, pages, scales, at = key.dtype, key.shape, key_cache.shape, k_scale.shape, key.get_device()
    tokens, hkv, dim = shape
    nblk, chkv, bs, row = pages
    groups = scales[2]
    kt, kh, k1 = key.stride()
    vt, vh, v1 = value.stride()
    kb, kch, kcr, kc1 = key_cache.stride()
    vb, vch, vcr, vc1 = value_cache.stride()
    if not (
        rt in dtypes and value.dtype is rt and value.shape == shape and k1 == 1 and v1 == 1
        and key_cache.dtype is torch.uint8 and value_cache.dtype is torch.uint8 and value_cache.shape == pages
        and chkv == hkv and 2 * row == dim and kcr == row and kc1 == 1 and vcr == row and vc1 == 1
        and k_scale.dtype is torch.float16 and v_scale.dtype is torch.float16 and scales == (nblk, hkv, groups, bs, 2)
        and v_scale.shape == scales and k_scale.is_contiguous() and v_scale.is_contiguous()
        and groups > 0 and dim % groups == 0 and slot_mapping.dtype is torch.int32 and slot_mapping.shape == (tokens,)
        and slot_mapping.is_contiguous() and key.is_cuda and value.get_device() == at and slot_mapping.get_device() == at
        and key_cache.get_device() == at and value_cache.get_device() == at and k_scale.get_device() == at
        and v_scale.get_device() == at
        and (error_count is None or (error_count.dtype is torch.int32 and error_count.get_device() == at))
    ):
        _refuse_kv4(key, value, slot_mapping, key_cache, value_cache, k_scale, v_scale, error_count, dtypes)
    if tokens <= 1:  # strides of dims of one element say nothing
        kt = vt = 8
    if hkv == 1:
        kh = vh = 8
        kch = vch = 16
    if nblk == 1:
        kb = vb = 16
    return _KV4.pack(
        key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), 0 if error_count is None else error_count.data_ptr(), kt, kh, vt, vh,
        kb, kch, vb, vch, tokens, hkv, dim, bs, nblk, dim // groups, _OUT_DTYPES[rt], 0)


def _refuse_kv4(key, value, slot_mapping, key_cache, value_cache, k_scale, v_scale, error_count, dtypes) -> None:
    """Say what is wrong with the tensors of a 4-bit append or gather."""
    if key.dtype not in dtypes:
        raise ValueError(f"key must be one of {dtypes}, got {key.dtype}")
    _dev(key, "key", key.dtype)
    _dev(value, "value", key.dtype)
    _dev(slot_mapping, "slot_mapping", torch.int32)
    for t, n in ((key_cache, "key_cache"), (value_cache, "value_cache")):
        _dev(t, n, torch.uint8)
    for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        _dev(t, n, torch.float16)
    if error_count is not None:
        _dev(error_count, "error_count", torch.int32)
    if not _one_device(key, value, slot_mapping, key_cache, value_cache, k_scale, v_scale):
        raise ValueError("the tensors must be on one device")
    raise ValueError(
        "4-bit caches: key and value [num_tokens, kv_heads, head_dim] with unit head-dim stride, slot_mapping "
        "contiguous [num_tokens], pages [num_blocks, kv_heads, block_size, head_dim / 2] contiguous within a block "
        f"and head, scales contiguous [num_blocks, kv_heads, groups, block_size, 2]; got {tuple(key.shape)}, "
        f"{tuple(value.shape)}, {tuple(slot_mapping.shape)}, {tuple(key_cache.shape)}, {tuple(value_cache.shape)}, "
        f"{tuple(k_scale.shape)}, {tuple(v_scale.shape)}")


def kv4_append(key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor, key_cache: torch.Tensor,
               value_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
               error_count: torch.Tensor | None = None, stream: int | None = None) -> None:
    """Quantise ``key[t]`` and ``value[t]``, ``[kv_heads, D]`` bf16 or fp16, to 4 bits at ``slot_mapping[t]``.

    The pools are ``alloc_kv4_pools``'s. Slots as for ``kv_append``: negative ones
    are skipped, those past the pool skipped and counted in ``error_count``; the
    others have to differ. Element error: half a scale (``(max - min) / 30`` of
    its group), and fp16's rounding of the group's bounds; values past fp16's
    range saturate, and a group with a NaN or an infinity reads back as NaN.
    """
    a = _kv4_args(key, value, slot_mapping, key_cache, value_cache, k_scale, v_scale, error_count, _HALVES)
    _launch("simpler_hip_kv4_append", a, key.get_device(), stream)


def kv4_gather(slot_mapping: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, key: torch.Tensor | None = None, value: torch.Tensor | None = None, *,
               dtype: torch.dtype = torch.bfloat16, error_count: torch.Tensor | None = None,
               stream: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``[num_tokens, kv_heads, D]`` of a 4-bit cache at ``slot_mapping``, as bf16, fp16 or fp32 ``(key, value)``.

    Negative slots give zero rows; those past the pool too, counted in
    ``error_count``. For what works on rows: attention of a prompt chunk over a
    cached prefix, moving a sequence to another cache.
    """
    if key is None or value is None:
        rows = torch.empty((2, slot_mapping.shape[0], key_cache.shape[1], 2 * key_cache.shape[3]), dtype=dtype,
                           device=key_cache.device).unbind()
        key, value = (rows[0] if key is None else key), (rows[1] if value is None else value)
    a = _kv4_args(key, value, slot_mapping, key_cache, value_cache, k_scale, v_scale, error_count, _ROWS)
    _launch("simpler_hip_kv4_gather", a, key.get_device(), stream)
    return key, value


# ---------------------------------------------------------------------------
# The prelude with rotary positions of several axes
# ---------------------------------------------------------------------------

# SimplerHipQkNormMropeArgs as _lib.QkNormMropeArgs lays it out
_MROPE = struct.Struct("@14P9q11i4if")
assert _MROPE.size == ctypes.sizeof(_lib.QkNormMropeArgs)


def qk_norm_mrope_append(q_proj: torch.Tensor, k_proj: torch.Tensor, v_proj: torch.Tensor, positions: torch.Tensor,
                         sections: list[int] | tuple[int, ...], rope_cos: torch.Tensor, rope_sin: torch.Tensor,
                         slot_mapping: torch.Tensor | None, key_cache: torch.Tensor, value_cache: torch.Tensor,
                         num_heads: int, q_out: torch.Tensor | None = None, *, interleaved: bool = False,
                         inv_rms: torch.Tensor | None = None, q_norm_weight: torch.Tensor | None = None,
                         k_norm_weight: torch.Tensor | None = None, eps: float = EPS,
                         error_count: torch.Tensor | None = None, stream: int | None = None) -> torch.Tensor:
    """``qk_norm_rope_append`` with positions of several axes (time, height, width); returns ``q_out`` ``[T, Hq, D]``.

    Pair i of a head (dims i and i + D/2) turns by the angle of its axis'
    position, ``rope_cos/sin[positions[axis(i), t], (i, i + D/2)]``:
    ``sections`` counts each axis' pairs, in order, or with ``interleaved`` pair i
    has axis ``a = i % len(sections)`` where ``i < len(sections) * sections[a]``,
    else axis 0. ``q_proj [T, Hq·D]``, ``k_proj``/``v_proj [T, Hkv·D]`` fp32, bf16 or
    fp16 (rows may be parts of a wider projection), ``positions [axes, T]`` int32,
    tables ``[max_position, D]`` fp32. ``inv_rms [T]`` and the norm weights ``[D]``
    (fp32) are optional, each of them. Results are rounded to the caches' dtype,
    bf16 or fp16. With ``slot_mapping=None`` key_cache and value_cache are rows
    ``[T, Hkv, D]`` that are simply filled, as ``kv4_append`` and the decode's append
    take them. Tokens whose position on axis 0 is negative are padding (zero q,
    no rows written); other positions outside the tables count in ``error_count``.
    """
    tokens, dim = q_proj.shape[0], key_cache.shape[-1]
    kst, vst, shape, dtype = key_cache.stride(), value_cache.stride(), key_cache.shape, key_cache.dtype
    if slot_mapping is None and len(shape) == 3:  # rows: one block, whose stride is not used
        nblk, bs, hkv, kst, vst = 1, max(tokens, 1), shape[1], (8, *kst), (8, *vst)
        paged = shape[0] == tokens
    else:
        paged = slot_mapping is not None and len(shape) == 4
        nblk, bs, hkv = shape[:3]
    proj, axes, at = q_proj.dtype, len(sections), q_proj.get_device()
    qs, ks, vs = q_proj.stride(), k_proj.stride(), v_proj.stride()
    i32, f32, rope = torch.int32, torch.float32, rope_cos.shape
    if not (
        paged and dtype in _HALVES and proj in _OUT_DTYPES and value_cache.dtype is dtype and value_cache.shape == shape
        and kst[-1] == 1 and vst[-1] == 1 and 1 <= axes <= 4 and 2 * sum(sections) == dim
        and q_proj.shape == (tokens, num_heads * dim) and k_proj.shape == (tokens, hkv * dim)
        and v_proj.shape == k_proj.shape and k_proj.dtype is proj and v_proj.dtype is proj
        and qs[1] == 1 and ks[1] == 1 and vs[1] == 1 and positions.dtype is i32 and positions.shape == (axes, tokens)
        and positions.is_contiguous() and len(rope) == 2 and rope[1] == dim and rope_sin.shape == rope
        and rope_cos.dtype is f32 and rope_sin.dtype is f32 and rope_cos.is_contiguous() and rope_sin.is_contiguous()
        and (q_out is None or (q_out.dtype is dtype and q_out.shape == (tokens, num_heads, dim)
                               and q_out.is_contiguous() and q_out.get_device() == at))
        and q_proj.is_cuda and k_proj.get_device() == at and v_proj.get_device() == at and positions.get_device() == at
        and rope_cos.get_device() == at and rope_sin.get_device() == at and key_cache.get_device() == at
        and value_cache.get_device() == at
        and (slot_mapping is None or (slot_mapping.dtype is i32 and slot_mapping.shape == (tokens,)
                                      and slot_mapping.is_contiguous() and slot_mapping.get_device() == at))
        and (inv_rms is None or _vector(inv_rms, tokens, at)) and (q_norm_weight is None or _vector(q_norm_weight, dim, at))
        and (k_norm_weight is None or _vector(k_norm_weight, dim, at))
        and (error_count is None or (error_count.dtype is i32 and error_count.get_device() == at))
    ):
        _refuse_mrope(q_proj, k_proj, v_proj, positions, sections, rope_cos, rope_sin, slot_mapping, key_cache,
                      value_cache, num_heads, q_out, inv_rms, q_norm_weight, k_norm_weight, error_count)
    if q_out is None:
        q_out = torch.empty((tokens, num_heads, dim), dtype=dtype, device=q_proj.device)
    one = tokens <= 1  # a stride of one row says nothing
    packed = _MROPE.pack(
        q_proj.data_ptr(), k_proj.data_ptr(), v_proj.data_ptr(), 0 if inv_rms is None else inv_rms.data_ptr(),
        0 if q_norm_weight is None else q_norm_weight.data_ptr(),
        0 if k_norm_weight is None else k_norm_weight.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(),
        positions.data_ptr(), 0 if slot_mapping is None else slot_mapping.data_ptr(), q_out.data_ptr(),
        key_cache.data_ptr(), value_cache.data_ptr(), 0 if error_count is None else error_count.data_ptr(),
        num_heads * dim if one else qs[0], hkv * dim if one else ks[0], hkv * dim if one else vs[0],
        kst[0], kst[1], kst[2], vst[0], vst[1], vst[2], tokens, num_heads, hkv, dim, bs, nblk, rope[0],
        _OUT_DTYPES[proj], _OUT_DTYPES[dtype], axes, 1 if interleaved else 0, *sections, *_NO_SECTIONS[axes:], eps)
    _launch("simpler_hip_qk_norm_mrope_append", packed, at, stream)
    return q_out


_NO_SECTIONS = (0, 0, 0, 0)


def _vector(t: torch.Tensor, n: int, at: int) -> bool:
    return t.dtype is torch.float32 and t.numel() == n and t.is_contiguous() and t.get_device() == at


def _refuse_mrope(q_proj, k_proj, v_proj, positions, sections, rope_cos, rope_sin, slot_mapping, key_cache, value_cache,
                  num_heads, q_out, inv_rms, q_norm_weight, k_norm_weight, error_count) -> None:
    """Say what is wrong with the arguments of ``qk_norm_mrope_append``."""
    tokens, dim, dtype, proj, axes = q_proj.shape[0], key_cache.shape[-1], key_cache.dtype, q_proj.dtype, len(sections)
    if slot_mapping is None and (key_cache.dim() != 3 or key_cache.shape[0] != tokens):
        raise ValueError("without slot_mapping, key_cache and value_cache are rows [num_tokens, kv_heads, head_dim]")
    if slot_mapping is not None and key_cache.dim() != 4:
        raise ValueError("key_cache and value_cache must be [num_blocks, block_size, kv_heads, head_dim]")
    if dtype not in _HALVES or proj not in _OUT_DTYPES:
        raise ValueError(f"caches must be bfloat16 or float16 and projections also or float32, got {dtype}, {proj}")
    if value_cache.shape != key_cache.shape or value_cache.dtype is not dtype or key_cache.stride(-1) != 1 \
            or value_cache.stride(-1) != 1:
        raise ValueError("value_cache must match key_cache, both with unit head-dim stride")
    if not 1 <= axes <= 4 or sum(sections) * 2 != dim:
        raise ValueError(f"sections must be one to four counts that sum to head_dim / 2 = {dim // 2}, got {sections}")
    hkv = key_cache.shape[-2]
    for t, n, w in ((q_proj, "q_proj", num_heads * dim), (k_proj, "k_proj", hkv * dim), (v_proj, "v_proj", hkv * dim)):
        if t.dtype is not proj or t.shape != (tokens, w) or t.stride(1) != 1:
            raise ValueError(f"{n} must be a {proj} [{tokens}, {w}] tensor with unit stride in its rows")
    if rope_cos.dim() != 2 or rope_cos.shape[1] != dim or rope_sin.shape != rope_cos.shape:
        raise ValueError("rope tables must be [max_position, head_dim]")
    for t, n, dt, shape in ((positions, "positions", torch.int32, (axes, tokens)),
                            (slot_mapping, "slot_mapping", torch.int32, (tokens,)),
                            (rope_cos, "rope_cos", torch.float32, rope_cos.shape),
                            (rope_sin, "rope_sin", torch.float32, rope_cos.shape), (inv_rms, "inv_rms", torch.float32, None),
                            (q_norm_weight, "q_norm_weight", torch.float32, (dim,)),
                            (k_norm_weight, "k_norm_weight", torch.float32, (dim,)),
                            (q_out, "q_out", dtype, (tokens, num_heads, dim)),
                            (error_count, "error_count", torch.int32, None)):
        if t is not None and (t.dtype is not dt or not t.is_contiguous() or (shape is not None and t.shape != shape)):
            raise ValueError(f"{n} must be a contiguous {dt} tensor{'' if shape is None else f' {list(shape)}'}")
    if inv_rms is not None and inv_rms.numel() != tokens:
        raise ValueError(f"inv_rms must have {tokens} elements")
    raise ValueError("the tensors must be on one device")


# ---------------------------------------------------------------------------
# Block tables and slot maps of a step
# ---------------------------------------------------------------------------


class ReleasedBlocks(NamedTuple):
    """What ``release_blocks`` returns: the step's lengths and free count."""

    context_lens: torch.Tensor  # [B]
    free_count: torch.Tensor  # [1]


class StepSlots(NamedTuple):
    """What ``assign_slots`` returns, all int32 on the device."""

    slot_mapping: torch.Tensor  # [num_tokens]: -1 where a token has no place
    positions: torch.Tensor  # [num_tokens]
    requests: torch.Tensor  # [num_tokens]
    starts: torch.Tensor  # [B + 1]: request b's tokens are starts[b] .. starts[b + 1]
    context_lens: torch.Tensor  # [B]
    granted: torch.Tensor  # [B]: new_lens, or 0 where refused
    free_count: torch.Tensor  # [1]


# SimplerHipReleaseBlocksArgs and SimplerHipAssignSlotsArgs as _lib lays them out
_RELEASE, _ASSIGN = struct.Struct("@8P4i"), struct.Struct("@13P6i")
assert _RELEASE.size == ctypes.sizeof(_lib.ReleaseBlocksArgs) and _ASSIGN.size == ctypes.sizeof(_lib.AssignSlotsArgs)


def _step_inputs(per_request, name, context_lens, block_table, free_blocks, free_count, error_count) -> tuple[int, ...]:
    """Addresses of a step's input tensors (and of ``error_count``, or 0), checked."""
    batch, width = block_table.shape
    i32, at = torch.int32, block_table.get_device()
    if not (
        block_table.dtype is i32 and block_table.is_cuda and block_table.is_contiguous() and per_request.dtype is i32
        and per_request.shape == (batch,) and per_request.is_contiguous() and per_request.get_device() == at
        and context_lens.dtype is i32 and context_lens.shape == (batch,) and context_lens.is_contiguous()
        and context_lens.get_device() == at and free_blocks.dtype is i32 and free_blocks.dim() == 1
        and free_blocks.is_contiguous() and free_blocks.get_device() == at and free_count.dtype is i32
        and free_count.shape == (1,) and free_count.get_device() == at
        and (error_count is None or (error_count.dtype is i32 and error_count.shape == (1,)
                                     and error_count.get_device() == at))
    ):
        for t, n, shape in ((block_table, "block_table", (batch, width)), (per_request, name, (batch,)),
                            (context_lens, "context_lens", (batch,)), (free_blocks, "free_blocks", free_blocks.shape[:1]),
                            (free_count, "free_count", (1,)), (error_count, "error_count", (1,))):
            if t is not None and (t.dtype is not i32 or not t.is_cuda or t.shape != shape or not t.is_contiguous()):
                raise ValueError(f"{n} must be a contiguous int32 device tensor {list(shape)}, got {t.dtype} "
                                 f"{list(t.shape)} on {t.device}")
        raise ValueError("the tensors must be on one device")
    return (per_request.data_ptr(), context_lens.data_ptr(), block_table.data_ptr(), free_blocks.data_ptr(),
            free_count.data_ptr(), 0 if error_count is None else error_count.data_ptr())


def release_blocks(ended: torch.Tensor, context_lens: torch.Tensor, block_table: torch.Tensor,
                   free_blocks: torch.Tensor, free_count: torch.Tensor, block_size: int,
                   error_count: torch.Tensor | None = None, stream: int | None = None) -> ReleasedBlocks:
    """Return the blocks of the requests with ``ended[b] != 0`` to the free list.

    The free ids are ``free_blocks[:free_count]`` (``free_blocks`` as long as the pool
    has blocks, ``free_count [1]``); the ``ceil(context_lens[b] / block_size)`` ids of each ended
    request's table row are put on top of them, request by request. Returns the
    lengths (0 where ended) and the new count; nothing is read back to the host.
    For requests that own their blocks alone: ids that two rows share would be
    returned twice. Everything int32 and contiguous; at most 4096 requests.
    """
    *inputs, errors = _step_inputs(ended, "ended", context_lens, block_table, free_blocks, free_count, error_count)
    (batch, width), device = block_table.shape, block_table.device
    count_out, lens_out = torch.empty(batch + 1, dtype=torch.int32, device=device).split_with_sizes((1, batch))
    at = count_out.data_ptr()
    _launch("simpler_hip_release_blocks", _RELEASE.pack(*inputs, at + 4, at, errors, batch, width, block_size,
                                                        free_blocks.shape[0]), device.index, stream)
    return ReleasedBlocks(lens_out, count_out)


def assign_slots(new_lens: torch.Tensor, context_lens: torch.Tensor, block_table: torch.Tensor,
                 free_blocks: torch.Tensor, free_count: torch.Tensor, block_size: int, num_tokens: int,
                 error_count: torch.Tensor | None = None, stream: int | None = None) -> StepSlots:
    """Blocks, positions and slots for a step's new tokens, built on the device.

    Request b has ``context_lens[b]`` tokens cached and brings ``new_lens[b]`` (0, 1 or
    a prompt's); the tokens of all requests are packed in request order, up to
    ``num_tokens`` of them. ``block_table`` gets the blocks that are missing, in
    place, from the top of the free list (``free_blocks[free_count - 1]`` first). The slots are
    those that ``kv_append``, ``kv4_append`` and the preludes take (-1: no place), the
    returned lengths those of the decode after the append. A request gets all of
    its tokens or none: it is refused (``granted[b] == 0``, counted in ``error_count``)
    where a length is negative, its tokens do not fit its table row or end past
    ``num_tokens``, or the free list does not cover it and every earlier request.
    Inputs stay as they are (the new lengths and count are outputs), so the same
    call gives the same results again. Everything int32 and contiguous; at most
    4096 requests.
    """
    if num_tokens < 0:
        raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
    *inputs, errors = _step_inputs(new_lens, "new_lens", context_lens, block_table, free_blocks, free_count, error_count)
    (batch, width), device, n = block_table.shape, block_table.device, num_tokens
    buf = torch.empty(3 * n + 3 * batch + 2, dtype=torch.int32, device=device)
    parts = buf.split_with_sizes((n, n, n, batch + 1, batch, batch, 1))
    at, b4, n4 = buf.data_ptr(), 4 * batch, 4 * n
    after = at + 3 * n4
    _launch("simpler_hip_assign_slots", _ASSIGN.pack(
        *inputs, at, at + n4, at + 2 * n4, after, after + b4 + 4, after + 2 * b4 + 4, after + 3 * b4 + 4, errors, batch,
        width, block_size, free_blocks.shape[0], n, 0), device.index, stream)
    return StepSlots(*parts)
