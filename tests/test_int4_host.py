"""4-bit caches, the several-axis prelude and the step's tables: what is refused
before anything is launched, the decode's plan and the packed arguments. No GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from simpler_amd import _lib, kv_cache
from simpler_amd import paged_attention as pa

WS = ctypes.c_void_p(0x100000)


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on the device (nothing here reads it)."""

    is_cuda = True
    device = torch.device("cuda", 0)

    def get_device(self):
        return 0


def dev(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype).as_subclass(OnDevice)


# ---- the decode ----

def decode_args(**kw) -> _lib.PaDecodeArgs:
    base = dict(query=0x1000, key_cache=0x2000, value_cache=0x3000, block_table=0x4000, context_lens=0x5000, out=0x6000,
                k_block_stride=8 * 64 * 64, k_token_stride=64, k_head_stride=64 * 64, v_block_stride=8 * 64 * 64,
                v_token_stride=64, v_head_stride=64 * 64, batch=32, q_len=1, num_heads=32, num_kv_heads=8, head_dim_k=128,
                head_dim_v=128, block_size=64, max_blocks_per_seq=128, num_blocks=1200, out_dtype=6, scale=0.088,
                kv_format=pa.KV_INT4_BF16, k_scale=0x7000, v_scale=0x8000, kv_group=64)
    a = _lib.PaDecodeArgs()
    for k, v in (base | kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("want,kw", [
    (-1, dict(kv_group=0)), (-1, dict(kv_group=48)), (-2, dict(kv_group=16)), (-1, dict(k_scale=0)),
    (-1, dict(v_scale=0)), (-1, dict(k_scale=0x7002)), (-1, dict(k_token_stride=128)), (-1, dict(k_head_stride=8)),
    (-1, dict(v_block_stride=0)), (-1, dict(key_cache=0x2008)), (-1, dict(head_dim_v=64, v_token_stride=32)),
    (-2, dict(block_size=48)), (-2, dict(block_size=256)), (-2, dict(out_dtype=1)),
    (-2, dict(kv_format=pa.KV_INT4_FP16)),  # fp16 query with a bf16 output
    (-2, dict(head_dim_k=96, head_dim_v=96, k_token_stride=48, v_token_stride=48, kv_group=32)),
    (-2, dict(head_dim_k=256, head_dim_v=256, k_token_stride=128, v_token_stride=128, kv_group=32)),  # eight groups
    (-2, dict(head_dim_k=64, head_dim_v=64, k_token_stride=32, v_token_stride=32, kv_group=16)),
    (-1, dict(kv_format=5)), (-1, dict(num_workers=-1)), (-2, dict(max_blocks_per_seq=1 << 25)),
    (-2, dict(max_blocks_per_seq=(1 << 23) - 2)),  # with what each tile's start is charged, past the lists' 32 bits
])
def test_decode_refusals(want, kw):
    lib = _lib.lib()
    assert lib.simpler_hip_pa_decode_workspace_size(ctypes.byref(decode_args())) > 0
    assert lib.simpler_hip_pa_decode(ctypes.byref(decode_args(**kw)), WS, 1 << 30, None) == want
    assert lib.simpler_hip_pa_decode_noalloc(ctypes.byref(decode_args(**kw)), None) == want


@pytest.mark.parametrize("dim,groups", [(64, (32, 64)), (128, (32, 64, 128)), (256, (64, 128))])
def test_decode_plans(dim, groups):
    lib = _lib.lib()
    for group in groups:
        for block in (16, 32, 64, 128):
            for fmt, out in ((pa.KV_INT4_BF16, 6), (pa.KV_INT4_FP16, 1), (pa.KV_INT4_BF16, 0)):
                for heads, q_len in ((8, 1), (32, 1), (32, 8), (128, 8)):
                    a = decode_args(head_dim_k=dim, head_dim_v=dim, k_token_stride=dim // 2, v_token_stride=dim // 2,
                                    kv_group=group, block_size=block, kv_format=fmt, out_dtype=out, num_heads=heads,
                                    q_len=q_len, k_head_stride=block * dim // 2, v_head_stride=block * dim // 2,
                                    max_blocks_per_seq=8192 // block)
                    assert pa.kernel_name(a) == "pa_int4_kernel" and pa.plan(a) > 0
                    need = lib.simpler_hip_pa_decode_workspace_size(ctypes.byref(a))
                    assert 256 < need <= 136 << 20  # the fixed scratch of the no-alloc entry
                    assert lib.simpler_hip_pa_decode(ctypes.byref(a), WS, need - 1, None) == -4
                    a.max_blocks_per_seq = 1
                    assert pa.kernel_name(a) == "pa_int4_direct_kernel"
                    a.num_workers = 5
                    assert pa.kernel_name(a) == "pa_int4_kernel" and pa.plan(a) == 5


def test_short_contexts_take_one_launch():
    """A wave's chunks are at most eight, and at most three more than a list worker's."""
    for batch, tokens, direct in ((32, 4096, True), (32, 4160, False), (8, 2048, True), (8, 2560, False), (128, 1024, True),
                                  (128, 1088, False), (1, 1536, True), (1, 2048, False), (5000, 512, True)):
        name = pa.kernel_name(decode_args(batch=batch, max_blocks_per_seq=tokens // 64))
        assert name == ("pa_int4_direct_kernel" if direct else "pa_int4_kernel"), (batch, tokens)


def test_append_and_prelude_entries():
    lib = _lib.lib()
    k, v = ctypes.c_void_p(0x9000), ctypes.c_void_p(0xA000)
    call = lambda a, kn=k, vn=v, n=1 << 30: lib.simpler_hip_pa_decode_append(ctypes.byref(a), kn, vn, WS, n, None)  # noqa: E731
    assert call(decode_args(), kn=None) == -1
    assert call(decode_args(), vn=None) == -1
    assert call(decode_args(), kn=ctypes.c_void_p(0x9008)) == -1
    assert call(decode_args(q_len=17)) == -2
    assert call(decode_args(), n=16) == -4
    pre = _lib.DecodePreludeArgs(*[0x1000] * 8, 100, 1e-6)
    assert lib.simpler_hip_pa_decode_prelude(ctypes.byref(decode_args()), ctypes.byref(pre), WS, 1 << 30, None) == -2
    assert call(decode_args(batch=0)) == 0


def int4_tensors(b=3, hq=8, hkv=2, d=128, group=64, bs=32, n=5, q_len=1, dtype=torch.bfloat16, out=torch.float32, **kw):
    q = dev(b, hq, d, dtype=dtype) if q_len == 1 else dev(b, q_len, hq, d, dtype=dtype)
    scale = lambda: dev(n, hkv, d // group, bs, 2, dtype=torch.float16)  # noqa: E731
    a = dict(query=q, key_cache=dev(n, hkv, bs, d // 2, dtype=torch.uint8),
             value_cache=dev(n, hkv, bs, d // 2, dtype=torch.uint8), block_table=dev(b, 7, dtype=torch.int32),
             context_lens=dev(b, dtype=torch.int32), out=dev(*q.shape, dtype=out), scale=0.125, k_scale=scale(),
             v_scale=scale())
    return a | kw


def test_make_args_packs_four_bit_pools():
    t = int4_tensors(dtype=torch.float16, q_len=4, causal=True, num_workers=9)
    a = pa.make_args(**t)
    assert (a.batch, a.q_len, a.num_heads, a.num_kv_heads, a.head_dim_k, a.head_dim_v) == (3, 4, 8, 2, 128, 128)
    assert (a.block_size, a.num_blocks, a.max_blocks_per_seq, a.kv_group, a.kv_format) == (32, 5, 7, 64, pa.KV_INT4_FP16)
    assert (a.k_block_stride, a.k_head_stride, a.k_token_stride) == (2 * 32 * 64, 32 * 64, 64)
    assert (a.causal, a.num_workers, a.out_dtype) == (1, 9, 0) and a.k_scale == t["k_scale"].data_ptr()
    both = dev(5, 2, 2, 32, 64, dtype=torch.uint8)  # K and V pages side by side in a block
    a = pa.make_args(**int4_tensors(key_cache=both[:, 0], value_cache=both[:, 1]))
    assert (a.k_block_stride, a.v_head_stride, a.kv_format) == (2 * 2 * 32 * 64, 32 * 64, pa.KV_INT4_BF16)
    assert a.value_cache - a.key_cache == 2 * 32 * 64


def test_make_args_takes_any_stride_of_one_page_and_head():
    t = int4_tensors(hkv=1, n=1)
    for name in ("key_cache", "value_cache"):
        t[name] = t[name].as_strided(t[name].shape, (0, 3, t[name].stride(2), 1))
    a = pa.make_args(**t)
    assert (a.k_block_stride, a.k_head_stride, a.v_block_stride, a.v_head_stride) == (16, 16, 16, 16)


class Elsewhere(OnDevice):
    def get_device(self):
        return 1


def test_make_args_refuses_tensors_of_two_devices():
    t = int4_tensors()
    for name in ("key_cache", "value_cache", "k_scale", "v_scale", "block_table", "context_lens", "out"):
        with pytest.raises(ValueError):
            pa.make_args(**(t | {name: t[name].as_subclass(Elsewhere)}))


@pytest.mark.parametrize("kw", [
    dict(query=dev(3, 8, 128)), dict(key_cache=dev(5, 2, 32, 32, dtype=torch.uint8)),
    dict(value_cache=dev(4, 2, 32, 64, dtype=torch.uint8)), dict(value_cache=dev(5, 2, 32, 64, dtype=torch.int8)),
    dict(key_cache=dev(5, 2, 32, 128, dtype=torch.uint8)[..., ::2]),
    dict(key_cache=dev(5, 32, 2, 64, dtype=torch.uint8).transpose(1, 2)),  # pages of rows that are not together
    dict(v_scale=dev(5, 2, 2, 32, 2)), dict(v_scale=None), dict(k_scale=dev(5, 2, 2, 16, 2, dtype=torch.float16)),
    dict(k_scale=dev(5, 2, 2, 32, 4, dtype=torch.float16)[..., ::2]),
    dict(k_scale=dev(5, 2, 3, 32, 2, dtype=torch.float16), v_scale=dev(5, 2, 3, 32, 2, dtype=torch.float16)),
    dict(out=dev(3, 8, 64)), dict(out=dev(3, 8, 128, dtype=torch.float16)), dict(block_table=dev(2, 7, dtype=torch.int32)),
    dict(context_lens=dev(3, dtype=torch.int64)), dict(query=dev(3, 128, 8, dtype=torch.bfloat16).transpose(1, 2)),
])
def test_make_args_refuses(kw):
    with pytest.raises((ValueError, TypeError, AttributeError)):
        pa.make_args(**int4_tensors(**kw))


def test_make_args_refuses_host_tensors():
    t = int4_tensors()
    for name in ("query", "key_cache", "k_scale", "block_table", "out"):
        with pytest.raises(ValueError):
            pa.make_args(**(t | {name: torch.empty(t[name].shape, dtype=t[name].dtype)}))


# ---- append and gather ----

def kv4_c(**kw) -> _lib.Kv4Args:
    a = _lib.Kv4Args()
    base = dict(key=0x1000, value=0x2000, slot_mapping=0x3000, key_cache=0x4000, value_cache=0x5000, k_scale=0x6000,
                v_scale=0x7000, key_token_stride=1024, key_head_stride=128, value_token_stride=1024,
                value_head_stride=128, k_block_stride=32768, k_head_stride=4096, v_block_stride=32768,
                v_head_stride=4096, num_tokens=3, num_kv_heads=8, head_dim=128, block_size=64, num_blocks=10,
                kv_group=64, dtype=6)
    for k, v in (base | kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("want,kw", [
    (-1, dict(key=0)), (-1, dict(value=0x2008)), (-1, dict(slot_mapping=0)), (-1, dict(k_scale=0x6001)),
    (-1, dict(num_tokens=-1)), (-1, dict(num_kv_heads=0)), (-1, dict(num_blocks=0)), (-1, dict(key_token_stride=1020)),
    (-1, dict(value_head_stride=0)), (-1, dict(k_block_stride=100)), (-2, dict(block_size=24)), (-2, dict(head_dim=96)),
    (-2, dict(kv_group=16)), (-2, dict(head_dim=256, kv_group=32)), (-2, dict(dtype=2)),
])
def test_append_and_gather_refusals(want, kw):
    lib = _lib.lib()
    for entry in (lib.simpler_hip_kv4_append, lib.simpler_hip_kv4_gather):
        assert entry(ctypes.byref(kv4_c(num_tokens=0, key=0)), None) == 0  # nothing to launch
        assert entry(ctypes.byref(kv4_c(**kw)), None) == want
        assert entry(None, None) == -1


def test_append_takes_16_bit_rows_and_gather_fp32_too():
    lib = _lib.lib()
    assert lib.simpler_hip_kv4_append(ctypes.byref(kv4_c(num_tokens=0, dtype=0)), None) == -2
    assert lib.simpler_hip_kv4_gather(ctypes.byref(kv4_c(num_tokens=0, dtype=0)), None) == 0


@pytest.mark.parametrize("args", [(4, 16, 2, 96, 32), (4, 16, 2, 64, 128), (4, 16, 2, 256, 32), (4, 24, 2, 128, 64),
                                  (4, 16, 2, 128, 48)])
def test_alloc_refuses(args):
    with pytest.raises(ValueError):
        kv_cache.alloc_kv4_pools(*args, device="cpu")


def test_alloc_shapes():
    p = kv_cache.alloc_kv4_pools(7, 32, 3, 256, 64, device="cpu")
    assert p.key_cache.shape == p.value_cache.shape == (7, 3, 32, 128) and p.k_scale.shape == (7, 3, 4, 32, 2)


def test_append_refuses_tensors():
    pools = [dev(5, 2, 32, 64, dtype=torch.uint8), dev(5, 2, 32, 64, dtype=torch.uint8),
             dev(5, 2, 2, 32, 2, dtype=torch.float16), dev(5, 2, 2, 32, 2, dtype=torch.float16)]
    k, v, s = (dev(9, 2, 128, dtype=torch.bfloat16), dev(9, 2, 128, dtype=torch.bfloat16), dev(9, dtype=torch.int32))
    for bad in ((dev(9, 2, 128), v, s), (k, dev(9, 2, 64, dtype=torch.bfloat16), s), (k, v, dev(8, dtype=torch.int32)),
                (k, v, dev(9, dtype=torch.int64)), (dev(9, 3, 128, dtype=torch.bfloat16), v, s),
                (dev(9, 2, 256, dtype=torch.bfloat16)[..., ::2], v, s), (torch.empty(9, 2, 128, dtype=torch.bfloat16), v, s)):
        with pytest.raises(ValueError):
            kv_cache.kv4_append(*bad, *pools)
    with pytest.raises(ValueError):
        kv_cache.kv4_append(k, v, s, *pools, error_count=dev(1))
    with pytest.raises(ValueError):
        kv_cache.kv4_gather(s, pools[0], pools[1], pools[2], pools[2].as_subclass(torch.Tensor)[:, :, :1], k, v)


# ---- the several-axis prelude ----

def mrope_c(**kw) -> _lib.QkNormMropeArgs:
    a = _lib.QkNormMropeArgs()
    base = dict(q_proj=0x1000, k_proj=0x2000, v_proj=0x3000, rope_cos=0x4000, rope_sin=0x5000, positions=0x6000,
                q_out=0x7000, key_cache=0x8000, value_cache=0x9000, q_stride=4096, k_stride=1024, v_stride=1024,
                k_block_stride=16384, k_token_stride=1024, k_head_stride=128, v_block_stride=16384, v_token_stride=1024,
                v_head_stride=128, num_tokens=2, num_heads=32, num_kv_heads=8, head_dim=128, block_size=16, num_blocks=4,
                max_position=100, proj_dtype=0, dtype=6, num_axes=3, sections=(16, 24, 24), eps=1e-6)
    for k, v in (base | kw).items():
        setattr(a, k, (ctypes.c_int32 * 4)(*v) if k == "sections" else v)
    return a


@pytest.mark.parametrize("want,kw", [
    (-1, dict(q_proj=0)), (-1, dict(positions=0)), (-1, dict(rope_sin=0)), (-1, dict(q_out=0)), (-1, dict(value_cache=0)),
    (-1, dict(num_tokens=-1)), (-1, dict(num_heads=0)), (-1, dict(head_dim=127)), (-1, dict(head_dim=2048)),
    (-1, dict(num_axes=0)), (-1, dict(num_axes=5)), (-1, dict(sections=(16, 24, 23))), (-1, dict(sections=(70, -3, -3))),
    (-1, dict(num_axes=2, sections=(16, 48, 0, 0), interleaved=1)),  # pairs past the head
    (-1, dict(k_stride=0)), (-1, dict(v_token_stride=-1)), (-1, dict(eps=-1.0)), (-1, dict(max_position=0)),
    (-2, dict(dtype=0)), (-2, dict(proj_dtype=3)),
])
def test_mrope_refusals(want, kw):
    entry = _lib.lib().simpler_hip_qk_norm_mrope_append
    assert entry(ctypes.byref(mrope_c(num_tokens=0, q_proj=0)), None) == 0
    assert entry(ctypes.byref(mrope_c(num_tokens=0, sections=(24, 20, 20), interleaved=1)), None) == 0
    assert entry(ctypes.byref(mrope_c(**kw)), None) == want


def test_mrope_refuses_tensors():
    f, b, i = torch.float32, torch.bfloat16, torch.int32
    good = dict(q_proj=dev(5, 512), k_proj=dev(5, 128), v_proj=dev(5, 128), positions=dev(3, 5, dtype=i),
                sections=(12, 10, 10), rope_cos=dev(99, 64), rope_sin=dev(99, 64), slot_mapping=dev(5, dtype=i),
                key_cache=dev(3, 16, 2, 64, dtype=b), value_cache=dev(3, 16, 2, 64, dtype=b), num_heads=8)
    for bad in (dict(q_proj=dev(5, 448)), dict(k_proj=dev(5, 128, dtype=b)), dict(positions=dev(2, 5, dtype=i)),
                dict(positions=dev(5, 3, dtype=i).t()), dict(sections=(12, 10, 9)), dict(sections=(8, 8, 8, 4, 4)),
                dict(rope_cos=dev(99, 32)), dict(rope_sin=dev(98, 64)), dict(slot_mapping=dev(4, dtype=i)),
                dict(slot_mapping=dev(5, dtype=torch.int64)), dict(slot_mapping=None), dict(key_cache=dev(3, 16, 2, 64, dtype=f)),
                dict(value_cache=dev(3, 16, 1, 64, dtype=b)), dict(inv_rms=dev(4)), dict(q_norm_weight=dev(64, dtype=b)),
                dict(k_norm_weight=dev(32)), dict(q_out=dev(5, 8, 64)), dict(error_count=dev(1)),
                dict(v_proj=torch.empty(5, 128)), dict(q_proj=dev(5, 1024)[:, ::2])):
        with pytest.raises(ValueError):
            kv_cache.qk_norm_mrope_append(**(good | bad))


# ---- the step's tables ----

def step_c(kind, **kw):
    a = _lib.AssignSlotsArgs() if kind == "assign" else _lib.ReleaseBlocksArgs()
    for n, _ in a._fields_:
        setattr(a, n, 0x1000 * (1 + [f for f, _ in a._fields_].index(n)))
    a.error_count = None
    base = dict(batch=4, max_blocks_per_seq=8, block_size=16, capacity=32) | (dict(num_tokens=7) if kind == "assign" else {})
    for k, v in (base | kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kind,want,kw", [
    ("assign", -1, dict(new_lens=0)), ("assign", -1, dict(slot_mapping=0)), ("assign", -1, dict(num_tokens=-1)),
    ("assign", -1, dict(block_size=0)), ("assign", -1, dict(max_blocks_per_seq=0)), ("assign", -1, dict(batch=-1)),
    ("assign", -1, dict(capacity=-1)), ("assign", -2, dict(batch=4097)), ("assign", -1, dict(starts=0)),
    ("assign", -1, dict(context_lens_out=0x2000)),  # an output in the place of an input
    ("release", -1, dict(ended=0)), ("release", -1, dict(free_count_out=0)), ("release", -1, dict(block_size=0)),
    ("release", -2, dict(batch=4097)), ("release", -1, dict(context_lens_out=0x2000)),
])
def test_step_refusals(kind, want, kw):
    lib = _lib.lib()
    entry = lib.simpler_hip_assign_slots if kind == "assign" else lib.simpler_hip_release_blocks
    assert entry(ctypes.byref(step_c(kind, **kw)), None) == want
    assert entry(None, None) == -1


def test_step_refuses_tensors():
    i = torch.int32
    good = dict(new_lens=dev(4, dtype=i), context_lens=dev(4, dtype=i), block_table=dev(4, 6, dtype=i),
                free_blocks=dev(30, dtype=i), free_count=dev(1, dtype=i), block_size=16, num_tokens=9)
    for bad in (dict(new_lens=dev(3, dtype=i)), dict(context_lens=dev(4, dtype=torch.int64)), dict(free_count=dev(2, dtype=i)),
                dict(block_table=dev(4, 12, dtype=i)[:, ::2]), dict(new_lens=torch.empty(4, dtype=i)),
                dict(error_count=dev(1)), dict(num_tokens=-1)):
        with pytest.raises(ValueError):
            kv_cache.assign_slots(**(good | bad))
    good = {k: v for k, v in good.items() if k not in ("new_lens", "num_tokens")} | {"ended": dev(4, dtype=i)}
    for bad in (dict(ended=dev(4, dtype=torch.bool)), dict(free_blocks=dev(30)), dict(context_lens=dev(5, dtype=i))):
        with pytest.raises(ValueError):
            kv_cache.release_blocks(**(good | bad))
