"""Decode over 4-bit caches (``paged_attention.paged_attention_decode`` with packed pages) on the GPU,
against plain attention in 64 bits over the values that the pages stand for."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from simpler_amd import kv_cache
from simpler_amd import paged_attention as pa
from tests.int4_cases import REL, make_int4_case, rel_l2

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def decode(case, device, out_dtype=FP32, **kw):
    args, opts = case.device_args(device)
    out = pa.paged_attention_decode(*args, out_dtype=out_dtype, **(opts | kw))
    torch.cuda.synchronize(device)
    return out.cpu()


def check(case, device, out_dtype=FP32, errors=False, **kw):
    got = decode(case, device, out_dtype, **kw)
    if not errors:
        pa.check_errors(device)
    assert got.dtype == out_dtype and torch.isfinite(got).all()
    rel = rel_l2(got.double().numpy(), case.reference())
    assert rel <= REL[out_dtype], rel
    return got


FORMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 64), (256, 128)]


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dim,group", FORMS)
def test_forms(dim, group, block, device):
    for dtype, out in ((BF16, BF16), (FP16, FP16), (BF16, FP32), (FP16, FP32)):
        case = make_int4_case([1, 333, 64, 1000], dim=dim, group=group, block=block, dtype=dtype, seed=dim + group + block)
        check(case, device, out)
        check(case, device, out, num_workers=6)  # on the work lists, cut within sequences


@pytest.mark.parametrize("heads,kv_heads,q_len", [(1, 1, 1), (7, 1, 1), (16, 1, 1), (17, 1, 1), (40, 2, 1), (5, 5, 1),
                                                 (32, 8, 8), (8, 2, 2), (64, 1, 3), (6, 3, 16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_per_kv_head(heads, kv_heads, q_len, dim, device):
    """1 to 192 query rows per kv head, causal where there are several tokens."""
    case = make_int4_case([700, 16, 257, 90], heads=heads, kv_heads=kv_heads, q_len=q_len, dim=dim, block=32, seed=heads)
    for out in (BF16, FP32):
        for workers in (0, 8, 64):
            check(case, device, out, num_workers=workers)


@pytest.mark.parametrize("lens", [[0], [1], [15], [16], [17], [63], [64], [65], [127, 128, 129], [0, 0, 5, 0], [4097, 1]])
def test_lengths(lens, device):
    for block in (16, 128):
        case = make_int4_case(lens, block=block, seed=sum(lens))
        for workers in (0, 4, 300):
            got = check(case, device, num_workers=workers)
            for b, n in enumerate(lens):
                assert n or (got[b] == 0).all()


@pytest.mark.parametrize("batch", [3, 200, 300, 700])
@pytest.mark.parametrize("heads", [2, 10, 18])
def test_short_sequences_by_the_thousand(batch, heads, device):
    """Tiles few and many: the workgroups of a short batch shrink from eight waves to one."""
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(0, 300, batch)]
    case = make_int4_case(lens, heads=heads, kv_heads=2, dim=64, group=32, block=32, seed=batch + heads)
    assert pa.kernel_name(pa.make_args(*case.device_args(device)[0], torch.empty_like(case.query, device=device),
                                       case.scale, k_scale=case.k_scale.to(device),
                                       v_scale=case.v_scale.to(device))) == "pa_int4_direct_kernel"
    check(case, device, BF16)
    check(case, device, FP32)


def test_many_sequences_of_mixed_lengths(device):
    rng = np.random.default_rng(3)
    lens = [int(n) for n in rng.integers(0, 90, 600)]
    lens[17] = 5000
    case = make_int4_case(lens, heads=4, kv_heads=1, dim=64, group=32, block=16, seed=9)
    check(case, device, BF16)
    check(case, device, BF16, num_workers=512)


def test_causal_rows_that_see_nothing_are_zero(device):
    """A sequence shorter than its query: the first rows see no token (and the length is reported)."""
    case = make_int4_case([3, 8, 200], q_len=8, block=16, seed=5)
    for workers in (0, 5):
        got = check(case, device, errors=True, num_workers=workers)
        assert (got[0, :5] == 0).all() and (got[0, 5:] != 0).any()
        with pytest.raises(pa.PagedAttentionError) as e:
            pa.check_errors(device)
        assert e.value.rc == -7


@pytest.mark.parametrize("magnitude,scale", [(8.0, None), (0.01, None), (1.0, 0.0), (1.0, -0.3), (1e-3, 4e3)])
def test_magnitudes_and_scales(magnitude, scale, device):
    case = make_int4_case([500, 70], magnitude=magnitude, scale=scale, seed=6)
    for out in (BF16, FP32):
        check(case, device, out)
        check(case, device, out, num_workers=7)


def test_value_scales_of_very_different_size(device):
    """V of 2^-12 to 2^10 along one sequence, large ones last, first and between: the frame follows them."""
    case = make_int4_case([640, 640, 640], dim=64, group=32, block=32, heads=4, kv_heads=1, seed=7)
    size = torch.exp2(torch.linspace(-12, 10, 20))
    order = [torch.arange(20), torch.arange(19, -1, -1), torch.randperm(20, generator=torch.Generator().manual_seed(1))]
    for b in range(3):
        ids = case.block_table[b, :20].long()
        case.v_scale[ids] = (case.v_scale[ids].float() * size[order[b]].view(20, 1, 1, 1, 1)).half()
    for out in (BF16, FP32):
        check(case, device, out)
        check(case, device, out, num_workers=10)


def poison_unseen(case, code=0xFF):
    """NaN scales and other codes in every row that no sequence holds."""
    n, bs = case.key_cache.shape[0], case.key_cache.shape[2]
    held = torch.zeros((n, bs), dtype=torch.bool)
    for b, length in enumerate(case.context_lens.tolist()):
        for p in range(length):
            held[case.block_table[b, p // bs], p % bs] = True
    for s in (case.k_scale, case.v_scale):
        s.masked_fill_(~held[:, None, None, :, None], float("nan"))
    # K rows are apart in a page; V rows share 4-row groups, so only whole groups are overwritten
    case.key_cache[~held[:, None, :].expand(-1, case.key_cache.shape[1], -1)] = code
    groups = held.view(n, bs // 4, 4).any(-1)
    v = case.value_cache.view(n, case.value_cache.shape[1], bs // 4, -1)
    v[~groups[:, None].expand(-1, v.shape[1], -1)] = code


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -65504.0])
def test_rows_past_the_context_do_not_matter(value, device):
    case = make_int4_case([37, 1, 130, 16], block=64, seed=8)
    want = decode(case, device, BF16)
    poison_unseen(case)
    for s in (case.k_scale, case.v_scale):
        s[torch.isnan(s)] = value
    case.block_table[0, 1:], case.block_table[3, 1:] = -5, 1 << 30  # entries past a sequence's blocks
    assert torch.equal(check(case, device, BF16), want)
    check(case, device, BF16, num_workers=3)


def test_nan_scales_reach_only_the_rows_that_see_them(device):
    """Causal rows before a token whose K or V scale is NaN or infinite do not see it; those after are NaN."""
    for name, bad in (("k_scale", float("nan")), ("v_scale", float("nan")), ("v_scale", float("inf")),
                      ("k_scale", float("inf"))):
        case = make_int4_case([70, 90], q_len=4, block=16, heads=4, kv_heads=1, seed=10)
        want = decode(case, device)
        at = 68  # the third query token's own position in sequence 0
        getattr(case, name)[case.block_table[0, at // 16], 0, 1, at % 16] = bad
        got = decode(case, device)
        assert torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1], want[1])
        assert torch.isnan(got[0, 2:]).all()


def test_blocks_outside_the_pool_are_skipped_and_reported(device):
    case = make_int4_case([200, 300, 64], block=32, seed=11)
    case.block_table[0, 0], case.block_table[1, 4], case.block_table[1, 5] = -1, 10**9, case.key_cache.shape[0]
    case.block_table[2, :2] = 77777
    for workers in (0, 9):
        got = check(case, device, errors=True, num_workers=workers)
        assert (got[2] == 0).all()
        with pytest.raises(pa.PagedAttentionError) as e:
            pa.check_errors(device)
        assert e.value.rc == -6


def test_lengths_outside_the_table_are_clamped_and_reported(device):
    case = make_int4_case([64, 64], block=16, extra_width=0, seed=12)
    want = decode(case, device)
    case.context_lens[:] = torch.tensor([1 << 30, -7])
    for workers in (0, 4):
        got = decode(case, device, num_workers=workers)
        torch.testing.assert_close(got[0], want[0], rtol=2e-6, atol=2e-6)  # the same sum, cut elsewhere
        assert (got[1] == 0).all()
        with pytest.raises(pa.PagedAttentionError) as e:
            pa.check_errors(device)
        assert e.value.rc == -7


def test_pages_in_other_layouts(device):
    """K and V pages side by side in a block, and every second block of a larger pool."""
    case = make_int4_case([300, 45, 128], block=32, dim=128, group=32, seed=13)
    want = decode(case, device, BF16)
    n, hkv, bs, row = case.key_cache.shape
    both = torch.full((n, 2, hkv, bs, row), 0xFF, dtype=torch.uint8, device=device)
    both[:, 0], both[:, 1] = case.key_cache.to(device), case.value_cache.to(device)
    wide = torch.full((2 * n, hkv + 1, bs, row), 0xFF, dtype=torch.uint8, device=device)
    wide[::2, :hkv] = case.value_cache.to(device)
    args, opts = case.device_args(device)
    for k, v in ((both[:, 0], both[:, 1]), (both[:, 0], wide[::2, :hkv])):
        got = pa.paged_attention_decode(args[0], k, v, args[3], args[4], out_dtype=BF16, **opts)
        assert torch.equal(got.cpu(), want)


def test_shared_blocks(device):
    """Sequences that share blocks (a prefix), and a block twice in one row."""
    case = make_int4_case([160, 160, 96], block=32, seed=14)
    case.block_table[1, :3] = case.block_table[0, :3]
    case.block_table[2, 1] = case.block_table[2, 0]
    check(case, device, BF16)


def test_same_bits_every_time_and_alone(device):
    case = make_int4_case([2000, 300, 4000], heads=16, kv_heads=4, block=16, seed=15)
    for out in (BF16, FP32):
        first = decode(case, device, out)
        for _ in range(3):
            assert torch.equal(decode(case, device, out), first)


def test_noalloc_entry_gives_the_same_bits(device):
    import ctypes

    from simpler_amd import _lib

    case = make_int4_case([900, 31, 0], heads=24, kv_heads=2, dtype=FP16, seed=16)
    args, opts = case.device_args(device)
    want = decode(case, device, FP16)
    out = torch.full(case.query.shape, float("nan"), dtype=FP16, device=device)
    a = pa.make_args(*args, out, opts["scale"], causal=opts["causal"], k_scale=opts["k_scale"], v_scale=opts["v_scale"])
    rc = _lib.lib().simpler_hip_pa_decode_noalloc(ctypes.byref(a), torch.cuda.current_stream(device).cuda_stream)
    torch.cuda.synchronize(device)
    assert rc == 0 and torch.equal(out.cpu(), want)


def test_main_and_merge_apart(device):
    case = make_int4_case([900, 3000], heads=24, kv_heads=2, seed=17)
    args, opts = case.device_args(device)
    out = torch.empty(case.query.shape, dtype=FP32, device=device)
    a = pa.make_args(*args, out, opts["scale"], k_scale=opts["k_scale"], v_scale=opts["v_scale"], num_workers=96)
    pa.launch(a, device, phases=pa.PHASE_MAIN)
    pa.launch(a, device, phases=pa.PHASE_MERGE)
    assert torch.equal(out.cpu(), decode(case, device, num_workers=96))


def test_two_streams_at_once(device):
    cases = [make_int4_case([3000, 500], heads=16, kv_heads=2, block=64, seed=s) for s in (18, 19)]
    want = [decode(c, device, BF16) for c in cases]
    sent = [c.device_args(device) for c in cases]
    streams = [torch.cuda.Stream(device) for _ in cases]
    torch.cuda.synchronize(device)
    outs = [[], []]
    for _ in range(5):
        for i, (args, opts) in enumerate(sent):
            with torch.cuda.stream(streams[i]):
                outs[i].append(pa.paged_attention_decode(*args, out_dtype=BF16, **opts))
    torch.cuda.synchronize(device)
    for i in range(2):
        assert all(torch.equal(o.cpu(), want[i]) for o in outs[i])


@pytest.mark.parametrize("q_len,dtype", [(1, BF16), (3, FP16)])
def test_append_and_decode_in_one_call(q_len, dtype, device):
    """The new rows where the lengths put them, as ``kv4_append`` writes them, then the decode over them."""
    for lens, block in (([33, 1, 64, 500], 32), ([17, 16, 300, 5], 16)):
        lens = [max(n, q_len) for n in lens]
        case = make_int4_case(lens, q_len=q_len, block=block, dtype=dtype, group=32, seed=20)
        gen = torch.Generator().manual_seed(21)
        shape = (len(lens), q_len, 2, 128) if q_len > 1 else (len(lens), 2, 128)
        k_new, v_new = (torch.randn(shape, generator=gen).to(dtype).to(device) for _ in range(2))
        args, opts = case.device_args(device)
        pos = (torch.tensor(lens)[:, None] - q_len + torch.arange(q_len)).long()
        slots = torch.gather(case.block_table.long(), 1, pos // block) * block + pos % block
        one = {n: t.clone() for n, t in zip(("k", "v", "ks", "vs"), (args[1], args[2], opts["k_scale"], opts["v_scale"]))}
        kv_cache.kv4_append(k_new.view(-1, 2, 128), v_new.view(-1, 2, 128), slots.flatten().to(torch.int32).to(device),
                            one["k"], one["v"], one["ks"], one["vs"])
        want = pa.paged_attention_decode(args[0], one["k"], one["v"], args[3], args[4], out_dtype=dtype, scale=case.scale,
                                         causal=case.causal, k_scale=one["ks"], v_scale=one["vs"])
        got = pa.paged_attention_decode_append(*args, k_new, v_new, out_dtype=dtype, **opts)
        pa.check_errors(device)
        assert torch.equal(got, want)
        for mine, theirs in zip((args[1], args[2], opts["k_scale"], opts["v_scale"]), one.values()):
            assert torch.equal(mine.view(torch.uint8), theirs.view(torch.uint8))


def test_appended_length_outside_the_table(device):
    """Tokens past the row or before its start are dropped; nothing else in the pools changes."""
    case = make_int4_case([30, 32], block=16, extra_width=0, seed=22)
    args, opts = case.device_args(device)
    args[4] = torch.tensor([33, 0], dtype=torch.int32, device=device)
    k = torch.ones((2, 2, 128), dtype=BF16, device=device)
    before = [t.clone() for t in (args[1], args[2], opts["k_scale"], opts["v_scale"])]
    pa.paged_attention_decode_append(*args, k, k, **opts)
    with pytest.raises(pa.PagedAttentionError) as e:
        pa.check_errors(device)
    assert e.value.rc == -7
    for a, b in zip((args[1], args[2], opts["k_scale"], opts["v_scale"]), before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_captured_graph_replays_with_new_inputs(device):
    case = make_int4_case([700, 40], heads=8, kv_heads=2, seed=23)
    other = make_int4_case([333, 120], heads=8, kv_heads=2, seed=24)
    args, opts = case.device_args(device)
    out = torch.empty(case.query.shape, dtype=BF16, device=device)
    stream = torch.cuda.Stream(device)
    with torch.cuda.stream(stream):
        pa.paged_attention_decode(*args, out, **opts)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            pa.paged_attention_decode(*args, out, **opts)
    want = [decode(c, device, BF16) for c in (case, other)]
    for i in (0, 1, 1, 0):
        c = (case, other)[i]
        args[0].copy_(c.query)
        args[4].copy_(c.context_lens)
        if i:  # the other case's lengths over this case's pages
            want[i] = pa.paged_attention_decode(*args, out_dtype=BF16, **opts).cpu()
        out.fill_(float("nan"))
        torch.cuda.synchronize(device)
        graph.replay()
        torch.cuda.synchronize(device)
        assert torch.equal(out.cpu(), want[i])


@pytest.mark.parametrize("scale", [-0.05, 0.0, 1e-6, 1.5])
def test_scales_of_the_scores(scale, device):
    """Negative, none, next to none and one that makes the softmax pick single tokens."""
    case = make_int4_case([5, 300, 64], heads=12, kv_heads=2, q_len=2, scale=scale, seed=77)
    for out in (BF16, FP32):
        for workers in (0, 5):
            check(case, device, out, num_workers=workers)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads", [3, 7, 16, 24, 40])
def test_a_bad_query_row_stays_by_itself(value, heads, device):
    """A row that is not finite shares its tile (and its lanes) with others, whose results do not change."""
    case = make_int4_case([200, 1, 90], heads=heads, kv_heads=1, seed=heads)
    for out in (BF16, FP32):
        for workers in (0, 3):
            want = decode(case, device, out, num_workers=workers)
            kept = case.query.clone()
            case.query[0, 1] = value
            got = decode(case, device, out, num_workers=workers)
            case.query = kept
            assert torch.isnan(got[0, 1]).all()
            got[0, 1] = want[0, 1]
            assert torch.equal(got, want)


def test_one_page_and_one_head_of_any_stride(device):
    """Strides of dims of one element say nothing: any are taken."""
    case = make_int4_case([60], heads=4, kv_heads=1, block=64, extra_width=0, pool_extra=0, seed=3)
    want = check(case, device)
    args, opts = case.device_args(device)
    for i in (1, 2):
        args[i] = args[i].as_strided(args[i].shape, (0, 1, args[i].stride(2), 1))
    out = pa.paged_attention_decode(*args, out_dtype=FP32, **opts)
    assert torch.equal(out.cpu(), want)


def test_lengths_and_rows_of_one_work_list(device):
    """Every number of workers from one to more than there are chunks, over tiles that end inside their slices."""
    case = make_int4_case([129, 0, 1, 640, 64, 300], heads=6, kv_heads=2, dim=64, group=32, block=128, seed=21)
    for workers in range(1, 40):
        check(case, device, FP32, num_workers=workers)


def test_pages_past_four_gigabytes(device):
    """Blocks at the end of a pool whose byte offsets pass 32 bits, as the same blocks of a small pool."""
    blocks, heads, bs, dim, group = 70000, 8, 128, 128, 64  # 4.6 GB of K, as much of V
    large = kv_cache.alloc_kv4_pools(blocks, bs, heads, dim, group, device=device)
    small = kv_cache.alloc_kv4_pools(4, bs, heads, dim, group, device=device)
    gen = torch.Generator(device).manual_seed(1)
    rows = torch.randn((2, 400, heads, dim), generator=gen, device=device, dtype=BF16)
    slots = torch.arange(400, device=device, dtype=torch.int32)
    kv_cache.kv4_append(rows[0], rows[1], slots, *small)
    kv_cache.kv4_append(rows[0], rows[1], slots + (blocks - 4) * bs, *large)
    query = torch.randn((2, 32, dim), generator=gen, device=device, dtype=BF16)
    table = torch.tensor([[0, 1, 2, 3], [3, 2, 1, 0]], dtype=torch.int32, device=device)
    lens = torch.tensor([400, 10], dtype=torch.int32, device=device)
    for workers in (0, 7):
        want, got = (pa.paged_attention_decode(query, p.key_cache, p.value_cache, t, lens, k_scale=p.k_scale,
                                               v_scale=p.v_scale, num_workers=workers)
                     for p, t in ((small, table), (large, table + (blocks - 4))))
        assert torch.equal(got, want)
        pa.check_errors(device)
