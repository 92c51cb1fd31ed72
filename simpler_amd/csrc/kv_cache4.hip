// The append into 4-bit caches and the read back (include/simpler_hip/
// kv_cache.h has the format), gfx950.
//
// Both are byte movers: 2 D bytes of a 16-bit row against D / 2 + 4 D / G of its
// 4-bit form. A lane holds 8 consecutive dims (one 16-byte load or store of a
// row, one 32-bit word of codes), so D / 8 lanes hold a row and a wave 4 (128
// dims) to 8 rows: consecutive tokens of one kv head, whose codes are then
// consecutive bytes of a page. K's word goes out as it is; V's four bytes are
// traded within the row's lanes for two 16-bit pieces each (dims 32 apart).
//
// The gather is bound by memory, the append by memory and its instructions in
// turn: 16001 tokens of 8 kv heads of 128 dims, bf16, append 26 us (84 MB, 3.2
// TB/s; 18.4 with the quantisation left out), gather 21 (4.0). A grid of 2048
// workgroups that go on to the next rows, their loads ahead, took 28.9 and 25.9,
// 128 or 512 threads the same as 256. Few tokens: 4.5 and 3.0 us, the latency.
//
// Quantisation. Least and greatest value of
// a group come from 16-bit integers of the floats' order, two to a register, by
// DPP moves over its G / 8 lanes. The code is round((x - z) / s):
// (x - z) times the reciprocal of 15 s, kept in 0 .. 1 (the product's clamp), is
// within 2^-22 of its value, 15 times it within 2^-18 of the quotient, so only
// where that falls closer than 2^-16 to a half is the quotient compared with the
// half exactly, in fp64 ((c + 1/2) s has 16 bits). The code is rounded off by a
// sum with 1.5 2^23, and eight of those sums make the word, the constants'
// share taken off at its end.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "simpler_hip/kv_cache.h"
#include "kv_slots.h"
#include "pa_decode_internal.h"

namespace simpler_hip_kv {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int16_t i16x2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads4 = 256;

struct Kv4Params {
    void *key, *value;
    const int32_t *slot;
    uint8_t *kc, *vc;
    uint32_t *ks, *vs;  // (s, z) pairs
    int32_t *err;
    int64_t key_ts, key_hs, val_ts, val_hs;
    int64_t k_bs, k_hs, v_bs, v_hs;
    int32_t tokens, hkv, bs_shift, num_blocks;
    Paged pg;  // append only; block_table null: `slot`
};

// 16-bit floats as 16-bit integers of the same order, and back; NaNs lie beyond
// the infinities.
__device__ __forceinline__ unsigned ordered(const unsigned two) {
    const i16x2_t sign = __builtin_bit_cast(i16x2_t, two) >> 15;
    return two ^ (__builtin_bit_cast(unsigned, sign) & 0x7fff7fffu);
}

__device__ __forceinline__ unsigned min_i16(const unsigned a, const unsigned b) {
    return __builtin_bit_cast(
        unsigned, __builtin_elementwise_min(__builtin_bit_cast(i16x2_t, a), __builtin_bit_cast(i16x2_t, b)));
}

__device__ __forceinline__ unsigned max_i16(const unsigned a, const unsigned b) {
    return __builtin_bit_cast(
        unsigned, __builtin_elementwise_max(__builtin_bit_cast(i16x2_t, a), __builtin_bit_cast(i16x2_t, b)));
}

// Both halves' least over aligned runs of N lanes (4, 8 or 16 lanes of a DPP
// row), in every lane.
template <int N>
__device__ __forceinline__ unsigned min_lanes(unsigned x) {
    static_assert(N == 4 || N == 8 || N == 16, "lanes per group");
    x = min_i16(x, __builtin_amdgcn_mov_dpp(x, 0xB1, 0xf, 0xf, true));                            // quad_perm 1,0,3,2
    x = min_i16(x, __builtin_amdgcn_mov_dpp(x, 0x4E, 0xf, 0xf, true));                            // quad_perm 2,3,0,1
    if constexpr (N >= 8) x = min_i16(x, __builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true));     // row_half_mirror
    if constexpr (N >= 16) x = min_i16(x, __builtin_amdgcn_mov_dpp(x, 0x140, 0xf, 0xf, true));    // row_mirror
    return x;
}

template <bool F16>
__device__ __forceinline__ float elem_to_float(const unsigned bits16) {
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16);
    return __uint_as_float(bits16 << 16);
}

__device__ __forceinline__ float elem(const u32x4_t &raw, const int i, const bool f16) {
    const unsigned b = raw[i / 2] >> (16 * (i & 1));
    return f16 ? elem_to_float<true>(b & 0xffffu) : __uint_as_float(b << 16);
}

// The lane's eight values, their group's (s, z) pair and the codes' word.
template <int LANES, bool F16>
__device__ __forceinline__ void quantise8(const u32x4_t raw, unsigned &word, unsigned &sz) {
#pragma clang fp contract(off)
    // the least in the low half, the complement of the greatest in the high half
    const unsigned a = ordered(raw[0]), b = ordered(raw[1]), c = ordered(raw[2]), d = ordered(raw[3]);
    const unsigned least = min_i16(min_i16(a, b), min_i16(c, d));
    const unsigned most = ~max_i16(max_i16(a, b), max_i16(c, d));
    const unsigned ends = min_lanes<LANES>(min_i16((least & 0xffffu) | most << 16, least >> 16 | (most & 0xffff0000u)));
    const unsigned bounds = ordered(ends ^ 0xffff0000u);
    const float lo = elem_to_float<F16>(bounds & 0xffffu), hi = elem_to_float<F16>(bounds >> 16);
    // an end at an infinity or past it
    const bool odd = min((int)(int16_t)ends, (int)(int16_t)(ends >> 16)) <= ~(F16 ? 0x7c00 : 0x7f80);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = elem(raw, i, F16);
    const _Float16 zh = (_Float16)__builtin_amdgcn_fmed3f(lo, -65504.f, 65504.f);
    // (hi - lo) / 15, correctly rounded: a quotient within an ulp and its exact remainder
    constexpr float kFifteenth = 1.f / 15.f;
    const float range = hi - lo, q0 = range * kFifteenth;
    const _Float16 sh = (_Float16)fminf(__builtin_fmaf(__builtin_fmaf(-15.f, q0, range), kFifteenth, q0), 65504.f);
    const float z = (float)zh, s = (float)sh;
    const float inv = s > 0.f ? __builtin_amdgcn_rcpf(15.f * s) : 0.f;  // s >= 2^-24: a normal fp32 number
    constexpr float kMagic = 12582912.f;  // 1.5 2^23: its sum with a code has the code in its last bits
    unsigned acc = 0;
    float off = 0.f;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float r = __builtin_amdgcn_fmed3f((x[i] - z) * inv, 0.f, 1.f);
        const float t = __builtin_fmaf(r, 15.f, kMagic);
        off = fmaxf(off, fabsf(__builtin_fmaf(r, 15.f, kMagic - t)));
        acc = (acc << 4) + __float_as_uint(t);
    }
    word = acc - 0x4b400000u * 0x11111111u;  // kMagic's bits, 8 times
    sz = (unsigned)__builtin_bit_cast(uint16_t, sh) | (unsigned)__builtin_bit_cast(uint16_t, zh) << 16;
    if (off > 0.5f - 0x1p-16f) {
        word = 0;
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const float v = elem(raw, i, F16), r = __builtin_amdgcn_fmed3f((v - z) * inv, 0.f, 1.f) * 15.f;
            const float below = floorf(r);
            unsigned c = (unsigned)__builtin_rintf(r);
            if (fabsf(r - below - 0.5f) < 0x1p-15f) {
                const double d = (double)v - (double)z, half = ((double)below + 0.5) * (double)s;
                c = (unsigned)below + (d > half || (d == half && ((unsigned)below & 1)) ? 1u : 0u);
            }
            word |= c << (4 * i);
        }
    }
    if (odd) {
        word = 0;
        sz = 0x7e007e00u;
    }
}

// Byte offset in a V page of the 16-bit piece of row t that holds dims 64 h + 32 u + 2 l + v.
template <int D>
__device__ __forceinline__ int v_piece(const int t, const int l, const int h) {
    return ((t >> 2) * 16 + l) * (D / 8) + 4 * (h + (D / 64) * ((t >> 1) & 1)) + 2 * (t & 1);
}

// A thread: dims 8c .. 8c+7 of K and V of a token and kv head. Workgroups of one
// head after the other over the same kRows tokens, so what runs at once reads
// whole token rows.
template <int D>
struct Share {
    static constexpr int kLanes = D / 8, kRows = kThreads4 / kLanes;
    int c, t, h;
    __device__ explicit Share(const int hkv)
        : c(threadIdx.x % kLanes), t((int)(blockIdx.x / (unsigned)hkv) * kRows + (int)threadIdx.x / kLanes),
          h((int)(blockIdx.x % (unsigned)hkv)) {}
};

// A token's cache row: block (-1: none, counted where `count` is set) and offset.
struct Cell {
    int blk, off;
};

__device__ __forceinline__ Cell cell_of(const Kv4Params &P, const int t, const bool count) {
    Cell r{-1, 0};
    if (t >= P.tokens) return r;
    const int mask = (1 << P.bs_shift) - 1;
    if (P.pg.block_table) {
        const int b = t / P.pg.q_len;
        const int64_t p = (int64_t)P.pg.context_lens[b] - P.pg.q_len + (t - b * P.pg.q_len);
        if (p < 0) {
            if (count) atomicOr(P.pg.error_flag, P.pg.bad_length);
        } else if (p < (int64_t)P.pg.max_blocks << P.bs_shift) {
            const int phys = P.pg.block_table[(int64_t)b * P.pg.max_blocks + (p >> P.bs_shift)];
            if ((unsigned)phys < (unsigned)P.num_blocks) r.blk = phys;  // else reported when the decode reads it
            r.off = (int)p & mask;
        }
        return r;
    }
    const int slot = P.slot[t];
    if (slot < 0) return r;
    r.blk = slot >> P.bs_shift;
    r.off = slot & mask;
    if (r.blk >= P.num_blocks) {
        if (count && P.err) atomicAdd(P.err, 1);
        r.blk = -1;
    }
    return r;
}

template <int D, int G, bool F16>
__global__ void __launch_bounds__(kThreads4) kv4_append_kernel(const Kv4Params P) {
    constexpr int NG = D / G;
    const int bs = 1 << P.bs_shift;
    const Share<D> me(P.hkv);
    const int c = me.c, h = me.h;
    const int64_t row = min(me.t, P.tokens - 1);
    const uint16_t *const kr = (const uint16_t *)P.key + row * P.key_ts + h * P.key_hs + 8 * c;
    const uint16_t *const vr = (const uint16_t *)P.value + row * P.val_ts + h * P.val_hs + 8 * c;
    const u32x4_t k_raw = *reinterpret_cast<const u32x4_t *>(kr), v_raw = *reinterpret_cast<const u32x4_t *>(vr);
    const Cell at = cell_of(P, me.t, c == 0 && h == 0);
    unsigned k_word, k_sz, v_word, v_sz;
    quantise8<G / 8, F16>(k_raw, k_word, k_sz);
    quantise8<G / 8, F16>(v_raw, v_word, v_sz);
    // V: lane c's byte i is the nibbles 2u, 2u+1 of piece (4 (c % 4) + i, c / 8),
    // u = (c / 4) % 2; with the lane 4 away it makes the pieces of two l each
    const unsigned other = __shfl_xor(v_word, 4, 64);
    if (at.blk < 0) return;
    const int64_t pair = (((int64_t)at.blk * P.hkv + h) * NG + 8 * c / G) * bs + at.off;
    if (c % (G / 8) == 0) {
        P.ks[pair] = k_sz;
        P.vs[pair] = v_sz;
    }
    uint8_t *const kp = P.kc + at.blk * P.k_bs + h * P.k_hs, *const vp = P.vc + at.blk * P.v_bs + h * P.v_hs;
    // codes and rows through the caches, for what reads them: stored past them the
    // gather alone takes 13.9 us (21.4), but with a kernel that reads its rows 39.6
    // (35.8), and after the append 44 (41); 16001 tokens, 8 heads of 128 dims
    *reinterpret_cast<unsigned *>(kp + at.off * (D / 2) + 4 * ((D / 32) * (c & 3) + (c >> 2))) = k_word;
    const bool high = c & 4;
    const unsigned u0 = high ? other : v_word, u1 = high ? v_word : other;
    // two pieces, of bytes 0 and 1 or 2 and 3 of u0 and u1: u0's byte, then u1's
    const unsigned both = __builtin_amdgcn_perm(u1, u0, high ? 0x07030602u : 0x05010400u);
    uint8_t *const piece = vp + v_piece<D>(at.off, 4 * (c & 3) + (high ? 2 : 0), c >> 3);
    *reinterpret_cast<uint16_t *>(piece) = (uint16_t)both;
    *reinterpret_cast<uint16_t *>(piece + D / 8) = (uint16_t)(both >> 16);  // the next l
}

enum { kRowF32 = 0, kRowBf16 = 1, kRowF16 = 2 };

template <int ROW>
__device__ __forceinline__ void store_row8(void *dst, const int64_t at, const unsigned word, const unsigned sz) {
    const float s = elem_to_float<true>(sz & 0xffffu), z = elem_to_float<true>(sz >> 16);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf((float)((word >> (4 * i)) & 15u), s, z);
    if constexpr (ROW == kRowF32) {
        f32x4_t *const out = reinterpret_cast<f32x4_t *>((float *)dst + at);
        out[0] = (f32x4_t){x[0], x[1], x[2], x[3]};
        out[1] = (f32x4_t){x[4], x[5], x[6], x[7]};
    } else {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (ROW == kRowBf16)
                w[i] = (unsigned)__builtin_bit_cast(uint16_t, (__bf16)x[2 * i]) |
                       (unsigned)__builtin_bit_cast(uint16_t, (__bf16)x[2 * i + 1]) << 16;
            else
                w[i] = (unsigned)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i]) |
                       (unsigned)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]) << 16;
        }
        *reinterpret_cast<u32x4_t *>((uint16_t *)dst + at) = w;
    }
}

template <int D, int G, int ROW>
__global__ void __launch_bounds__(kThreads4) kv4_gather_kernel(const Kv4Params P) {
    constexpr int NG = D / G;
    const int bs = 1 << P.bs_shift;
    const Share<D> me(P.hkv);
    const int c = me.c, t = me.t, h = me.h;
    const Cell at = cell_of(P, t, c == 0 && h == 0);
    unsigned k_word = 0, k_sz = 0, both = 0, v_sz = 0;
    if (at.blk >= 0) {
        const int64_t pair = (((int64_t)at.blk * P.hkv + h) * NG + 8 * c / G) * bs + at.off;
        k_sz = P.ks[pair];
        v_sz = P.vs[pair];
        const uint8_t *const kp = P.kc + at.blk * P.k_bs + h * P.k_hs, *const vp = P.vc + at.blk * P.v_bs + h * P.v_hs;
        k_word = *reinterpret_cast<const unsigned *>(kp + at.off * (D / 2) + 4 * ((D / 32) * (c & 3) + (c >> 2)));
        const uint8_t *const piece = vp + v_piece<D>(at.off, 4 * (c & 3) + (c & 4 ? 2 : 0), c >> 3);
        both = *reinterpret_cast<const uint16_t *>(piece) |
               (unsigned)*reinterpret_cast<const uint16_t *>(piece + D / 8) << 16;
    }
    // V: the append's trade, back: two pieces hold two bytes of this lane's word and two of the lane 4 away
    const unsigned other = __shfl_xor(both, 4, 64);
    if (t >= P.tokens) return;
    const unsigned v_word =
        c & 4 ? __builtin_amdgcn_perm(both, other, 0x07050301u) : __builtin_amdgcn_perm(other, both, 0x06040200u);
    store_row8<ROW>(P.key, t * P.key_ts + h * P.key_hs + 8 * c, k_word, k_sz);
    store_row8<ROW>(P.value, t * P.val_ts + h * P.val_hs + 8 * c, v_word, v_sz);
}

typedef void (*Kv4Fn)(Kv4Params);

template <int D, int G>
Kv4Fn pick_form(const bool gather, const int dtype) {
    if (gather)
        return dtype == SIMPLER_HIP_DT_FLOAT32    ? kv4_gather_kernel<D, G, kRowF32>
               : dtype == SIMPLER_HIP_DT_BFLOAT16 ? kv4_gather_kernel<D, G, kRowBf16>
                                                  : kv4_gather_kernel<D, G, kRowF16>;
    return dtype == SIMPLER_HIP_DT_FLOAT16 ? kv4_append_kernel<D, G, true> : kv4_append_kernel<D, G, false>;
}

// The kernel for a head dim and group, or null.
Kv4Fn pick_kernel(const int d, const int g, const bool gather, const int dtype) {
    switch (d * 1000 + g) {
        case 64032: return pick_form<64, 32>(gather, dtype);
        case 64064: return pick_form<64, 64>(gather, dtype);
        case 128032: return pick_form<128, 32>(gather, dtype);
        case 128064: return pick_form<128, 64>(gather, dtype);
        case 128128: return pick_form<128, 128>(gather, dtype);
        case 256064: return pick_form<256, 64>(gather, dtype);
        case 256128: return pick_form<256, 128>(gather, dtype);
        default: return nullptr;
    }
}

// log2 of a block size that 4-bit pages take, or -1
int block_shift(const int bs) { return bs == 16 ? 4 : bs == 32 ? 5 : bs == 64 ? 6 : bs == 128 ? 7 : -1; }

int launch(Kv4Fn fn, const Kv4Params &P, const int d, hipStream_t stream) {
    const int rows = kThreads4 / (d / 8);
    const int64_t groups = ((int64_t)P.tokens + rows - 1) / rows * P.hkv;
    if (groups * kThreads4 >= (int64_t)1 << 32) return SIMPLER_HIP_ERR_UNSUPPORTED;  // a launch's threads
    hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(kThreads4), 0, stream, P);
    return hipGetLastError() == hipSuccess ? SIMPLER_HIP_OK : SIMPLER_HIP_ERR_LAUNCH;
}

bool misaligned(const void *p, const unsigned a) { return !p || ((uintptr_t)p & (a - 1)); }

int run(const SimplerHipKv4Args *a, const bool gather, void *stream) {
    if (!a || a->num_tokens < 0 || a->num_kv_heads < 1 || a->num_kv_heads > 65535 || a->num_blocks < 1)
        return SIMPLER_HIP_ERR_INVALID;
    if (a->dtype != SIMPLER_HIP_DT_BFLOAT16 && a->dtype != SIMPLER_HIP_DT_FLOAT16 &&
        !(gather && a->dtype == SIMPLER_HIP_DT_FLOAT32))
        return SIMPLER_HIP_ERR_UNSUPPORTED;
    const Kv4Fn fn = pick_kernel(a->head_dim, a->kv_group, gather, a->dtype);
    const int shift = block_shift(a->block_size);
    if (!fn || shift < 0) return SIMPLER_HIP_ERR_UNSUPPORTED;
    if (a->num_tokens == 0) return SIMPLER_HIP_OK;
    if (!a->slot_mapping) return SIMPLER_HIP_ERR_INVALID;
    const void *aligned[4] = {a->key, a->value, a->key_cache, a->value_cache};
    for (const void *p : aligned)
        if (misaligned(p, 16)) return SIMPLER_HIP_ERR_INVALID;
    if (misaligned(a->k_scale, 4) || misaligned(a->v_scale, 4)) return SIMPLER_HIP_ERR_INVALID;
    const int64_t rows[4] = {a->key_token_stride, a->key_head_stride, a->value_token_stride, a->value_head_stride};
    for (int64_t s : rows)
        if (s <= 0 || s % 8) return SIMPLER_HIP_ERR_INVALID;
    const int64_t pages[4] = {a->k_block_stride, a->k_head_stride, a->v_block_stride, a->v_head_stride};
    for (int64_t s : pages)
        if (s <= 0 || s % 16) return SIMPLER_HIP_ERR_INVALID;
    Kv4Params P{};
    P.key = a->key;
    P.value = a->value;
    P.slot = a->slot_mapping;
    P.kc = (uint8_t *)a->key_cache;
    P.vc = (uint8_t *)a->value_cache;
    P.ks = (uint32_t *)a->k_scale;
    P.vs = (uint32_t *)a->v_scale;
    P.err = a->error_count;
    P.key_ts = a->key_token_stride;
    P.key_hs = a->key_head_stride;
    P.val_ts = a->value_token_stride;
    P.val_hs = a->value_head_stride;
    P.k_bs = a->k_block_stride;
    P.k_hs = a->k_head_stride;
    P.v_bs = a->v_block_stride;
    P.v_hs = a->v_head_stride;
    P.tokens = a->num_tokens;
    P.hkv = a->num_kv_heads;
    P.bs_shift = shift;
    P.num_blocks = a->num_blocks;
    return launch(fn, P, a->head_dim, (hipStream_t)stream);
}

}  // namespace
}  // namespace simpler_hip_kv

namespace simpler_hip {

using namespace simpler_hip_kv;

int launch_paged_append4(const SimplerHipPaDecodeArgs *a, const void *key_new, const void *value_new,
                         unsigned *error_flag, unsigned bad_length, void *stream) {
    if ((int64_t)a->batch * a->q_len >= (int64_t)1 << 31 || a->num_kv_heads > 65535) return SIMPLER_HIP_ERR_UNSUPPORTED;
    const int tokens = a->batch * a->q_len, d = a->head_dim_k;
    if (tokens == 0) return SIMPLER_HIP_OK;
    const int dtype =
        a->kv_format == SIMPLER_HIP_KV_INT4_FP16 ? SIMPLER_HIP_DT_FLOAT16 : SIMPLER_HIP_DT_BFLOAT16;
    Kv4Params P{};
    P.key = const_cast<void *>(key_new);
    P.value = const_cast<void *>(value_new);
    P.kc = (uint8_t *)a->key_cache;
    P.vc = (uint8_t *)a->value_cache;
    P.ks = (uint32_t *)a->k_scale;
    P.vs = (uint32_t *)a->v_scale;
    P.key_ts = P.val_ts = (int64_t)a->num_kv_heads * d;
    P.key_hs = P.val_hs = d;
    P.k_bs = a->k_block_stride;
    P.k_hs = a->k_head_stride;
    P.v_bs = a->v_block_stride;
    P.v_hs = a->v_head_stride;
    P.tokens = tokens;
    P.hkv = a->num_kv_heads;
    P.bs_shift = block_shift(a->block_size);
    P.num_blocks = a->num_blocks;
    P.pg = paged_of(a, error_flag, bad_length);
    return launch(pick_kernel(d, a->kv_group, false, dtype), P, d, (hipStream_t)stream);
}

}  // namespace simpler_hip

extern "C" int simpler_hip_kv4_append(const SimplerHipKv4Args *a, void *stream) {
    return simpler_hip_kv::run(a, false, stream);
}

extern "C" int simpler_hip_kv4_gather(const SimplerHipKv4Args *a, void *stream) {
    return simpler_hip_kv::run(a, true, stream);
}
