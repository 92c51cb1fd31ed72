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
// Quantisation. Least and greatest value of a group by DPP moves over its G / 8
// lanes. The code is round((x - z) / s): (x - z) times a reciprocal of s is
// within 2^-17 of the quotient, so only where it falls closer than 2^-16 to a
// half is the quotient compared with that half exactly, in fp64 ((c + 1/2) s has
// 16 bits); the division itself would cost more than the rest together.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "simpler_hip/kv_cache.h"
#include "kv_slots.h"
#include "pa_decode_internal.h"

namespace simpler_hip_kv {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

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

// Least, greatest or combined value over aligned runs of N lanes (4, 8 or 16
// lanes of a DPP row), in every lane.
template <int N, typename T, typename F>
__device__ __forceinline__ T combine_lanes(T x, F f) {
    static_assert(N == 4 || N == 8 || N == 16, "lanes per group");
#define SIMPLER_DPP(ctrl) \
    __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xf, 0xf, false))
    x = f(x, SIMPLER_DPP(0xB1));                     // quad_perm 1,0,3,2
    x = f(x, SIMPLER_DPP(0x4E));                     // quad_perm 2,3,0,1
    if constexpr (N >= 8) x = f(x, SIMPLER_DPP(0x141));   // row_half_mirror
    if constexpr (N >= 16) x = f(x, SIMPLER_DPP(0x140));  // row_mirror
#undef SIMPLER_DPP
    return x;
}

template <bool F16>
__device__ __forceinline__ float elem_to_float(const unsigned bits16) {
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16);
    return __uint_as_float(bits16 << 16);
}

// The lane's eight values, their group's (s, z) pair and the codes' word.
template <int LANES, bool F16>
__device__ __forceinline__ void quantise8(const u32x4_t raw, unsigned &word, unsigned &sz) {
#pragma clang fp contract(off)
    float x[8];
    unsigned mag = 0;  // largest magnitude's bits: an exponent of ones is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = elem_to_float<F16>(raw[i] & 0xffffu);
        x[2 * i + 1] = elem_to_float<F16>(raw[i] >> 16);
        mag = max(mag, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
    }
    float lo = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
    float hi = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    lo = combine_lanes<LANES>(lo, [](float a, float b) { return fminf(a, b); });
    hi = combine_lanes<LANES>(hi, [](float a, float b) { return fmaxf(a, b); });
    mag = combine_lanes<LANES>(mag, [](unsigned a, unsigned b) { return max(a, b); });
    const bool finite = mag < (F16 ? 0x7c00u : 0x7f80u);
    const _Float16 zh = (_Float16)fminf(fmaxf(lo, -65504.f), 65504.f);
    const _Float16 sh = (_Float16)fminf(__fdiv_rn(hi - lo, 15.f), 65504.f);
    const float z = (float)zh, s = (float)sh;
    const float inv = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;  // s >= 2^-24: a normal fp32 number
    word = 0;
    bool near = false;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[i] = fminf(fmaxf((x[i] - z) * inv, 0.f), 15.f);
        near |= fabsf(r[i] - floorf(r[i]) - 0.5f) < 0x1p-16f;
        word |= (unsigned)__builtin_rintf(r[i]) << (4 * i);
    }
    if (near && finite) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float below = floorf(r[i]);
            unsigned c = (unsigned)__builtin_rintf(r[i]);
            if (fabsf(r[i] - below - 0.5f) < 0x1p-16f) {
                const double d = (double)x[i] - (double)z, half = ((double)below + 0.5) * (double)s;
                c = (unsigned)below + (d > half || (d == half && ((unsigned)below & 1)) ? 1u : 0u);
            }
            word |= c << (4 * i);
        }
    }
    if (!finite) word = 0;
    sz = finite ? (unsigned)__builtin_bit_cast(uint16_t, sh) | (unsigned)__builtin_bit_cast(uint16_t, zh) << 16
                : 0x7e007e00u;
}

// Byte offset in a V page of the 16-bit piece of row t that holds dims 64 h + 32 u + 2 l + v.
template <int D>
__device__ __forceinline__ int v_piece(const int t, const int l, const int h) {
    return ((t >> 2) * 16 + l) * (D / 8) + 4 * (h + (D / 64) * ((t >> 1) & 1)) + 2 * (t & 1);
}

// grid: x = groups of kRows tokens, y = kv head, z = K or V
template <int D, int G, bool F16>
__global__ void __launch_bounds__(kThreads4) kv4_append_kernel(const Kv4Params P) {
    constexpr int L = D / 8, NG = D / G, kRows = kThreads4 / L;
    const int c = threadIdx.x % L;  // dims 8c .. 8c+7
    const int t = blockIdx.x * kRows + threadIdx.x / L, h = blockIdx.y;
    const bool is_k = blockIdx.z == 0;
    const int bs = 1 << P.bs_shift;
    const bool in = t < P.tokens;
    int blk = -1, off = 0;
    if (in) {
        if (P.pg.block_table) {
            const int b = t / P.pg.q_len;
            const int64_t p = (int64_t)P.pg.context_lens[b] - P.pg.q_len + (t - b * P.pg.q_len);
            if (p < 0) {
                if (c == 0 && h == 0 && is_k) atomicOr(P.pg.error_flag, P.pg.bad_length);
            } else if (p < (int64_t)P.pg.max_blocks << P.bs_shift) {
                const int phys = P.pg.block_table[(int64_t)b * P.pg.max_blocks + (p >> P.bs_shift)];
                if ((unsigned)phys < (unsigned)P.num_blocks) blk = phys;  // else reported when the decode reads it
                off = (int)p & (bs - 1);
            }
        } else {
            const int slot = P.slot[t];
            if (slot >= 0) {
                blk = slot >> P.bs_shift;
                off = slot & (bs - 1);
                if (blk >= P.num_blocks) {
                    if (c == 0 && h == 0 && is_k && P.err) atomicAdd(P.err, 1);
                    blk = -1;
                }
            }
        }
    }
    const uint16_t *src = is_k ? (const uint16_t *)P.key + (in ? t : 0) * P.key_ts + h * P.key_hs
                               : (const uint16_t *)P.value + (in ? t : 0) * P.val_ts + h * P.val_hs;
    unsigned word, sz;
    quantise8<G / 8, F16>(*reinterpret_cast<const u32x4_t *>(src + 8 * c), word, sz);
    // V: lane c's byte i is the nibbles 2u, 2u+1 of piece (4 (c % 4) + i, c / 8),
    // u = (c / 4) % 2; with the lane 4 away it makes the pieces of two l each
    const unsigned other = __shfl_xor(word, 4, 64);
    if (blk < 0) return;
    const int64_t at = (((int64_t)blk * P.hkv + h) * NG + 8 * c / G) * bs + off;
    if (c % (G / 8) == 0) (is_k ? P.ks : P.vs)[at] = sz;
    if (is_k) {
        uint8_t *page = P.kc + blk * P.k_bs + h * P.k_hs;
        *reinterpret_cast<unsigned *>(page + off * (D / 2) + 4 * ((D / 32) * (c & 3) + (c >> 2))) = word;
    } else {
        uint8_t *page = P.vc + blk * P.v_bs + h * P.v_hs;
        const bool high = c & 4;
        const unsigned u0 = high ? other : word, u1 = high ? word : other;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = 2 * (high ? 1 : 0) + k;
            const unsigned piece = ((u0 >> (8 * i)) & 0xffu) | ((u1 >> (8 * i)) & 0xffu) << 8;
            *reinterpret_cast<uint16_t *>(page + v_piece<D>(off, 4 * (c & 3) + i, c >> 3)) = (uint16_t)piece;
        }
    }
}

enum { kRowF32 = 0, kRowBf16 = 1, kRowF16 = 2 };

template <int D, int G, int ROW>
__global__ void __launch_bounds__(kThreads4) kv4_gather_kernel(const Kv4Params P) {
    constexpr int L = D / 8, NG = D / G, kRows = kThreads4 / L;
    const int c = threadIdx.x % L;
    const int t = blockIdx.x * kRows + threadIdx.x / L, h = blockIdx.y;
    const bool is_k = blockIdx.z == 0;
    if (t >= P.tokens) return;
    const int bs = 1 << P.bs_shift;
    const int slot = P.slot[t];
    const int blk = slot >> P.bs_shift, off = slot & (bs - 1);
    const bool there = slot >= 0 && blk < P.num_blocks;
    if (slot >= 0 && !there && c == 0 && h == 0 && is_k && P.err) atomicAdd(P.err, 1);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (there) {
        const unsigned sz = (is_k ? P.ks : P.vs)[(((int64_t)blk * P.hkv + h) * NG + 8 * c / G) * bs + off];
        unsigned word;
        if (is_k) {
            const uint8_t *page = P.kc + blk * P.k_bs + h * P.k_hs;
            word = *reinterpret_cast<const unsigned *>(page + off * (D / 2) + 4 * ((D / 32) * (c & 3) + (c >> 2)));
        } else {
            const uint8_t *page = P.vc + blk * P.v_bs + h * P.v_hs + ((c >> 2) & 1);
            word = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) word |= (unsigned)page[v_piece<D>(off, 4 * (c & 3) + i, c >> 3)] << (8 * i);
        }
        const float s = elem_to_float<true>(sz & 0xffffu), z = elem_to_float<true>(sz >> 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf((float)((word >> (4 * i)) & 15u), s, z);
    }
    const int64_t at = (is_k ? t * P.key_ts + h * P.key_hs : t * P.val_ts + h * P.val_hs) + 8 * c;
    void *dst = is_k ? P.key : P.value;
    if constexpr (ROW == kRowF32) {
        *reinterpret_cast<f32x4_t *>((float *)dst + at) = (f32x4_t){x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4_t *>((float *)dst + at + 4) = (f32x4_t){x[4], x[5], x[6], x[7]};
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
    hipLaunchKernelGGL(fn, dim3((unsigned)((P.tokens + rows - 1) / rows), (unsigned)P.hkv, 2), dim3(kThreads4), 0,
                       stream, P);
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
