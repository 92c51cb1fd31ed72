// The decode prelude with rotary positions of several axes
// (simpler_hip_qk_norm_mrope_append, include/simpler_hip/kv_cache.h), gfx950:
// q/k RMS norm, rotary turn by each pair's own axis, cache write.
//
// A byte mover: every projection value is read once and written once in 16
// bits; the cos/sin rows are shared by a token's heads. A lane holds eight pairs
// (dims 8c .. 8c+7 and those D/2 further: 16-byte loads and stores), so D/16
// lanes hold a head and a wave 8 heads of 128 dims; the turn needs no exchange,
// the norm's sum one over D/16 lanes. A wave works on one token, whose cos/sin
// rows it gathers by axis into LDS once (a lane per pair) while its first heads'
// loads are in flight, and goes through the token's heads with kAhead sets of
// them loaded ahead: all of them where there are tokens enough to fill the
// card, one set where there are few (sets_per_wave). Head dims other than 64,
// 128 and 256 take a wave per head, elements of a half side by side.
//
// Bound by memory, and by its latency and the launch where tokens are few: 9001
// tokens of 32 + 2 x 8 heads of 128 dims, bf16, 50.9 us (4.5 TB/s of 221 MB;
// copies reach 5.2); 32 tokens, fp32 with norms, 4.9 us.
//
// fp32 arithmetic in the golden's order without fused multiply-adds, as in
// kv_cache.hip (simpler_setup/goldens/qwen3_14b_decode.py:99-103,207-226).

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "simpler_hip/kv_cache.h"
#include "pa_decode_internal.h"

namespace simpler_hip_kv {
namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreadsR = 256;
constexpr int kMaxDim = 1024;
enum { kF32 = 0, kBf16 = 1, kF16 = 2 };

struct RotaryParams {
    const void *q, *k, *v;
    const float *inv_rms, *q_w, *k_w, *cos, *sin;
    const int32_t *pos, *slot;
    uint16_t *q_out, *kc, *vc;
    int32_t *err;
    int64_t q_s, k_s, v_s, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs;
    int32_t tokens, hq, hkv, d, bs, num_blocks, max_pos, axes, interleaved;
    int32_t sect[SIMPLER_HIP_MROPE_MAX_AXES];
    int32_t sets, sets_per_wave;  // sets of heads that a wave takes side by side
    int32_t f16;                  // results are fp16, else bf16
    float eps;
};

__device__ __forceinline__ int axis_of(const RotaryParams &P, const int pair) {
    if (P.interleaved) {
        const int a = pair % P.axes;
        int size = P.sect[0];
#pragma unroll
        for (int i = 1; i < SIMPLER_HIP_MROPE_MAX_AXES; ++i) size = a == i ? P.sect[i] : size;
        return pair < P.axes * size ? a : 0;
    }
    int axis = 0, end = 0;
#pragma unroll
    for (int i = 0; i + 1 < SIMPLER_HIP_MROPE_MAX_AXES; ++i) {
        end += P.sect[i];  // sections past the last axis are 0
        if (pair >= end && i + 1 < P.axes) axis = i + 1;
    }
    return axis;
}

__device__ __forceinline__ uint16_t round16(const float x, const bool f16) {
    return f16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : __builtin_bit_cast(uint16_t, (__bf16)x);
}

template <int T>
__device__ __forceinline__ float load1(const void *p, const int64_t i) {
    if constexpr (T == kF32) return ((const float *)p)[i];
    if constexpr (T == kBf16) return __uint_as_float((unsigned)((const uint16_t *)p)[i] << 16);
    return (float)((const _Float16 *)p)[i];
}

// Eight values from two 16-byte pieces (fp32) or one.
template <int T>
__device__ __forceinline__ void unpack8(const u32x4_t *w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (T == kF32) {
            x[i] = __uint_as_float(w[i / 4][i % 4]);
        } else {
            const unsigned b = w[0][i / 2] >> (16 * (i % 2));
            x[i] = T == kBf16 ? __uint_as_float(b << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
        }
    }
}

__device__ __forceinline__ u32x4_t pack8(const float (&x)[8], const bool f16) {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = round16(x[2 * i], f16) | (unsigned)round16(x[2 * i + 1], f16) << 16;
    return w;
}

// A token's place: whether its positions are usable (ok), and its cache rows
// (blk, off) if it has any. Counts a bad position or slot once per token where
// `count` is set.
struct Place {
    bool ok, write;
    int blk, off;
    int p0, p1, p2, p3;  // its positions, 0 where not ok
};
static_assert(SIMPLER_HIP_MROPE_MAX_AXES == 4, "a token's positions");

__device__ __forceinline__ Place place_of(const RotaryParams &P, const int t, const bool count) {
    Place r;
    r.blk = 0;
    r.off = t;
    r.p0 = P.pos[t];
    r.p1 = P.axes > 1 ? P.pos[(int64_t)P.tokens + t] : 0;
    r.p2 = P.axes > 2 ? P.pos[2 * (int64_t)P.tokens + t] : 0;
    r.p3 = P.axes > 3 ? P.pos[3 * (int64_t)P.tokens + t] : 0;
    const bool padding = r.p0 < 0;  // whatever the rest says
    auto outside = [&](const int a, const int p) { return P.sect[a] > 0 && (unsigned)p >= (unsigned)P.max_pos; };
    bool bad = !padding && (outside(0, r.p0) || outside(1, r.p1) || outside(2, r.p2) || outside(3, r.p3));
    r.ok = r.write = !bad && !padding;
    if (!r.ok) r.p0 = r.p1 = r.p2 = r.p3 = 0;
    if (P.slot && !padding) {
        const int slot = P.slot[t];
        r.write = slot >= 0;
        if (r.write) {
            r.blk = slot / P.bs;
            r.off = slot - r.blk * P.bs;
            if (r.blk >= P.num_blocks) {
                r.write = false;
                bad |= r.ok;
            }
        }
    }
    r.write &= r.ok;
    if (bad && count && P.err) atomicAdd(P.err, 1);
    return r;
}

__device__ __forceinline__ int pos_of(const RotaryParams &P, const Place &at, const int pair) {
    const int axis = axis_of(P, pair);
    return axis == 0 ? at.p0 : axis == 1 ? at.p1 : axis == 2 ? at.p2 : at.p3;
}

// D: 64, 128 or 256. A wave: one token, sets_per_wave sets of 1024 / D heads
// (q, then k, then v heads).
template <int D, int T>
__global__ void __launch_bounds__(kThreadsR) mrope_kernel(const RotaryParams P) {
#pragma clang fp contract(off)
    constexpr int L = D / 16, H = 64 / L, half = D / 2;
    constexpr int kPieces = T == kF32 ? 2 : 1;  // 16-byte loads per eight values
    constexpr int kAhead = T == kF32 ? 2 : 3;
    __shared__ __attribute__((aligned(16))) float staged[kThreadsR / 64][4 * D];  // cos, sin, q's and k's weights
    const int lane = threadIdx.x & 63, c = lane % L, sub = lane / L;
    float *const lds = staged[threadIdx.x >> 6];
    const int waves = (P.sets + P.sets_per_wave - 1) / P.sets_per_wave;  // per token
    const unsigned wave = blockIdx.x * (kThreadsR / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = (int)(wave / (unsigned)waves), part = (int)(wave - (unsigned)t * waves);
    if (t >= P.tokens) return;
    const int heads = P.hq + 2 * P.hkv;
    const int set0 = part * P.sets_per_wave, set1 = min(P.sets, set0 + P.sets_per_wave);
    struct Raw {
        u32x4_t lo[kPieces], hi[kPieces];
    };
    auto load = [&](const int set) {
        const int u = min(set * H + sub, heads - 1);
        const bool is_q = u < P.hq, is_k = u < P.hq + P.hkv;
        const int h = is_q ? u : is_k ? u - P.hq : u - P.hq - P.hkv;
        const void *src = is_q ? P.q : is_k ? P.k : P.v;
        const int64_t i = t * (is_q ? P.q_s : is_k ? P.k_s : P.v_s) + (int64_t)h * D + 8 * c;
        const char *const at = (const char *)src + i * (T == kF32 ? 4 : 2);
        Raw r;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            r.lo[k] = *reinterpret_cast<const u32x4_t *>(at + 16 * k);
            r.hi[k] = *reinterpret_cast<const u32x4_t *>(at + half * (T == kF32 ? 4 : 2) + 16 * k);
        }
        return r;
    };
    Raw ahead[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        if (set0 + j < set1) ahead[j] = load(set0 + j);

    const Place at = place_of(P, t, part == 0 && lane == 0);
    const float inv = P.inv_rms ? P.inv_rms[t] : 1.f;
#pragma unroll
    for (int k = 0; k < (half + 63) / 64; ++k) {
        const int pair = lane + 64 * k;
        if (pair < half) {
            const int64_t row = (int64_t)pos_of(P, at, pair) * D + pair;
            lds[pair] = P.cos[row];
            lds[pair + half] = P.cos[row + half];
            lds[D + pair] = P.sin[row];
            lds[D + pair + half] = P.sin[row + half];
        }
    }
    if (P.q_w || P.k_w) {
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            const int i = lane + 64 * k;
            lds[2 * D + i] = P.q_w ? P.q_w[i] : 1.f;
            lds[3 * D + i] = P.k_w ? P.k_w[i] : 1.f;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own LDS writes, in order
    __builtin_amdgcn_wave_barrier();

    for (int base = set0; base < set1; base += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int set = base + j;
            if (set >= set1) break;
            float lo[8], hi[8];
            unpack8<T>(ahead[j].lo, lo);
            unpack8<T>(ahead[j].hi, hi);
            if (set + kAhead < set1) ahead[j] = load(set + kAhead);
            const int u = set * H + sub;
            const bool in = u < heads, is_q = u < P.hq, is_k = !is_q && u < P.hq + P.hkv;
            const int h = is_q ? u : is_k ? u - P.hq : u - P.hq - P.hkv;
            if (P.inv_rms) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    lo[i] *= inv;
                    hi[i] *= inv;
                }
            }
            asm volatile("" ::: "memory");  // the staged values are read per set: kept, they would take half the registers
            const bool norm = is_q ? P.q_w != nullptr : is_k && P.k_w != nullptr;
            if (__any(norm)) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ss += lo[i] * lo[i];
                    ss += hi[i] * hi[i];
                }
#pragma unroll
                for (int d = 1; d < L; d <<= 1) ss += __shfl_xor(ss, d, 64);
                if (norm) {
                    const float r = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)D) + P.eps));
                    const float *const w = lds + (is_q ? 2 * D : 3 * D) + 8 * c;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        lo[i] = (lo[i] * r) * w[i];
                        hi[i] = (hi[i] * r) * w[half + i];
                    }
                }
            }
            if (is_q || is_k) {
                const float *const cs = lds + 8 * c, *const sn = lds + D + 8 * c;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = lo[i] * cs[i] - hi[i] * sn[i];
                    hi[i] = hi[i] * cs[half + i] + lo[i] * sn[half + i];
                    lo[i] = x;
                }
            }
            if (in && (is_q || at.write)) {
                uint16_t *dst = is_q   ? P.q_out + ((int64_t)t * P.hq + h) * D
                                : is_k ? P.kc + at.blk * P.k_bs + at.off * P.k_ts + h * P.k_hs
                                       : P.vc + at.blk * P.v_bs + at.off * P.v_ts + h * P.v_hs;
                // through the caches, for the attention that reads them: past them 47.0 us against
                // 50.9 (the sizes above), but 71.3 against 68.1 with a kernel that reads q after it
                const u32x4_t none = {0, 0, 0, 0};
                *reinterpret_cast<u32x4_t *>(dst + 8 * c) = at.ok ? pack8(lo, P.f16) : none;
                *reinterpret_cast<u32x4_t *>(dst + 8 * c + half) = at.ok ? pack8(hi, P.f16) : none;
            }
        }
    }
}

// Any even head dim to kMaxDim, any alignment of elements: a wave per (token,
// head), lane i takes pairs i, i + 64, ...
template <int T>
__global__ void __launch_bounds__(64) mrope_any_kernel(const RotaryParams P) {
#pragma clang fp contract(off)
    constexpr int kPer = kMaxDim / 2 / 64;
    const int heads = P.hq + 2 * P.hkv;
    const int t = blockIdx.x / heads, u = blockIdx.x - t * heads, lane = threadIdx.x;
    const int half = P.d / 2;
    const bool is_q = u < P.hq, is_k = !is_q && u < P.hq + P.hkv;
    const int h = is_q ? u : is_k ? u - P.hq : u - P.hq - P.hkv;
    const Place at = place_of(P, t, u == 0 && lane == 0);
    if (!is_q && !at.write) return;
    const void *src = is_q ? P.q : is_k ? P.k : P.v;
    const int64_t i0 = t * (is_q ? P.q_s : is_k ? P.k_s : P.v_s) + (int64_t)h * P.d;
    const float *w = is_q ? P.q_w : is_k ? P.k_w : nullptr;
    float lo[kPer], hi[kPer], ss = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = lane + 64 * j;
        lo[j] = hi[j] = 0.f;
        if (i < half) {
            lo[j] = load1<T>(src, i0 + i);
            hi[j] = load1<T>(src, i0 + i + half);
            if (P.inv_rms) {
                lo[j] *= P.inv_rms[t];
                hi[j] *= P.inv_rms[t];
            }
            ss += lo[j] * lo[j];
            ss += hi[j] * hi[j];
        }
    }
    float r = 1.f;
    if (w) {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) ss += __shfl_xor(ss, d, 64);
        r = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(ss, (float)P.d) + P.eps));
    }
    uint16_t *dst = is_q   ? P.q_out + ((int64_t)t * P.hq + h) * P.d
                    : is_k ? P.kc + at.blk * P.k_bs + at.off * P.k_ts + h * P.k_hs
                           : P.vc + at.blk * P.v_bs + at.off * P.v_ts + h * P.v_hs;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = lane + 64 * j;
        if (i >= half) continue;
        float a = lo[j], b = hi[j];
        if (w) {
            a = (a * r) * w[i];
            b = (b * r) * w[i + half];
        }
        if (is_q || is_k) {
            const int p = pos_of(P, at, i);
            const float *cr = P.cos + (int64_t)p * P.d, *sr = P.sin + (int64_t)p * P.d;
            const float x = a * cr[i] - b * sr[i];
            b = b * cr[i + half] + a * sr[i + half];
            a = x;
        }
        dst[i] = at.ok ? round16(a, P.f16) : 0;
        dst[i + half] = at.ok ? round16(b, P.f16) : 0;
    }
}

typedef void (*RotaryFn)(RotaryParams);

template <int T>
RotaryFn pick_rotary(const int d, const bool vec) {
    if (vec && d == 64) return mrope_kernel<64, T>;
    if (vec && d == 128) return mrope_kernel<128, T>;
    if (vec && d == 256) return mrope_kernel<256, T>;
    return mrope_any_kernel<T>;
}

// Sets of heads per wave: all of a token's where that still gives the card's
// 1024 SIMDs kWavesPerSimd waves each, fewer for fewer tokens (48 heads of 128
// dims: 1024 tokens bf16 9.8 us, one set per wave 11.5; 4096 25.3 / 29.0; 2048
// fp32 18.4 / 22.2; to 512 the same).
constexpr int kWavesPerSimd = 2;
int sets_per_wave(const int64_t tokens, const int sets) {
    const int64_t per = tokens * sets / (1024 * kWavesPerSimd);
    return (int)std::min<int64_t>(std::max<int64_t>(per, 1), sets);
}

bool unaligned(const void *p, const unsigned a) { return ((uintptr_t)p & (a - 1)) != 0; }

}  // namespace
}  // namespace simpler_hip_kv

using namespace simpler_hip_kv;

extern "C" int simpler_hip_qk_norm_mrope_append(const SimplerHipQkNormMropeArgs *a, void *stream) {
    if (!a || a->num_tokens < 0 || a->num_heads < 1 || a->num_kv_heads < 1 || a->block_size < 1 || a->num_blocks < 1 ||
        a->max_position < 1)
        return SIMPLER_HIP_ERR_INVALID;
    if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > kMaxDim) return SIMPLER_HIP_ERR_INVALID;
    if (a->num_axes < 1 || a->num_axes > SIMPLER_HIP_MROPE_MAX_AXES) return SIMPLER_HIP_ERR_INVALID;
    const bool f16 = a->dtype == SIMPLER_HIP_DT_FLOAT16;
    if (!f16 && a->dtype != SIMPLER_HIP_DT_BFLOAT16) return SIMPLER_HIP_ERR_UNSUPPORTED;
    if (a->proj_dtype != SIMPLER_HIP_DT_FLOAT32 && a->proj_dtype != SIMPLER_HIP_DT_BFLOAT16 &&
        a->proj_dtype != SIMPLER_HIP_DT_FLOAT16)
        return SIMPLER_HIP_ERR_UNSUPPORTED;
    int64_t pairs = 0;
    for (int i = 0; i < a->num_axes; ++i) {
        if (a->sections[i] < 0) return SIMPLER_HIP_ERR_INVALID;
        pairs += a->sections[i];
        // an axis' last interleaved pair is num_axes (sections - 1) + axis
        if (a->interleaved && i > 0 && a->sections[i] > 0 &&
            (int64_t)a->num_axes * (a->sections[i] - 1) + i >= a->head_dim / 2)
            return SIMPLER_HIP_ERR_INVALID;
    }
    if (pairs != a->head_dim / 2) return SIMPLER_HIP_ERR_INVALID;
    const int64_t strides[9] = {a->q_stride,       a->k_stride,      a->v_stride,       a->k_block_stride, a->k_token_stride,
                                a->k_head_stride,  a->v_block_stride, a->v_token_stride, a->v_head_stride};
    for (int64_t s : strides)
        if (s <= 0) return SIMPLER_HIP_ERR_INVALID;
    if (!(a->eps >= 0.f)) return SIMPLER_HIP_ERR_INVALID;
    if (a->num_tokens == 0) return SIMPLER_HIP_OK;
    if (!a->q_proj || !a->k_proj || !a->v_proj || !a->rope_cos || !a->rope_sin || !a->positions || !a->q_out ||
        !a->key_cache || !a->value_cache)
        return SIMPLER_HIP_ERR_INVALID;
    RotaryParams P{};
    P.q = a->q_proj;
    P.k = a->k_proj;
    P.v = a->v_proj;
    P.inv_rms = a->inv_rms;
    P.q_w = a->q_norm_weight;
    P.k_w = a->k_norm_weight;
    P.cos = a->rope_cos;
    P.sin = a->rope_sin;
    P.pos = a->positions;
    P.slot = a->slot_mapping;
    P.q_out = (uint16_t *)a->q_out;
    P.kc = (uint16_t *)a->key_cache;
    P.vc = (uint16_t *)a->value_cache;
    P.err = a->error_count;
    P.q_s = a->q_stride;
    P.k_s = a->k_stride;
    P.v_s = a->v_stride;
    P.k_bs = a->k_block_stride;
    P.k_ts = a->k_token_stride;
    P.k_hs = a->k_head_stride;
    P.v_bs = a->v_block_stride;
    P.v_ts = a->v_token_stride;
    P.v_hs = a->v_head_stride;
    P.tokens = a->num_tokens;
    P.hq = a->num_heads;
    P.hkv = a->num_kv_heads;
    P.d = a->head_dim;
    P.bs = a->block_size;
    P.num_blocks = a->num_blocks;
    P.max_pos = a->max_position;
    P.axes = a->num_axes;
    P.interleaved = a->interleaved;
    for (int i = 0; i < a->num_axes; ++i) P.sect[i] = a->sections[i];
    P.f16 = f16;
    P.eps = a->eps;
    // The vector form: 16 bytes per load and store.
    bool vec = a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256;
    for (int64_t s : strides) vec &= s % 8 == 0;
    const void *const aligned[6] = {a->q_proj, a->k_proj, a->v_proj, a->q_out, a->key_cache, a->value_cache};
    for (const void *p : aligned) vec &= !unaligned(p, 16);
    const int64_t heads = (int64_t)a->num_heads + 2 * (int64_t)a->num_kv_heads;
    const RotaryFn fn = a->proj_dtype == SIMPLER_HIP_DT_FLOAT32    ? pick_rotary<kF32>(a->head_dim, vec)
                        : a->proj_dtype == SIMPLER_HIP_DT_BFLOAT16 ? pick_rotary<kBf16>(a->head_dim, vec)
                                                                   : pick_rotary<kF16>(a->head_dim, vec);
    int64_t groups;
    int threads = 64;
    if (vec) {
        const int per = 1024 / a->head_dim;
        P.sets = (int)((heads + per - 1) / per);
        P.sets_per_wave = sets_per_wave(a->num_tokens, P.sets);
        const int64_t waves = (int64_t)a->num_tokens * ((P.sets + P.sets_per_wave - 1) / P.sets_per_wave);
        if (waves >= (int64_t)1 << 31) return SIMPLER_HIP_ERR_UNSUPPORTED;
        threads = kThreadsR;
        groups = (waves + kThreadsR / 64 - 1) / (kThreadsR / 64);
    } else {
        groups = a->num_tokens * heads;
    }
    if (heads >= (int64_t)1 << 30 || groups >= (int64_t)1 << 31) return SIMPLER_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3((unsigned)threads), 0, (hipStream_t)stream, P);
    return hipGetLastError() == hipSuccess ? SIMPLER_HIP_OK : SIMPLER_HIP_ERR_LAUNCH;
}
