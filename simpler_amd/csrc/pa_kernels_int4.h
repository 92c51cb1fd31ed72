// GQA decode over 4-bit caches: pages of 4-bit codes with an fp16 scale s and
// zero z per token and group of G dims (include/simpler_hip/kv_cache.h); a code
// c stands for c s + z.
//
// Mathematics. Nothing is dequantised into a 16-bit value. With per-token s, z
//   q . k_t = sum_g s_tg (sum_{d in g} q_d c_td) + z_tg (sum_{d in g} q_d)
//   out_d   = (sum_t (p_t s_tg) c'_td + sum_t p_t z'_tg) / sum_t p_t
// (c' = c - 8, z' = z + 8 s: centred codes, so that the two sums do not cancel
// each other where attention averages many tokens). The sums over d and over t
// run on the matrix cores with fp16 operands, which hold codes exactly:
// - Q as fp16 times a power of two per row, exact for bf16 and fp16 queries
//   (elements 2^-27 below the row's largest lose bits, less than fp32 sums do).
// - K's codes as fp16 subnormals: masking a nibble in place gives c 2^-24 or
//   c 2^-20, no conversion; the factors go into Q and the softmax scale. The
//   matrix core aligns products by their operands' nominal exponents, so small
//   terms lose some 2^-15 of the largest one: 2e-5 of a logit, far below a
//   16-bit result's rounding. EXACT (fp32 output) converts to centred integers.
// - V's codes by (nibble | 0x6400) = 1024 + c and one packed subtraction to c'.
// - p_t s_tg rounded to fp16 (2^-11 relative at most, half a step; the error
//   averages out over tokens); EXACT splits it into two fp16 terms (2^-22).
// l = sum p and sum p z' stay in fp32, unrounded (z' itself is held in fp16
// unless EXACT: 2^-11 of a value near 0, below the fp16 p s).
//
// Softmax frame: p is taken relative to 2^F, F = (row's frame maximum) + k. The
// frame moves only when a score passes it by 2^8, and k, one exponent for the
// wave, keeps s 2^-k at 2^6 or less: p s then stays in fp16's normal range
// whatever the scales' magnitude, and nothing is rescaled in most chunks.
//
// Layout. A wave takes 64 tokens (a chunk) at a time, four 16-token tiles, with
// any block size that is a multiple of 16: S^T = K Q^T leaves a lane row
// pc = lane % 16 and tokens 4 qd + e (qd = lane / 16) of each tile, which is the
// A operand of P V over two tiles. The pages' order of nibbles is the operands'
// own: a lane loads D/8 consecutive bytes per tile for K and for V.
// Few rows. Up to 8 (4) query rows per kv head would leave half (three quarters)
// of the score lanes without a row. There lane pc takes row pc % (16 / C) of
// token tile pc / (16 / C) out of every C tiles (C = 2, 4): Q is in all the
// columns, a lane keeps its own tile's products, and the softmax runs on 64 / C
// tokens' worth of registers per chunk. In P V a lane's operand is zero where the
// k-steps are another tile's, so the C copies of a row add up to it at the end.
// Scales: lane i loads token i's, the wave shares them through LDS.
// K(i+1) is loaded into K(i)'s registers right after QK(i), V(i+1) after PV(i).
//
// What bounds it, measured (8 kv heads of 128 dims unless said; one call with its
// merge, which takes 5 to 8 us of it; GB/s of all the bytes it has to move):
// - Up to 8 rows: HBM. 32 sequences of 1024 to 8192 tokens, 4 rows, G = 64: 42.5 us,
//   4310 GB/s; the main kernel 36.5 us (5020), its loads without the arithmetic 34.9.
//   8 of 32768, 8 rows, G = 128: 57.5 us, 4970 GB/s.
// - 16 rows and more, or many groups: VALU instructions, on codes, scales and softmax
//   of 64 tokens x 16 rows about 800 per chunk (G = 32), half of the SIMD's issue
//   slots over the kernel and 70% while both its waves run. 13 sequences of 700 to
//   9000, 32 rows, G = 32, fp16: 50.3 us, 1760 GB/s. With fp32 output the splits
//   add to them: 37 of 300 to 5000, 4 kv heads of 64 dims, 7 rows: 23.2 us, 1350 GB/s.
// - Short contexts: latency, about 2.1 us per chunk of a wave after 6 us
//   (int4_direct_waves in pa_decode.hip).
// Tried without gain: three waves per SIMD by fewer registers, a scheduling
// barrier between the tiles, pages loaded through the caches (2 to 5% slower), the
// row tiles of a kv head as waves of a workgroup (their K and V come from L2).
#pragma once

#include "pa_kernels_direct.h"

namespace simpler_hip {
namespace pa {

// Four 16-bit pairs out of the eight nibbles of x, nibble n of the low and of
// the high half: as fp16 subnormals c 2^-24 (n even) and c 2^-20 (n odd).
__device__ __forceinline__ u32x4_t nibbles_subnormal(const unsigned x) {
    const unsigned y = x >> 8;
    return (u32x4_t){x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
}

// The same pairs as fp16 integers c - 8, exact: 1024 + c - 1032 and
// (1024 + 16 c) / 16 - 72. The masks and the 1024s come in registers (`low`,
// `high`, `k1024`), for one v_and_or_b32 per pair: as literals they take an and
// and an or.
__device__ __forceinline__ u32x4_t nibbles_centred(const unsigned x, const unsigned low, const unsigned high,
                                                   const unsigned k1024) {
    const f16x2_t off = (f16x2_t){(_Float16)-1032.f, (_Float16)-1032.f};
    const f16x2_t sixteenth = (f16x2_t){(_Float16)0.0625f, (_Float16)0.0625f};
    const f16x2_t off16 = (f16x2_t){(_Float16)-72.f, (_Float16)-72.f};
    const unsigned y = x >> 8;
    const f16x2_t a = __builtin_bit_cast(f16x2_t, (x & low) | k1024) + off;
    const f16x2_t b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, (x & high) | k1024), sixteenth, off16);
    const f16x2_t c = __builtin_bit_cast(f16x2_t, (y & low) | k1024) + off;
    const f16x2_t d = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, (y & high) | k1024), sixteenth, off16);
    return (u32x4_t){__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, c),
                     __builtin_bit_cast(unsigned, d)};
}

__device__ __forceinline__ float half_lo(const unsigned x) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(x & 0xffffu));
}
__device__ __forceinline__ float half_hi(const unsigned x) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(x >> 16));
}

constexpr int kInt4Chunk = 64;  // tokens a wave takes at a time

// LDS of one wave: the chunk's K and V scales, one or (EXACT) two words each.
template <int NG, bool EXACT>
constexpr int int4_wave_lds() {
    return 2 * NG * kInt4Chunk * (EXACT ? 8 : 4);
}

// Two neighbouring output values of a 16-bit (bf16, or fp16 with f16) or fp32 output.
template <bool F32>
__device__ __forceinline__ void int4_store2(void *out, const int64_t off, const float a, const float b, const bool f16) {
    if constexpr (F32) {
        *reinterpret_cast<f32x2_t *>(reinterpret_cast<float *>(out) + off) = (f32x2_t){a, b};
    } else {
        *reinterpret_cast<unsigned *>(reinterpret_cast<uint16_t *>(out) + off) =
            f16 ? Elem<_Float16>::pack2(a, b) : pack_bf16x2(a, b);
    }
}

// Tokens [seg_begin, seg_end) (seg_begin a multiple of 16, seg_end at most ctx)
// of the row tiles rt .. rt + RTW - 1 of (b, kvh): the final output where they
// are the whole tile, else a piece each (see finish_segment). D: head dim, NG:
// groups per row. `lds`: this wave's int4_wave_lds bytes.
template <int D, int NG, int RTW, int C, bool EXACT>
__device__ __forceinline__ void run_int4_segment(const KernelParams &P, const int b, const int kvh, const int rt,
                                                 const int ctx, const int seg_begin, const int seg_end,
                                                 const bool whole, float *const part_o, float *const part_ml,
                                                 char *const lds) {
    constexpr int KS = D / 32;    // 32-dim k-steps of QK
    constexpr int GM = KS / NG;   // k-steps per group
    constexpr int DT = D / 16;    // 16-dim tiles of PV
    constexpr int GT = DT / NG;   // dim tiles per group
    constexpr int LW = D / 32;    // words of codes per lane and tile
    constexpr int DH = D / 64;    // words per lane, tile and token pair of V
    constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
    constexpr float kSlack = 8.f;  // a score may pass the frame by 2^kSlack
    constexpr int R16 = 16 / C;   // rows of a tile
    constexpr int NS = 4 / C;     // sets of C token tiles
    static_assert(D % 64 == 0 && KS % NG == 0, "head dims: multiples of 64, groups of whole k-steps");
    static_assert(C == 1 || RTW == 1, "several row tiles: 16 rows each");
    const int lane = threadIdx.x & 63, qd = lane >> 4, pc = lane & 15;
    const int tq = pc / R16, pr = pc % R16;  // this lane's token tile of a set, its row
    const int sh = P.page_shift, bs = 1 << sh;
    const bool f16 = P.half16;
    // constants of the conversions, kept in registers
    unsigned low = 0x000f000fu, high = 0x00f000f0u, k1024 = 0x64006400u;
    asm volatile("" : "+s"(low), "+s"(high));
    asm volatile("" : "+v"(k1024));
    auto centred = [&](const unsigned x) { return nibbles_centred(x, low, high, k1024); };

    // ---- the query's rows ----
    u32x4_t raw[RTW][KS];
    int rowlim[RTW];  // first token the row does not see (within the segment's end)
#pragma unroll
    for (int r = 0; r < RTW; ++r) {
        rowlim[r] = 0;
#pragma unroll
        for (int j = 0; j < KS; ++j) raw[r][j] = (u32x4_t){0u, 0u, 0u, 0u};
        if (pr < min(16, P.rows - (rt + r) * 16)) {
            const int row = (rt + r) * 16 + pr, i = row / P.group, hh = row - i * P.group;
            const uint16_t *qrow = P.q + ((int64_t)(b * P.q_len + i) * P.num_heads + kvh * P.group + hh) * D;
#pragma unroll
            for (int j = 0; j < KS; ++j) raw[r][j] = ld16(qrow + 32 * j + 8 * qd);
            rowlim[r] = min(seg_end, P.causal ? ctx - (P.q_len - 1 - i) : ctx);
        }
    }
    const int32_t *const table_row = P.block_table + (int64_t)b * (P.max_blocks * P.block_size >> sh);
    const __attribute__((address_space(4))) int32_t *bt_row =
        (const __attribute__((address_space(4))) int32_t *)table_row;
    const char *k_head = reinterpret_cast<const char *>(P.k) + (int64_t)kvh * P.k_head_stride;
    const char *v_head = reinterpret_cast<const char *>(P.v) + (int64_t)kvh * P.v_head_stride;
    const unsigned *k_sc = reinterpret_cast<const unsigned *>(P.k_scale);
    const unsigned *v_sc = reinterpret_cast<const unsigned *>(P.v_scale);
    const uint32_t k_lane = pc * (D / 2) + qd * (D / 8), v_lane = lane * (D / 8);

    const int last_tile = (seg_end - 1) & ~15;  // tiles past it read this one again (masked)
    int raw_id[4];
    auto read_ids = [&](const int tok0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) raw_id[t] = bt_row[min(tok0 + 16 * t, last_tile) >> sh];
    };
    int page[4];       // the chunk's tiles' blocks
    unsigned bad = 0;  // tiles in out-of-pool blocks
    auto resolve = [&] {
        bad = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            int id = __builtin_amdgcn_readfirstlane(raw_id[t]);
            if ((unsigned)id >= (unsigned)P.num_pool_blocks) {
                bad |= 1u << t;
                id = 0;
            }
            page[t] = id;
        }
    };
    auto row_of = [&](const int tok0, const int t) { return min(tok0 + 16 * t, last_tile) & (bs - 1); };  // in its page
    unsigned ksr[NG], vsr[NG];
    auto load_scales = [&](const int tok0) {
        const int64_t pg = qd == 0 ? page[0] : qd == 1 ? page[1] : qd == 2 ? page[2] : page[3];
        const int64_t at = (pg * P.kv_heads + kvh) * (int64_t)(NG * bs) + row_of(tok0, qd) + pc;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            ksr[g] = k_sc[at + g * bs];
            vsr[g] = v_sc[at + g * bs];
        }
    };
    unsigned kreg[4][LW], vreg[4][LW];
    auto load_codes = [&](unsigned (&dst)[LW], const char *p) {
        if constexpr (LW == 2) {
            const u32x2_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t *>(p));
            dst[0] = w[0], dst[1] = w[1];
        } else {
#pragma unroll
            for (int i = 0; i < LW / 4; ++i) {
                const u32x4_t w = stream_ld16(p + 16 * i);
                dst[4 * i] = w[0], dst[4 * i + 1] = w[1], dst[4 * i + 2] = w[2], dst[4 * i + 3] = w[3];
            }
        }
    };
    auto load_k = [&](const int tok0) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
            load_codes(kreg[t], k_head + page[t] * P.k_block_stride + row_of(tok0, t) * (D / 2) + k_lane);
    };
    auto load_v = [&](const int tok0) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
            load_codes(vreg[t], v_head + page[t] * P.v_block_stride + row_of(tok0, t) * (D / 2) + v_lane);
    };

    // Everything that the first chunk needs is on its way before the query is
    // waited for: its rows, then (the block ids are scalar loads) scales, K, V.
    read_ids(seg_begin);
    resolve();
    load_scales(seg_begin);
    load_k(seg_begin);
    load_v(seg_begin);
    read_ids(seg_begin + kInt4Chunk);

    // ---- Q in the codes' nibble order, exponent-aligned ----
    u32x4_t qv[RTW][KS];
    float zq[RTW][NG];  // sum of the group's q, in the units of the scores
    float xs[RTW];      // scores to log2 units
#pragma unroll
    for (int r = 0; r < RTW; ++r) {
        float f[KS][8], amax = 0.f;
        if (f16) {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) f[j][2 * i] = half_lo(raw[r][j][i]), f[j][2 * i + 1] = half_hi(raw[r][j][i]);
        } else {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f[j][2 * i] = __uint_as_float(raw[r][j][i] << 16);
                    f[j][2 * i + 1] = __uint_as_float(raw[r][j][i] & 0xffff0000u);
                }
        }
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[j][i]));
        amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
        amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
        // the row times 2^(140 - eb): its largest element in [2^13, 2^14)
        const int eb = min(max((int)(__float_as_uint(amax) >> 23), 27), 240);
        float up = __uint_as_float((unsigned)(267 - eb) << 23);
        if (P.scale < 0.f) up = -up;  // the scores' sign, so that their maximum is the softmax's
        const float sub = EXACT ? 1.f : 0.0625f;  // nibbles at bits 4..7: 16 c
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float s = 0.f;
#pragma unroll
            for (int j = g * GM; j < (g + 1) * GM; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) s += f[j][i];
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            zq[r][g] = s * up * (EXACT ? 1.f : 0x1p-24f);
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            const float u16 = up * sub;
            qv[r][j] = (u32x4_t){Elem<_Float16>::pack2(f[j][0] * up, f[j][4] * up),
                                 Elem<_Float16>::pack2(f[j][1] * u16, f[j][5] * u16),
                                 Elem<_Float16>::pack2(f[j][2] * up, f[j][6] * up),
                                 Elem<_Float16>::pack2(f[j][3] * u16, f[j][7] * u16)};
        }
        xs[r] = fabsf(P.scale) * kLog2e * __uint_as_float((unsigned)(eb - 13) << 23) * (EXACT ? 1.f : 0x1p24f);
        xs[r] = fmaxf(xs[r], 0x1p-120f);  // scale 0: masked scores stay -inf (0 times inf is NaN)
    }
    // tokens before this one are seen by every row of the wave's tiles
    const int all_see = P.causal ? ctx - (P.q_len - 1 - (rt * 16) / P.group) : ctx;

    f32x4_t acc[RTW][DT];
    float lsum[RTW], zacc[RTW][NG], fy[RTW], nf[RTW], thr[RTW];
    int kexp = -64;  // exponent of the frame that the V scales set
    float slim = 0x1p-58f;
#pragma unroll
    for (int r = 0; r < RTW; ++r) {
#pragma unroll
        for (int j = 0; j < DT; ++j) acc[r][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < NG; ++g) zacc[r][g] = 0.f;
        lsum[r] = 0.f;
        fy[r] = -INFINITY;
        nf[r] = 0.f;
        thr[r] = -INFINITY;
    }

    unsigned *const kst = reinterpret_cast<unsigned *>(lds);  // [g][token]: s, z (EXACT: fp32 s, z + 8 s)
    unsigned *const vst = kst + NG * kInt4Chunk * (EXACT ? 2 : 1);
    bool first = true;

    auto step = [&](const int tok0, auto has_next) {
        constexpr bool NEXT = decltype(has_next)::value;
        // ---- the chunk's scales into LDS; zeros for tokens that are not there ----
        const unsigned bad_now = bad;
        const bool there = tok0 + lane < seg_end && !((bad_now >> qd) & 1);
        float smax = 0.f;
        // A token with a scale or zero that is not finite makes the rows that
        // see it NaN and must not reach the others (0 times NaN): V's goes in
        // as 0, and the token's score is NaN, which masking removes.
        bool odd = false;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const unsigned k_high = ksr[g] & 0x7c007c00u, v_high = vsr[g] & 0x7c007c00u;
            odd |= (k_high & 0xffffu) == 0x7c00u || k_high >> 16 == 0x7c00u || (v_high & 0xffffu) == 0x7c00u ||
                   v_high >> 16 == 0x7c00u;
        }
        wave_lds_sync();
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const unsigned kw = !there ? 0u : odd ? 0x7e007e00u : ksr[g], vw = there && !odd ? vsr[g] : 0u;
            const float vs = half_lo(vw), vz = __builtin_fmaf(8.f, vs, half_hi(vw));
            smax = fmaxf(smax, vs);
            if constexpr (EXACT) {
                const float ks = half_lo(kw);
                reinterpret_cast<f32x2_t *>(kst)[g * kInt4Chunk + lane] =
                    (f32x2_t){ks, __builtin_fmaf(8.f, ks, half_hi(kw))};
                reinterpret_cast<f32x2_t *>(vst)[g * kInt4Chunk + lane] = (f32x2_t){vs, vz};
            } else {
                kst[g * kInt4Chunk + lane] = kw;
                vst[g * kInt4Chunk + lane] = Elem<_Float16>::pack2(vs, vz);
            }
        }
        if (bad_now && lane == 0) atomicOr(P.error_flag, kErrBadBlock);
        if constexpr (NEXT) {
            resolve();
            load_scales(tok0 + kInt4Chunk);
            read_ids(tok0 + 2 * kInt4Chunk);
        }
        wave_lds_sync();
        // scale and zero of tokens 4qd .. 4qd+3 of this lane's tile of set u
        auto scales_of = [&](const unsigned *st, const int g, const int u, f32x4_t &s, f32x4_t &z) {
            const int at = g * kInt4Chunk + 16 * C * u + 16 * tq + 4 * qd;
            if constexpr (EXACT) {
                const f32x4_t *p = reinterpret_cast<const f32x4_t *>(st) + at / 2;
                const f32x4_t a = p[0], c = p[1];
                s = (f32x4_t){a[0], a[2], c[0], c[2]};
                z = (f32x4_t){a[1], a[3], c[1], c[3]};
            } else {
                const u32x4_t w = *reinterpret_cast<const u32x4_t *>(st + at);
                s = (f32x4_t){half_lo(w[0]), half_lo(w[1]), half_lo(w[2]), half_lo(w[3])};
                z = (f32x4_t){half_hi(w[0]), half_hi(w[1]), half_hi(w[2]), half_hi(w[3])};
            }
        };

        // ---- scores ----
        f32x4_t y[RTW][NS];
#pragma unroll
        for (int u = 0; u < NS; ++u) {
            f32x4_t own[RTW][NG];  // q . c of this lane's tile
#pragma unroll
            for (int i = 0; i < C; ++i) {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    f32x4_t dot[RTW];
#pragma unroll
                    for (int j = g * GM; j < (g + 1) * GM; ++j) {
                        const u32x4_t a = EXACT ? centred(kreg[u * C + i][j]) : nibbles_subnormal(kreg[u * C + i][j]);
#pragma unroll
                        for (int r = 0; r < RTW; ++r)
                            dot[r] = Elem<_Float16>::mma32(a, qv[r][j],
                                                           j == g * GM ? (f32x4_t){0.f, 0.f, 0.f, 0.f} : dot[r]);
                    }
#pragma unroll
                    for (int r = 0; r < RTW; ++r)
#pragma unroll
                        for (int e = 0; e < 4; ++e) own[r][g][e] = i == 0 || tq == i ? dot[r][e] : own[r][g][e];
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4_t s, z;
                scales_of(kst, g, u, s, z);
#pragma unroll
                for (int r = 0; r < RTW; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // (adding 0 in a fused form takes fp16 operands as they are)
                        const float zz = __builtin_fmaf(z[e], zq[r][g], g == 0 ? 0.f : y[r][u][e]);
                        y[r][u][e] = __builtin_fmaf(s[e], own[r][g][e], zz);
                    }
            }
        }
        if constexpr (NEXT) load_k(tok0 + kInt4Chunk);

        // ---- frame ----
        if (tok0 + kInt4Chunk > min(seg_end, all_see) || bad_now) {  // some row does not see some token
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                const int t = C * u + tq;
#pragma unroll
                for (int r = 0; r < RTW; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (tok0 + 16 * t + 4 * qd + e >= rowlim[r] || ((bad_now >> t) & 1)) y[r][u][e] = -INFINITY;
            }
        }
        float ymax[RTW];
        bool move = first || smax > slim;
#pragma unroll
        for (int r = 0; r < RTW; ++r) {
            ymax[r] = -INFINITY;
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) ymax[r] = fmaxf(ymax[r], y[r][u][e]);
            move |= ymax[r] > thr[r];
        }
        if (__any(move)) {
            first = false;
#pragma unroll
            for (int i = 1; i < 64; i <<= 1) smax = fmaxf(smax, __shfl_xor(smax, i, 64));
            const int ex = (int)(__float_as_uint(smax) >> 23) - 127;  // smax < 2^(ex + 1); fp16, so normal in fp32
            const int knew = smax > 0.f ? max(kexp, min(ex, 16) - 5) : kexp;
            const float kdown = ldexpf(1.f, kexp - knew);
            kexp = knew;
            slim = ldexpf(1.f, knew + 6);
#pragma unroll
            for (int r = 0; r < RTW; ++r) {
                float m = fmaxf(ymax[r], __shfl_xor(ymax[r], 16, 64));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                if constexpr (C >= 2) m = fmaxf(m, __shfl_xor(m, 8, 64));
                if constexpr (C >= 4) m = fmaxf(m, __shfl_xor(m, 4, 64));
                m = fmaxf(m, fy[r]);
                const float a =
                    (fy[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((fy[r] - m) * xs[r])) * kdown;
                fy[r] = m;
                nf[r] = m == -INFINITY ? 0.f : -__builtin_fmaf(m, xs[r], (float)knew);
                thr[r] = m == -INFINITY ? m : m + kSlack / xs[r];
                lsum[r] *= a;
#pragma unroll
                for (int g = 0; g < NG; ++g) zacc[r][g] *= a;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ae = __shfl(a, 4 * qd + e, 64);  // rows 4qd+e
#pragma unroll
                    for (int j = 0; j < DT; ++j) acc[r][j][e] *= ae;
                }
            }
        }

        // ---- p, its sums, and P V: two tiles at a time ----
        f32x4_t p[RTW][2];  // of the sets in hand
        u32x2_t ps[RTW][NG][2], pl[RTW][NG][2];  // p s, the A operands (EXACT: and what its rounding left)
        auto weights = [&](const int i, const int u) {
#pragma unroll
            for (int r = 0; r < RTW; ++r) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    p[r][i][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[r][u][e], xs[r], nf[r]));
                lsum[r] += (p[r][i][0] + p[r][i][1]) + (p[r][i][2] + p[r][i][3]);
            }
        };
        auto scaled = [&](const int i, const int u, const int g) {
            f32x4_t s, z;
            scales_of(vst, g, u, s, z);
#pragma unroll
            for (int r = 0; r < RTW; ++r) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = __builtin_fmaf(p[r][i][e], s[e], 0.f);
                    zacc[r][g] = __builtin_fmaf(p[r][i][e], z[e], zacc[r][g]);
                }
                const u32x2_t w = {Elem<_Float16>::pack2(v[0], v[1]), Elem<_Float16>::pack2(v[2], v[3])};
                ps[r][g][i] = w;
                if constexpr (EXACT)
                    pl[r][g][i] = (u32x2_t){Elem<_Float16>::pack2(v[0] - half_lo(w[0]), v[1] - half_hi(w[0])),
                                            Elem<_Float16>::pack2(v[2] - half_lo(w[1]), v[3] - half_hi(w[1]))};
            }
        };
#pragma unroll
        for (int t = 0; t < 4; t += 2) {
            if constexpr (C == 1) {
                weights(0, t);
                weights(1, t + 1);
            } else if (t % C == 0) {
                weights(0, t / C);
#pragma unroll
                for (int g = 0; g < NG; ++g) scaled(0, t / C, g);
            }
            // A's first four k of a lane are tile t's tokens, the others tile t + 1's: with C > 1 a lane has one
            // of the set's tiles and zeros for the others
            auto operand = [&](const u32x2_t (&w)[2]) {
                if constexpr (C == 1) return (u32x4_t){w[0][0], w[0][1], w[1][0], w[1][1]};
                const bool even = tq == t % C, odd = tq == t % C + 1;
                return (u32x4_t){even ? w[0][0] : 0u, even ? w[0][1] : 0u, odd ? w[0][0] : 0u, odd ? w[0][1] : 0u};
            };
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if constexpr (C == 1) {
                    scaled(0, t, g);
                    scaled(1, t + 1, g);
                }
                u32x4_t pa[RTW], pb[RTW];
#pragma unroll
                for (int r = 0; r < RTW; ++r) {
                    pa[r] = operand(ps[r][g]);
                    if constexpr (EXACT) pb[r] = operand(pl[r][g]);
                }
#pragma unroll
                for (int h = 0; h < DH; ++h) {
                    if (4 * h + 3 < g * GT || 4 * h >= (g + 1) * GT) continue;  // no dim tile of this group
                    const u32x4_t a = centred(vreg[t][h]), c = centred(vreg[t][DH + h]);
                    const u32x4_t a2 = centred(vreg[t + 1][h]), c2 = centred(vreg[t + 1][DH + h]);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int j = 4 * h + n;
                        if (j / GT != g) continue;
                        const u32x4_t vv = (u32x4_t){a[n], c[n], a2[n], c2[n]};
#pragma unroll
                        for (int r = 0; r < RTW; ++r) {
                            acc[r][j] = Elem<_Float16>::mma32(pa[r], vv, acc[r][j]);
                            if constexpr (EXACT) acc[r][j] = Elem<_Float16>::mma32(pb[r], vv, acc[r][j]);
                        }
                    }
                }
            }
        }
        if constexpr (NEXT) load_v(tok0 + kInt4Chunk);
    };

    int tok0 = seg_begin;
    for (; tok0 + kInt4Chunk < seg_end; tok0 += kInt4Chunk) step(tok0, std::true_type{});
    step(tok0, std::false_type{});

    // ---- output or pieces: lane holds rows 4qd+e, dims 32u + 2pc, + 1; with
    // C > 1 each tile of a set has its own copy of a row, summed here ----
    auto over_tiles = [&](float x) {  // over the copies in the lanes pc
        if constexpr (C >= 2) x += __shfl_xor(x, 8, 64);
        if constexpr (C >= 4) x += __shfl_xor(x, 4, 64);
        return x;
    };
#pragma unroll
    for (int r = 0; r < RTW; ++r) {
        const int rows_here = min(16, P.rows - (rt + r) * 16);
        if (rows_here <= 0) break;
        float l = lsum[r];
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        l = over_tiles(l);
        float z[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            z[g] = zacc[r][g] + __shfl_xor(zacc[r][g], 16, 64);
            z[g] += __shfl_xor(z[g], 32, 64);
            z[g] = over_tiles(z[g]);
        }
        if constexpr (C > 1) {
#pragma unroll
            for (int j = 0; j < DT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[r][j][e] += __shfl_xor(acc[r][j][e], 32, 64);
                    if constexpr (C >= 4) acc[r][j][e] += __shfl_xor(acc[r][j][e], 16, 64);
                }
        }
        float *const po = part_o + r * (2 * 16 * D), *const pml = part_ml + r * (2 * 32);
        const int part = C == 4 ? qd : C == 2 ? qd >> 1 : 0;  // lanes with the same rows share the dims out
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = (4 * qd + e) % R16;
            const float le = __shfl(l, row, 64), inv = le > 0.f ? 1.f / le : le != le ? le : 0.f;
            float ze[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) ze[g] = __shfl(z[g], row, 64);
            if (row >= rows_here) continue;
            const int64_t off = out_row_offset(P, b, kvh, (rt + r) * 16 + row, D) + 2 * pc;
#pragma unroll
            for (int u = 0; u < D / 32; ++u) {
                if (C > 1 && u % C != part) continue;
                const float v0 = acc[r][2 * u][e] + ze[2 * u / GT], v1 = acc[r][2 * u + 1][e] + ze[2 * u / GT];
                if (whole)
                    int4_store2<EXACT>(P.out, off + 32 * u, le != 0.f ? v0 * inv : 0.f, le != 0.f ? v1 * inv : 0.f, f16);
                else
                    *reinterpret_cast<f32x2_t *>(po + row * D + 32 * u + 2 * pc) = (f32x2_t){v0, v1};
            }
        }
        if (!whole && qd == 0 && tq == 0) {
            pml[pc] = fy[r] == -INFINITY ? kNegClamp : -nf[r] * kLn2;
            pml[16 + pc] = l;
        }
    }
}

// One wave per worker, RTW row tiles each; work lists as in pa_decode_kernel.
template <int D, int NG, int RTW, int C, bool EXACT>
__global__ void __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2)))
pa_int4_kernel(const KernelParams P) {
    __shared__ __attribute__((aligned(16))) char lds[int4_wave_lds<NG, EXACT>()];
    flag_bad_lengths(P);
    const int w = blockIdx.x, unit = P.block_size;
    const int tpb = lane_tiles(P);
    const int list = w % P.lanes;
    int start = 0, end = 0, b = 0, prefix = 0, ctx0 = 0;
    locate_slice(P, w / P.lanes, &start, &end, &b, &prefix, &ctx0);
    start = __builtin_amdgcn_readfirstlane(start);
    end = __builtin_amdgcn_readfirstlane(end);
    b = __builtin_amdgcn_readfirstlane(b);
    prefix = __builtin_amdgcn_readfirstlane(prefix);
    if (start >= end) return;
    int ctx = __builtin_amdgcn_readfirstlane(ctx0);
    int nb = (ctx + unit - 1) / unit;
    if (nb == 0) return;
    // A tile takes seg_cost units of work, for the set-up and the end of a wave's
    // part of it, then one per 64 tokens (or smaller page); the slice runs those it holds.
    int j = (start - prefix) / (nb + P.seg_cost), t0 = prefix + j * (nb + P.seg_cost), slot = 0;
    while (nb > 0) {
        const int blk0 = max(0, start - t0 - P.seg_cost), blk1 = min(nb, end - t0 - P.seg_cost);
        if (blk1 > blk0) {
            const int jt = list_tile0(P, list, b) + j;
            const int kvh = jt / P.row_groups, rg = jt - kvh * P.row_groups;
            const int64_t piece = (int64_t)w * RTW * 2 + slot;
            run_int4_segment<D, NG, RTW, C, EXACT>(P, b, kvh, rg * RTW, ctx, blk0 * unit, min(ctx, blk1 * unit),
                                                   blk1 - blk0 == nb, P.part_o + piece * 16 * D, P.part_ml + piece * 32,
                                                   lds);
            slot = 1;
        }
        t0 += nb + P.seg_cost;
        if (t0 >= end) break;
        if (++j == tpb) {
            j = 0;
            do {
                ++b;
                ctx = __builtin_amdgcn_readfirstlane(ctx_of(P, b));
                nb = (ctx + unit - 1) / unit;
            } while (nb == 0 && b + 1 < P.batch);
        }
    }
}

// Short contexts: one workgroup per 16-row tile, its chunks shared out among
// the waves, which meet in LDS (pa_kernels_direct.h).
template <int D>
constexpr int int4_direct_waves() {
    return D <= 128 ? 8 : 4;  // their pieces share the 160 KB of LDS
}
template <int D, int NG, bool EXACT>
constexpr int int4_direct_lds() {
    return 16 * D * 4 + 32 * 4 + int4_wave_lds<NG, EXACT>();
}

template <int D, int NG, int C, typename OutT>
__global__ void __launch_bounds__((64 * int4_direct_waves<D>())) pa_int4_direct_kernel(const KernelParams P) {
    constexpr bool EXACT = std::is_same<OutT, float>::value;
    constexpr int LW = int4_direct_lds<D, NG, EXACT>();
    extern __shared__ __attribute__((aligned(16))) char int4_lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int per_seq = P.kv_heads * P.row_tiles;
    const int b = blockIdx.x / per_seq, jr = blockIdx.x - b * per_seq;
    const int kvh = jr / P.row_tiles, rt = jr - kvh * P.row_tiles;
    const int rows_here = min(16, P.rows - rt * 16);
    const int len = P.context_lens[b];
    const int cap = P.max_blocks * P.block_size;
    if (threadIdx.x == 0 && (len < (P.causal ? P.q_len : 0) || len > cap)) atomicOr(P.error_flag, kErrBadLength);
    const int ctx = __builtin_amdgcn_readfirstlane(min(max(len, 0), cap));
    const int chunks = (ctx + kInt4Chunk - 1) / kInt4Chunk;
    const int per = (chunks + waves - 1) / waves;
    const int units = rows_here * (D / 4);
    if (chunks == 0) {  // empty context: defined as a zero output
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            const int row = u / (D / 4);
            OutStore<OutT>::store4(P.out, out_row_offset(P, b, kvh, rt * 16 + row, D) + 4 * (u - row * (D / 4)),
                                   (f32x4_t){0.f, 0.f, 0.f, 0.f});
        }
        return;
    }
    char *const lds = int4_lds + wave * LW;
    float *const part = reinterpret_cast<float *>(lds);
    const int lo = wave * per, hi = min(chunks, lo + per);
    if (lo < hi)
        run_int4_segment<D, NG, 1, C, EXACT>(P, b, kvh, rt, ctx, lo * kInt4Chunk, min(ctx, hi * kInt4Chunk),
                                          chunks <= per, part, part + 16 * D, lds + 16 * D * 4 + 32 * 4);
    const int pieces = (chunks + per - 1) / per;
    if (pieces == 1) return;  // wave 0 stored the output
    __syncthreads();
    direct_merge<D, OutT, int4_direct_waves<D>(), LW>(P, b, kvh, rt, units, pieces, int4_lds);
}

// The kernels for `rows` query rows per kv head. Two row tiles per wave: not
// with 256 dims, whose accumulators alone are 128 registers then.
// Token tiles side by side for up to four rows: four, two where 128 dims are one
// group and the output has 16 bits. us per call, 4 / 2 tiles, 32 sequences of 1024
// to 8192, 8 kv heads, 4 rows: 64 dims, G = 64 32.5 / 34.8, G = 32 and fp32 40.2 / 43.2;
// 128 dims, G = 32 45.7 / 47.1, G = 64 42.5 / 42.3, G = 128 40.2 / 39.7 and with one row
// 42.3 / 37.9, with fp32 41.1 / 42.0; 256 dims (16 x 4 kv heads), one row 28.2 / 29.5.
// (For 5 to 8 rows, 2 tiles / 1: 6 rows of 128 dims 35.7 / 36.6, 7 rows of 64
// dims, fp32 23.1 / 24.4.)
template <int D, int NG, bool EXACT>
constexpr int int4_few() {
    return D == 128 && NG == 1 && !EXACT ? 2 : 4;
}

template <int D, int NG, bool EXACT>
KernelPair int4_set(const int rows) {
    KernelPair k{};
    k.main = rows <= 4 ? pa_int4_kernel<D, NG, 1, int4_few<D, NG, EXACT>(), EXACT>
             : rows <= 8 ? pa_int4_kernel<D, NG, 1, 2, EXACT> : pa_int4_kernel<D, NG, 1, 1, EXACT>;
    if constexpr (D <= 128) k.main_pair = pa_int4_kernel<D, NG, 2, 1, EXACT>;
    return k;
}

template <int D, int NG>
KernelPair int4_pair(const int rows, const int out_dtype) {
    return out_dtype == SIMPLER_HIP_DT_FLOAT32 ? int4_set<D, NG, true>(rows) : int4_set<D, NG, false>(rows);
}

template <int D, int NG, typename OutT>
DirectFn int4_direct_set(const int rows) {
    constexpr int lds = int4_direct_lds<D, NG, std::is_same<OutT, float>::value>();
    return {rows <= 4   ? pa_int4_direct_kernel<D, NG, 4, OutT>
            : rows <= 8 ? pa_int4_direct_kernel<D, NG, 2, OutT> : pa_int4_direct_kernel<D, NG, 1, OutT>,
            int4_direct_waves<D>(), lds};
}

template <int D, int NG>
DirectFn int4_direct(const int rows, const int out_dtype) {
    return out_dtype == SIMPLER_HIP_DT_FLOAT32    ? int4_direct_set<D, NG, float>(rows)
           : out_dtype == SIMPLER_HIP_DT_BFLOAT16 ? int4_direct_set<D, NG, __bf16>(rows)
                                                  : int4_direct_set<D, NG, _Float16>(rows);
}

}  // namespace pa
}  // namespace simpler_hip
