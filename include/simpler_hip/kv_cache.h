/* KV-cache append and the fused decode prelude (q/k RMS norm + RoPE + append)
 * on gfx950 (MI355X).
 *
 * These replace the step before paged-attention decode in simpler's Qwen3
 * decode layer: the current token's K/V written into the paged BSND pool at
 * slot_mapping (simpler_setup/goldens/qwen3_14b_decode.py:106-115,261-269),
 * and the prelude that produces them and the query
 * (qwen3_14b_decode.py:207-226): per-head RMS norm with a learned weight,
 * half-split RoPE at position seq_len - 1, bf16 rounding. In the reference the
 * prelude and the cache write are phase 0 of the fused attention task
 * (examples/a2a3/tensormap_and_ringbuffer/qwen3_14b_decode/kernels/vendor/
 * paged_attention_cce/kernel/fai_body.hpp:199-230, rope_qkv with
 * slot_mapping, k_cache, v_cache); here they are their own launches on the
 * caller's stream, ahead of simpler_hip_pa_decode.
 *
 * All pointers are device pointers; strides are in elements; caches are
 * [num_blocks, block_size, num_kv_heads, head_dim] bf16 with unit stride in the
 * head dim. A slot is physical_block * block_size + offset_in_block. Negative
 * slots are skipped (padding tokens). Slots past the pool and positions
 * outside the RoPE table are skipped and counted in *error_count when that
 * optional device counter is given. Both calls allocate nothing and are
 * asynchronous on `stream` (a hipStream_t, NULL = default stream).
 */
#ifndef SIMPLER_HIP_KV_CACHE_H
#define SIMPLER_HIP_KV_CACHE_H

#include <stdint.h>

#include "simpler_hip/pa_decode.h" /* error codes */

#ifdef __cplusplus
extern "C" {
#endif

#pragma GCC visibility push(default)

typedef struct SimplerHipKvAppendArgs {
    const void *key;             /* [num_tokens, num_kv_heads, head_dim_k] bf16 */
    const void *value;           /* [num_tokens, num_kv_heads, head_dim_v] bf16; NULL: K only (MLA latent) */
    const int32_t *slot_mapping; /* [num_tokens] */
    void *key_cache;
    void *value_cache; /* NULL when value is NULL */
    int32_t *error_count;
    int64_t key_token_stride, key_head_stride;
    int64_t value_token_stride, value_head_stride;
    int64_t k_block_stride, k_token_stride, k_head_stride;
    int64_t v_block_stride, v_token_stride, v_head_stride;
    int32_t num_tokens, num_kv_heads, head_dim_k, head_dim_v, block_size, num_blocks;
} SimplerHipKvAppendArgs;

/* Write each token's K (and V) rows into the paged caches at its slot
 * (qwen3_14b_decode.py:261-269). head dims: multiples of 8, at most 1024;
 * 16-byte aligned rows. */
int simpler_hip_kv_append(const SimplerHipKvAppendArgs *args, void *stream);

typedef struct SimplerHipQkNormRopeAppendArgs {
    const float *q_proj;         /* [batch, num_heads * head_dim] fp32 */
    const float *k_proj;         /* [batch, num_kv_heads * head_dim] fp32 */
    const float *v_proj;         /* [batch, num_kv_heads * head_dim] fp32 */
    const float *inv_rms;        /* [batch] fp32: rsqrt(mean(h^2) + eps) of the hidden state */
    const float *q_norm_weight;  /* [head_dim] fp32 */
    const float *k_norm_weight;  /* [head_dim] fp32 */
    const float *rope_cos;       /* [max_position, head_dim] fp32 */
    const float *rope_sin;       /* [max_position, head_dim] fp32 */
    const int32_t *seq_lens;     /* [batch]: the token's position is seq_len - 1 */
    const int32_t *slot_mapping; /* [batch] */
    void *q_out;                 /* [batch, num_heads, head_dim] bf16 */
    void *key_cache;
    void *value_cache;
    int32_t *error_count;
    int64_t k_block_stride, k_token_stride, k_head_stride;
    int64_t v_block_stride, v_token_stride, v_head_stride;
    int32_t batch, num_heads, num_kv_heads, head_dim, block_size, num_blocks, max_position;
    float eps;
} SimplerHipQkNormRopeAppendArgs;

/* q = rope(rmsnorm(q_proj * inv_rms) * q_norm_weight), k likewise with
 * k_norm_weight, v = v_proj * inv_rms, all rounded to bf16; q to q_out, k and
 * v into the caches at slot_mapping (qwen3_14b_decode.py:207-226,261-269).
 * head_dim even, at most 1024. A token whose position is outside the RoPE
 * table gets a zero q and no cache write. */
int simpler_hip_qk_norm_rope_append(const SimplerHipQkNormRopeAppendArgs *args, void *stream);

/*
 * Caches of 4 bits per value. A row of head_dim values is cut into groups of
 * `kv_group`; a group is held as codes c in 0..15 with an fp16 scale s and zero
 * z and stands for c s + z. In fp32, each operation rounded to nearest even:
 *   lo, hi = the group's least and greatest value
 *   z = fp16(min(max(lo, -65504), 65504)),  s = fp16(min((hi - lo) / 15, 65504))
 *   c = min(max(round((x - z) / s), 0), 15), exact, ties to even; 0 where s is 0
 * so an element is at most s / 2 from its value, plus fp16's rounding of lo and
 * hi. A group with an infinity or NaN has NaN for s and z.
 *
 * Pages: key_cache and value_cache hold block_size * head_dim / 2 bytes per
 * (block, kv head), at blk*block_stride + head*head_stride bytes; scales are
 * fp16 [num_blocks, num_kv_heads, head_dim / kv_group, block_size, 2] (s, z).
 * Inside a page (little endian; nibble 0 is a byte's low one):
 *   K, row t of head_dim / 2 bytes: 32-bit word (head_dim/32) a + j, nibble i
 *     holds dim 32 j + 8 a + i  (a < 4, i < 8).
 *   V, rows 4 g .. 4 g + 3 together, 2 head_dim bytes: word (head_dim/32) l + p,
 *     l < 16, p = h + (head_dim/64) b, holds rows 4 g + 2 b (low half) and + 1
 *     (high half); nibble 2 u + v of a half is dim 64 h + 32 u + 2 l + v.
 * This is the order in which simpler_hip_pa_decode's matrix operands take
 * them. head_dim 64, 128 or 256; kv_group 32, 64 or 128, at most four groups
 * per row; block_size 16, 32, 64 or 128. No counterpart in the reference.
 *
 * simpler_hip_kv4_append quantises rows of `dtype` BFLOAT16 or FLOAT16 into
 * their slots; simpler_hip_kv4_gather reads slots back as rows of `dtype`
 * BFLOAT16, FLOAT16 or FLOAT32 (key and value are written then). Negative slots
 * are skipped by the append and give zero rows; slots past the pool likewise,
 * and are counted in *error_count. Slots in one append have to differ. Row
 * strides in elements: multiples of 8; rows and pages 16-byte aligned.
 */
typedef struct SimplerHipKv4Args {
    void *key;   /* [num_tokens, num_kv_heads, head_dim] */
    void *value; /* the same */
    const int32_t *slot_mapping;
    void *key_cache;
    void *value_cache;
    void *k_scale;
    void *v_scale;
    int32_t *error_count;
    int64_t key_token_stride, key_head_stride;
    int64_t value_token_stride, value_head_stride;
    int64_t k_block_stride, k_head_stride; /* bytes */
    int64_t v_block_stride, v_head_stride;
    int32_t num_tokens, num_kv_heads, head_dim, block_size, num_blocks, kv_group, dtype, reserved;
} SimplerHipKv4Args;

int simpler_hip_kv4_append(const SimplerHipKv4Args *args, void *stream);
int simpler_hip_kv4_gather(const SimplerHipKv4Args *args, void *stream);

/*
 * The prelude with rotary positions of several axes (time, height, width, ...),
 * for tokens of text, images and video: pair i of a head (dims i and i +
 * head_dim/2) turns by the angle of its axis' position,
 *   lo' = lo cos[p, i] - hi sin[p, i],  hi' = hi cos[p, i + D/2] + lo sin[p, i + D/2],
 *   p = positions[axis(i), token].
 * Sections count the pairs of each axis and sum to head_dim / 2. In order:
 * the first sections[0] pairs turn by axis 0, the next sections[1] by axis 1,
 * and so on. Interleaved: pair i turns by axis a = i mod num_axes where i <
 * num_axes * sections[a], else by axis 0.
 * Before that, as simpler_hip_qk_norm_rope_append: q and k are scaled by
 * inv_rms and RMS normed with their weights, v scaled by inv_rms; each of
 * inv_rms, q_norm_weight and k_norm_weight may be NULL, which leaves its step
 * out. One axis with sections {head_dim / 2} and positions seq_len - 1 is that
 * entry. All results are rounded to `dtype`: q to q_out, k and v into the caches
 * at slot_mapping; with slot_mapping NULL token t's rows go to t * token_stride
 * of key_cache and value_cache (plain rows, e.g. for simpler_hip_kv4_append).
 * A token whose position on axis 0 is negative is padding: a zero q, no cache
 * rows. One with another position outside the RoPE table likewise, and it is
 * counted in *error_count. head_dim: even, at most 1024.
 */
#define SIMPLER_HIP_MROPE_MAX_AXES 4
typedef struct SimplerHipQkNormMropeArgs {
    const void *q_proj;           /* [num_tokens, num_heads * head_dim] of proj_dtype */
    const void *k_proj;           /* [num_tokens, num_kv_heads * head_dim] */
    const void *v_proj;           /* [num_tokens, num_kv_heads * head_dim] */
    const float *inv_rms;         /* [num_tokens] or NULL */
    const float *q_norm_weight;   /* [head_dim] or NULL */
    const float *k_norm_weight;   /* [head_dim] or NULL */
    const float *rope_cos;        /* [max_position, head_dim] */
    const float *rope_sin;        /* [max_position, head_dim] */
    const int32_t *positions;     /* [num_axes, num_tokens] */
    const int32_t *slot_mapping;  /* [num_tokens] or NULL */
    void *q_out;                  /* [num_tokens, num_heads, head_dim] of dtype */
    void *key_cache;
    void *value_cache;
    int32_t *error_count;
    int64_t q_stride, k_stride, v_stride; /* elements per token of the projections */
    int64_t k_block_stride, k_token_stride, k_head_stride;
    int64_t v_block_stride, v_token_stride, v_head_stride;
    int32_t num_tokens, num_heads, num_kv_heads, head_dim, block_size, num_blocks, max_position;
    int32_t proj_dtype; /* FLOAT32, BFLOAT16 or FLOAT16 */
    int32_t dtype;      /* BFLOAT16 or FLOAT16 */
    int32_t num_axes, interleaved;
    int32_t sections[SIMPLER_HIP_MROPE_MAX_AXES];
    float eps;
} SimplerHipQkNormMropeArgs;

int simpler_hip_qk_norm_mrope_append(const SimplerHipQkNormMropeArgs *args, void *stream);

#pragma GCC visibility pop

#ifdef __cplusplus
}
#endif

#endif /* SIMPLER_HIP_KV_CACHE_H */
