// Where a launch's tokens go in the paged caches: a caller's slot mapping, or
// (the decode entries' paged form) the block-table row of each sequence.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "simpler_hip/pa_decode.h"

namespace simpler_hip_kv {

// The paged form's token -> (position, slot) inputs; block_table null: the
// caller's slot mapping (and seq_lens) instead.
struct Paged {
    const int32_t *block_table, *context_lens;
    unsigned *error_flag;  // the decode workspace's error word
    unsigned bad_length;   // its bit for a length below q_len (or a position outside the RoPE table)
    int32_t q_len, max_blocks;
};

__device__ __forceinline__ bool slot_ok(int slot, int32_t num_blocks, int32_t block_size, int32_t *err) {
    if (slot < 0) return false;  // padding token
    if ((int64_t)slot >= (int64_t)num_blocks * block_size) {
        if (threadIdx.x == 0 && err) atomicAdd(err, 1);
        return false;
    }
    return true;
}

// Paged form: position and slot of launch token t, or slot -1 where the
// token is not written: a position below 0 (a length below q_len, reported
// by the caller of this), one past the block-table row (a length the decode
// reports), or an out-of-pool block (reported when the decode reads it).
__device__ __forceinline__ int paged_slot(const Paged &G, const int t, const int32_t block_size,
                                          const int32_t num_blocks, int *pos) {
    const int b = t / G.q_len;
    const int p = G.context_lens[b] - G.q_len + (t - b * G.q_len);
    *pos = p;
    if (p < 0 || p >= G.max_blocks * block_size) return -1;
    const int phys = G.block_table[(int64_t)b * G.max_blocks + p / block_size];
    if ((unsigned)phys >= (unsigned)num_blocks) return -1;
    return phys * block_size + p % block_size;
}

inline Paged paged_of(const SimplerHipPaDecodeArgs *a, unsigned *error_flag, unsigned bad_length) {
    Paged G{};
    G.block_table = a->block_table;
    G.context_lens = a->context_lens;
    G.error_flag = error_flag;
    G.bad_length = bad_length;
    G.q_len = a->q_len;
    G.max_blocks = a->max_blocks_per_seq;
    return G;
}

}  // namespace simpler_hip_kv
