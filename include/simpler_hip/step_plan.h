/* Block tables and slot maps of a serving step, built on the GPU from the
 * requests' lengths, for gfx950 (MI355X).
 *
 * A serving loop keeps, per request slot, the number of cached tokens
 * (context_lens) and a row of the block table, and a stack of free block ids.
 * simpler_hip_release_blocks returns the blocks of requests that ended to the
 * stack; simpler_hip_assign_slots takes blocks from it for the new tokens of
 * the others and says where every token goes: what simpler's host code derives
 * per sequence for one token (simpler_setup/goldens/qwen3_14b_decode.py:106-115)
 * for any number of tokens per request, with nothing read back to the host, so
 * that a step can be captured in a HIP graph.
 *
 * Neither changes its inputs but for block_table's new entries and
 * free_blocks' entries past the count: the new lengths and the new count are
 * outputs of their own, and the same call again gives the same results. No
 * output may overlap an input. All pointers are device pointers to int32,
 * contiguous. Both calls allocate nothing and are asynchronous on `stream`.
 */
#ifndef SIMPLER_HIP_STEP_PLAN_H
#define SIMPLER_HIP_STEP_PLAN_H

#include <stdint.h>

#include "simpler_hip/pa_decode.h" /* error codes */

#ifdef __cplusplus
extern "C" {
#endif

#pragma GCC visibility push(default)

#define SIMPLER_HIP_STEP_MAX_BATCH 4096

typedef struct SimplerHipReleaseBlocksArgs {
    const int32_t *ended;        /* [batch]: nonzero for a request whose blocks are returned */
    const int32_t *context_lens; /* [batch] */
    const int32_t *block_table;  /* [batch, max_blocks_per_seq] */
    int32_t *free_blocks;        /* [capacity]: the free ids are the first free_count of them */
    const int32_t *free_count;   /* [1] */
    int32_t *context_lens_out;   /* [batch]: 0 where ended, else context_lens */
    int32_t *free_count_out;     /* [1] */
    int32_t *error_count;        /* or NULL */
    int32_t batch, max_blocks_per_seq, block_size, capacity;
} SimplerHipReleaseBlocksArgs;

/* free_blocks[free_count ..] = the first ceil(len / block_size) table entries of
 * every ended request, request by request; free_count_out = free_count + their
 * number. A length outside [0, max_blocks_per_seq * block_size] counts as the
 * nearest one inside and in *error_count; ids that do not fit the capacity are
 * dropped, which counts as one error. free_count is clamped to [0, capacity]. */
int simpler_hip_release_blocks(const SimplerHipReleaseBlocksArgs *args, void *stream);

typedef struct SimplerHipAssignSlotsArgs {
    const int32_t *new_lens;     /* [batch]: new tokens of each request, 0 for none */
    const int32_t *context_lens; /* [batch]: tokens cached so far */
    int32_t *block_table;        /* [batch, max_blocks_per_seq] */
    const int32_t *free_blocks;  /* [capacity] */
    const int32_t *free_count;   /* [1] */
    int32_t *slot_mapping;       /* [num_tokens] */
    int32_t *positions;          /* [num_tokens] */
    int32_t *requests;           /* [num_tokens] */
    int32_t *starts;             /* [batch + 1]: request b's tokens are starts[b] .. starts[b + 1] */
    int32_t *context_lens_out;   /* [batch] */
    int32_t *granted;            /* [batch]: new_lens, or 0 where refused */
    int32_t *free_count_out;     /* [1] */
    int32_t *error_count;        /* or NULL: refused requests are counted */
    int32_t batch, max_blocks_per_seq, block_size, capacity, num_tokens, reserved;
} SimplerHipAssignSlotsArgs;

/* The tokens of all requests, packed in request order (request b's are the
 * next new_lens[b]): token i of request b gets position context_lens[b] + i and
 * the slot of that position in the request's table row, which gets the blocks
 * it lacks from the top of the stack, free_blocks[free_count - 1] first, request
 * by request. A request gets all of its tokens or none: it is refused where
 * context_lens or new_lens is negative, where its tokens do not fit the table
 * row (or a length of 2^31 - 1) or end past num_tokens, or where it needs blocks
 * and the stack does not cover it together with every earlier request that
 * passed the other checks. A refused request's tokens keep their place with
 * slot, position and request -1, as do places past the last token; a negative
 * block id gives slot -1; starts and slots are 2^31 - 1 at most. batch at most
 * SIMPLER_HIP_STEP_MAX_BATCH. */
int simpler_hip_assign_slots(const SimplerHipAssignSlotsArgs *args, void *stream);

#pragma GCC visibility pop

#ifdef __cplusplus
}
#endif

#endif /* SIMPLER_HIP_STEP_PLAN_H */
