// Block tables and slot maps of a serving step (include/simpler_hip/
// step_plan.h), gfx950.
//
// Both kernels are a prefix sum over the requests (blocks given back, blocks
// and tokens taken) and then independent work per block and per token. They are
// bound by latency: a decode step moves a few KB. So each is one launch, in
// which every workgroup works the sums out for itself from the lengths (two
// loads of `batch` ints, 16 KB at most, from L2 for all but the first) and
// keeps them in LDS, instead of a scan launch and an expansion that waits for
// it. The tokens, the blocks and the requests are shared out among the
// workgroups; a token finds its request by binary search in the sums. Measured:
// 256 requests of a token each 2.7 us (release) and 4.7 us (assign), 1024
// requests with 60 prompts of up to 8000 tokens 4.1 and 8.7. Four tokens per
// thread, one search for them, took 7.7 and 10.8 (their table entries are read
// one after the other); 64-bit scans through LDS 1.2 and 2.4 us more.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "simpler_hip/step_plan.h"

namespace simpler_hip_step {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;

// a + b, at most 2^32 - 1: sums that pass it (lengths that no step has) stay there.
__device__ __forceinline__ unsigned sat_add(const unsigned a, const unsigned b) {
    return __builtin_elementwise_add_sat(a, b);
}

// Inclusive sum over the lanes, by DPP moves: within rows of 16, then each row's
// last lane into the rows after it.
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
#define SIMPLER_DPP(ctrl, rows) (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
    x = sat_add(x, SIMPLER_DPP(0x111, 0xf));  // row_shr 1
    x = sat_add(x, SIMPLER_DPP(0x112, 0xf));  // row_shr 2
    x = sat_add(x, SIMPLER_DPP(0x114, 0xf));  // row_shr 4
    x = sat_add(x, SIMPLER_DPP(0x118, 0xf));  // row_shr 8
    x = sat_add(x, SIMPLER_DPP(0x142, 0xa));  // lane 15 of rows 0 and 2 into rows 1 and 3
    x = sat_add(x, SIMPLER_DPP(0x143, 0xc));  // lane 31 into rows 2 and 3
#undef SIMPLER_DPP
    return x;
}

// Inclusive sum of x over the workgroup's threads; *total: of all of them.
__device__ __forceinline__ unsigned block_scan(unsigned x, unsigned (&sums)[kWaves], unsigned *total) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    x = wave_scan(x);
    __syncthreads();  // the last use of `sums` is over
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    unsigned before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before = sat_add(before, sums[w]);
        all = sat_add(all, sums[w]);
    }
    *total = all;
    return sat_add(before, x);
}

__device__ __forceinline__ int saturate(const unsigned x) { return (int)min(x, 0x7fffffffu); }

// Blocks of a length of 0 or more.
__device__ __forceinline__ int blocks_of(const int len, const int bs) {
    return (int)(((unsigned)len + (unsigned)(bs - 1)) / (unsigned)bs);
}

// Tokens that a table row holds, as far as a length counts.
__device__ __forceinline__ int row_capacity(const int width, const int bs) {
    return (int)min((int64_t)width * bs, (int64_t)0x7fffffff);
}

// First index in 0 .. n whose (non-decreasing) value is above x.
__device__ __forceinline__ int first_above(const int *v, const int n, const int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] > x)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

struct ReleaseParams {
    const int32_t *ended, *lens, *table, *count;
    int32_t *free_blocks, *lens_out, *count_out, *err;
    int32_t batch, width, bs, capacity;
};

__global__ void __launch_bounds__(kThreads) release_kernel(const ReleaseParams P) {
    extern __shared__ int upto[];  // blocks given back by requests 0 .. b
    __shared__ unsigned sums[kWaves];
    const int cap = row_capacity(P.width, P.bs);
    const int count = min(max(P.count[0], 0), P.capacity);
    unsigned carry = 0;
    int bad = 0;
    for (int base = 0; base < P.batch; base += kThreads) {
        const int b = base + threadIdx.x;
        int n = 0;
        if (b < P.batch) {
            const int ended = P.ended[b], len = P.lens[b];
            bad += ended && (len < 0 || len > cap);
            n = ended ? blocks_of(min(max(len, 0), cap), P.bs) : 0;
        }
        unsigned total;
        const unsigned incl = block_scan(n, sums, &total);
        if (b < P.batch) upto[b] = saturate(sat_add(carry, incl));
        carry = sat_add(carry, total);
    }
    __syncthreads();
    const int room = P.capacity - count, all = saturate(carry), given = min(all, room);
    const int thread = blockIdx.x * kThreads + threadIdx.x, threads = gridDim.x * kThreads;
    for (int i = thread; i < given; i += threads) {
        const int b = first_above(upto, P.batch, i);
        P.free_blocks[count + i] = P.table[(int64_t)b * P.width + i - (b ? upto[b - 1] : 0)];
    }
    for (int b = thread; b < P.batch; b += threads) P.lens_out[b] = P.ended[b] ? 0 : P.lens[b];
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) {
            P.count_out[0] = count + given;
            bad += all > room;
        }
        if (bad && P.err) atomicAdd(P.err, bad);
    }
}

struct AssignParams {
    const int32_t *new_lens, *lens, *free_blocks, *count;
    int32_t *table, *slots, *positions, *requests, *starts, *lens_out, *granted, *count_out, *err;
    int32_t batch, width, bs, capacity, tokens;
};

__global__ void __launch_bounds__(kThreads) assign_kernel(const AssignParams P) {
    extern __shared__ int lds[];
    int *const ends = lds;                // tokens of requests 0 .. b
    int *const upto = lds + P.batch;      // blocks that requests 0 .. b ask for
    int *const lens = lds + 2 * P.batch;  // of the requests that get their tokens, else -1
    __shared__ unsigned sums[kWaves];
    const int cap = row_capacity(P.width, P.bs);
    const int count = min(max(P.count[0], 0), P.capacity);
    unsigned tok_carry = 0, blk_carry = 0;
    int taken = 0;  // by this thread's requests
    int refused = 0;
    const bool lead = blockIdx.x == 0;
    for (int base = 0; base < P.batch; base += kThreads) {
        const int b = base + threadIdx.x;
        int len = 0, n = 0;
        if (b < P.batch) {
            len = P.lens[b];
            n = P.new_lens[b];
        }
        unsigned total;
        const unsigned end = sat_add(tok_carry, block_scan(max(n, 0), sums, &total));
        tok_carry = sat_add(tok_carry, total);
        const bool fits = n >= 0 && len >= 0 && n <= cap && len <= cap - n && end <= (unsigned)P.tokens;
        const int need = fits ? blocks_of(len + n, P.bs) - blocks_of(len, P.bs) : 0;
        const unsigned asked = sat_add(blk_carry, block_scan(need, sums, &total));
        blk_carry = sat_add(blk_carry, total);
        if (b < P.batch) {
            const bool ok = fits && (need == 0 || asked <= (unsigned)count);
            ends[b] = saturate(end);
            upto[b] = saturate(asked);
            lens[b] = ok ? len : -1;
            if (ok) taken += need;
            refused += !ok;
            if (lead) {
                P.starts[b + 1] = ends[b];
                P.granted[b] = ok ? n : 0;
                P.lens_out[b] = ok ? len + n : len;
            }
        }
    }
    __syncthreads();

    struct Request {
        int len, had, first;  // first: blocks asked for before it
        bool ok;
    };
    auto request = [&](const int b) {
        Request r;
        r.len = lens[b];
        r.ok = r.len >= 0;
        r.first = b ? upto[b - 1] : 0;
        r.had = blocks_of(max(r.len, 0), P.bs);
        return r;
    };
    const int thread = blockIdx.x * kThreads + threadIdx.x, threads = gridDim.x * kThreads;

    // the blocks: entry i of all that are asked for, as far as the stack goes
    const int given = (int)min(blk_carry, (unsigned)count);
    for (int i = thread; i < given; i += threads) {
        const int b = first_above(upto, P.batch, i);
        const Request r = request(b);
        if (r.ok) P.table[(int64_t)b * P.width + r.had + i - r.first] = P.free_blocks[count - 1 - i];
    }

    // the tokens
    const int used = saturate(tok_carry);
    for (int64_t i = thread; i < P.tokens; i += threads) {
        const int t = (int)i;
        int slot = -1, pos = -1, req = -1;
        if (t < used) {
            const int b = first_above(ends, P.batch, t);
            const Request r = request(b);
            if (r.ok) {
                pos = r.len + t - (b ? ends[b - 1] : 0);
                req = b;
                const int blk = (int)((unsigned)pos / (unsigned)P.bs);
                const int phys = blk < r.had ? P.table[(int64_t)b * P.width + blk]
                                             : P.free_blocks[count - 1 - (r.first + blk - r.had)];
                slot = phys < 0 ? -1 : (int)min((int64_t)phys * P.bs + (pos - blk * P.bs), (int64_t)0x7fffffff);
            }
        }
        P.slots[t] = slot;
        P.positions[t] = pos;
        P.requests[t] = req;
    }
    if (lead) {
        unsigned all_taken, all_refused;
        (void)block_scan(taken, sums, &all_taken);
        (void)block_scan(refused, sums, &all_refused);
        if (threadIdx.x == 0) {
            P.starts[0] = 0;
            P.count_out[0] = count - (int)all_taken;
            if (all_refused && P.err) atomicAdd(P.err, (int)all_refused);
        }
    }
}

bool bad_common(const int32_t batch, const int32_t width, const int32_t bs, const int32_t capacity) {
    return batch < 0 || width < 1 || bs < 1 || capacity < 0;
}

// Enough workgroups for `items` of a thread each, as many as the card has CUs at most.
unsigned grid_for(const int64_t items) {
    return (unsigned)std::min<int64_t>(std::max<int64_t>((items + kThreads - 1) / kThreads, 1), 256);
}

}  // namespace
}  // namespace simpler_hip_step

using namespace simpler_hip_step;

extern "C" int simpler_hip_release_blocks(const SimplerHipReleaseBlocksArgs *a, void *stream) {
    if (!a || bad_common(a->batch, a->max_blocks_per_seq, a->block_size, a->capacity)) return SIMPLER_HIP_ERR_INVALID;
    if (!a->free_count || !a->free_count_out || (a->capacity > 0 && !a->free_blocks) ||
        (a->batch > 0 && (!a->ended || !a->context_lens || !a->block_table || !a->context_lens_out)))
        return SIMPLER_HIP_ERR_INVALID;
    if ((a->batch > 0 && a->context_lens_out == a->context_lens) || a->free_count_out == a->free_count)
        return SIMPLER_HIP_ERR_INVALID;
    if (a->batch > SIMPLER_HIP_STEP_MAX_BATCH) return SIMPLER_HIP_ERR_UNSUPPORTED;
    ReleaseParams P{a->ended,           a->context_lens,   a->block_table, a->free_count,         a->free_blocks,
                    a->context_lens_out, a->free_count_out, a->error_count, a->batch, a->max_blocks_per_seq,
                    a->block_size,      a->capacity};
    const unsigned grid = grid_for((int64_t)a->batch * 8);
    hipLaunchKernelGGL(release_kernel, dim3(grid), dim3(kThreads), (size_t)std::max(a->batch, 1) * 4,
                       (hipStream_t)stream, P);
    return hipGetLastError() == hipSuccess ? SIMPLER_HIP_OK : SIMPLER_HIP_ERR_LAUNCH;
}

extern "C" int simpler_hip_assign_slots(const SimplerHipAssignSlotsArgs *a, void *stream) {
    if (!a || bad_common(a->batch, a->max_blocks_per_seq, a->block_size, a->capacity)) return SIMPLER_HIP_ERR_INVALID;
    if (!a->free_count || !a->free_count_out || !a->starts || (a->capacity > 0 && !a->free_blocks) ||
        (a->batch > 0 && (!a->new_lens || !a->context_lens || !a->block_table || !a->context_lens_out || !a->granted)))
        return SIMPLER_HIP_ERR_INVALID;
    if (a->num_tokens < 0 || (a->num_tokens > 0 && (!a->slot_mapping || !a->positions || !a->requests)))
        return SIMPLER_HIP_ERR_INVALID;
    if ((a->batch > 0 && (a->context_lens_out == a->context_lens || a->granted == a->new_lens)) ||
        a->free_count_out == a->free_count)
        return SIMPLER_HIP_ERR_INVALID;
    if (a->batch > SIMPLER_HIP_STEP_MAX_BATCH) return SIMPLER_HIP_ERR_UNSUPPORTED;
    AssignParams P{a->new_lens,  a->context_lens, a->free_blocks,      a->free_count, a->block_table,
                   a->slot_mapping, a->positions, a->requests,         a->starts,     a->context_lens_out,
                   a->granted,   a->free_count_out, a->error_count,    a->batch,      a->max_blocks_per_seq,
                   a->block_size, a->capacity,    a->num_tokens};
    const unsigned grid = grid_for(std::max(a->num_tokens, a->batch));
    hipLaunchKernelGGL(assign_kernel, dim3(grid), dim3(kThreads), (size_t)std::max(a->batch, 1) * 12,
                       (hipStream_t)stream, P);
    return hipGetLastError() == hipSuccess ? SIMPLER_HIP_OK : SIMPLER_HIP_ERR_LAUNCH;
}
