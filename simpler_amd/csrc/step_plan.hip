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
// workgroups; a token finds its request by binary search in the sums.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "simpler_hip/step_plan.h"

namespace simpler_hip_step {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kTokensPerThread = 4;  // consecutive ones: one search for them

__device__ __forceinline__ int64_t wave_scan(int64_t x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    return x;
}

// Inclusive sum of x over the workgroup's threads; *total: of all of them.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t (&sums)[kWaves], int64_t *total) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    x = wave_scan(x);
    __syncthreads();  // the last use of `sums` is over
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sums[w];
        all += sums[w];
    }
    *total = all;
    return x + before;
}

__device__ __forceinline__ int saturate(const int64_t x) { return (int)min(x, (int64_t)0x7fffffff); }

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
    __shared__ int64_t sums[kWaves];
    const int64_t cap = (int64_t)P.width * P.bs;
    const int count = min(max(P.count[0], 0), P.capacity);
    int64_t carry = 0;
    int bad = 0;
    for (int base = 0; base < P.batch; base += kThreads) {
        const int b = base + threadIdx.x;
        int n = 0;
        if (b < P.batch && P.ended[b]) {
            const int len = P.lens[b];
            bad += len < 0 || len > cap;
            n = (int)((min(max((int64_t)len, (int64_t)0), cap) + P.bs - 1) / P.bs);
        }
        int64_t total;
        const int64_t incl = block_scan(n, sums, &total);
        if (b < P.batch) upto[b] = saturate(carry + incl);
        carry += total;
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
    int *const ends = lds;            // tokens of requests 0 .. b
    int *const upto = lds + P.batch;  // blocks that requests 0 .. b ask for
    __shared__ int64_t sums[kWaves];
    const int64_t cap = (int64_t)P.width * P.bs;
    const int count = min(max(P.count[0], 0), P.capacity);
    int64_t tok_carry = 0, blk_carry = 0;
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
        int64_t total;
        const int64_t end = tok_carry + block_scan(max(n, 0), sums, &total);
        tok_carry += total;
        const bool fits = n >= 0 && len >= 0 && (int64_t)len + n <= cap && end <= P.tokens;
        const int had = fits ? (int)(((int64_t)len + P.bs - 1) / P.bs) : 0;
        const int need = fits ? (int)(((int64_t)len + n + P.bs - 1) / P.bs) - had : 0;
        const int64_t asked = blk_carry + block_scan(need, sums, &total);
        blk_carry += total;
        if (b < P.batch) {
            const bool ok = fits && (need == 0 || asked <= count);
            ends[b] = saturate(end);
            upto[b] = saturate(asked);
            if (ok) taken += need;
            refused += !ok;
            if (lead) {
                P.starts[b + 1] = ends[b];
                P.granted[b] = ok ? n : 0;
                P.lens_out[b] = ok ? len + n : len;
            }
        }
    }
    if (lead) {
        int64_t all_taken, all_refused;
        (void)block_scan(taken, sums, &all_taken);
        (void)block_scan(refused, sums, &all_refused);
        if (threadIdx.x == 0) {
            P.starts[0] = 0;
            P.count_out[0] = count - (int)all_taken;
            if (all_refused && P.err) atomicAdd(P.err, (int)all_refused);
        }
    }
    __syncthreads();

    // What request b has, may take and gets, as above.
    struct Request {
        int len, had, first;  // first: blocks asked for before it
        bool ok;
    };
    auto request = [&](const int b) {
        const int n = P.new_lens[b];
        Request r;
        r.len = P.lens[b];
        r.first = b ? upto[b - 1] : 0;
        r.ok = n >= 0 && r.len >= 0 && (int64_t)r.len + n <= cap && ends[b] <= P.tokens &&
               (upto[b] == r.first || upto[b] <= count);
        r.had = (int)(((int64_t)max(r.len, 0) + P.bs - 1) / P.bs);
        return r;
    };
    const int thread = blockIdx.x * kThreads + threadIdx.x, threads = gridDim.x * kThreads;

    // the blocks: entry i of all that are asked for, as far as the stack goes
    const int given = (int)min(blk_carry, (int64_t)count);
    for (int i = thread; i < given; i += threads) {
        const int b = first_above(upto, P.batch, i);
        const Request r = request(b);
        if (r.ok) P.table[(int64_t)b * P.width + r.had + i - r.first] = P.free_blocks[count - 1 - i];
    }

    // the tokens
    const int used = saturate(tok_carry);
    for (int64_t t0 = (int64_t)thread * kTokensPerThread; t0 < P.tokens; t0 += (int64_t)threads * kTokensPerThread) {
        int b = first_above(ends, P.batch, (int)t0);
        Request r{};
        int start = 0;
        if (b < P.batch) {
            r = request(b);
            start = b ? ends[b - 1] : 0;
        }
#pragma unroll
        for (int k = 0; k < kTokensPerThread; ++k) {
            if (t0 + k >= P.tokens) break;
            const int t = (int)t0 + k;
            if (t < used && t >= ends[b]) {
                b = first_above(ends, P.batch, t);
                r = request(b);
                start = ends[b - 1];  // t >= ends[b - 1] of the request before
            }
            int slot = -1, pos = -1, req = -1;
            if (t < used && r.ok) {
                pos = r.len + (t - start);
                req = b;
                const int blk = pos / P.bs;
                const int phys = blk < r.had ? P.table[(int64_t)b * P.width + blk]
                                             : P.free_blocks[count - 1 - (r.first + blk - r.had)];
                slot = phys < 0 ? -1 : phys * P.bs + (pos - blk * P.bs);
            }
            P.slots[t] = slot;
            P.positions[t] = pos;
            P.requests[t] = req;
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
    if ((a->batch > 0 && a->context_lens_out == a->context_lens) || a->free_count_out == a->free_count) return SIMPLER_HIP_ERR_INVALID;
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
    const unsigned grid = grid_for(std::max<int64_t>(((int64_t)a->num_tokens + kTokensPerThread - 1) / kTokensPerThread,
                                                     a->batch));
    hipLaunchKernelGGL(assign_kernel, dim3(grid), dim3(kThreads), (size_t)std::max(a->batch, 1) * 8,
                       (hipStream_t)stream, P);
    return hipGetLastError() == hipSuccess ? SIMPLER_HIP_OK : SIMPLER_HIP_ERR_LAUNCH;
}
