// moe_offsets.hpp -- rows of each expert, from pairs that come grouped by expert.
#pragma once

#include "bk_common.hpp"

namespace bk {
namespace {

constexpr int kMaxExperts = 1024;

// expert_counts / expert_offsets from expert_ids (one workgroup, 1024 threads).
// The ids come grouped by expert, so a wave's 64 of them are a few runs of
// equal ids: the first lane of each run adds the run's length to the expert's
// LDS counter (any order of the ids counts right; ids outside [0, E) nowhere),
// and the counts' prefix sum runs over the 16 waves.  One ballot per expert
// and 64 ids, and the sum by one thread, took 29 us at the ids of 512 tokens, 6 of 64 experts,
// and 7.7 at 8192 of 8; now 4.6 and 5.7.
__global__ __launch_bounds__(1024) void moe_offsets_kernel(const int32_t *__restrict__ expert_ids,
                                                           int size_m, int num_experts,
                                                           int32_t *__restrict__ counts,
                                                           int32_t *__restrict__ offsets) {
    __shared__ int cnt[kMaxExperts];
    __shared__ int wsum[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    cnt[tid] = 0;
    __syncthreads();
    constexpr int U = 4;   // ids per lane requested before the first is used
    for (int i0 = 0; i0 < size_m; i0 += 1024 * U) {
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * 1024 + tid;
            id[u] = i < size_m ? expert_ids[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int prev = __shfl_up(id[u], 1, 64);
            const uint64_t heads = __ballot(lane == 0 || id[u] != prev);
            if (((heads >> lane) & 1) && id[u] >= 0 && id[u] < num_experts) {
                const uint64_t next = lane < 63 ? heads >> (lane + 1) : 0;
                atomicAdd(&cnt[id[u]], next ? __ffsll((unsigned long long)next) : 64 - lane);
            }
        }
    }
    __syncthreads();
    const int c = tid < num_experts ? cnt[tid] : 0;
    int run = c;                                  // inclusive sum over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(run, off, 64);
        if (lane >= off) run += v;
    }
    if (lane == 63) wsum[wave] = run;
    __syncthreads();
    for (int w = 0; w < wave; ++w) run += wsum[w];
    if (tid < num_experts) {
        counts[tid] = c;
        offsets[tid + 1] = run;
    }
    if (tid == 0) offsets[0] = 0;
}

}  // namespace
}  // namespace bk
