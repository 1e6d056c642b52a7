// The end of a block of tiles in the kernel of received weights (attention_tree.cu): the sums of its keys, which lie in shared memory, are added to the weights. Plain C++ beside
// its loads, so that the host can run it too.
#pragma once
#include "kv8.cuh"

namespace tz {

__host__ __device__ __forceinline__ float weigh_load(const float* p) {
#ifdef __CUDA_ARCH__
    return ld_l2(p);
#else
    return *p;
#endif
}

// Thread `tid` of ALL adds the sums of the keys of tiles t0 .. t1 - 1, of `total` keys in all, from s_sum [GROUPS][MOST][TILE]. The tiles are the last ones before the n-th, whose chunks' rows
// are remembered in s_rows [ROWS_MOST][TILE / CHUNK] (-1: none). given_up: a wait was given up, so that neither rows nor sums need have been written; nothing is then.
template <int GROUPS, int MOST, int ROWS_MOST, int ALL, int TILE, int CHUNK>
__host__ __device__ __forceinline__ void weigh_add(bool given_up, int tid, int n, int t0, int t1, int total, const int* s_rows, const float* s_sum, float* weight) {
    if (given_up) return;
    constexpr int kBatch = 8;                            // loads in flight
    for (int k0 = tid; k0 < (t1 - t0) * TILE; k0 += kBatch * ALL) {
        int row[kBatch];
        float old[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int k = k0 + u * ALL, i = k / TILE;
            const bool there = k < (t1 - t0) * TILE && t0 * TILE + k < total;
            row[u] = there ? s_rows[(n - (t1 - t0) + i) % ROWS_MOST * (TILE / CHUNK) + (k % TILE) / CHUNK] : -1;
            if (row[u] >= 0) row[u] += k % CHUNK;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) old[u] = weigh_load(weight + (row[u] > 0 ? row[u] : 0));      // (something, where there is none)
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            float sum = 0.0f;
            if (row[u] < 0) continue;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) sum += s_sum[g * MOST * TILE + k0 + u * ALL];
            weight[row[u]] = old[u] + sum;
        }
    }
}

}  // namespace tz
