// The k best continuations of a group of beams over beams x vocabulary.
//
// score(beam, token) = cum[beam] + (x - log sum exp x), in 64 bits: sums of log-probabilities lie close together between beams, and 32
// bits would order some of them wrongly. A row's k best are found by its logits alone (same order), the rows' lists then meet.
#include "common.cuh"
#include "../../include/tenzo_kernels.h"

#include <cfloat>

namespace tz {

constexpr int kBsThreads = 512;

// A logit as it counts: NaN never chosen before anything else, infinity as the largest number.
__device__ __forceinline__ float beam_logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }
// Order of the floats as integers, and -0 as +0.
__device__ __forceinline__ uint32_t beam_key(float f) {
    const uint32_t b = f == 0.0f ? 0u : __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct BeamRow {                                          // one of a row's best
    double score;
    int token;
};

// One CTA a row: the sum of exponentials, then k times the largest of what is left.
__global__ void __launch_bounds__(kBsThreads) beam_rows_kernel(const tenzo_beam_select_args a) {
    __shared__ double s_sum[kBsThreads / 32];
    __shared__ unsigned long long s_key[kBsThreads / 32];
    __shared__ float s_max[kBsThreads / 32];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* x = a.logits + (size_t)row * a.row_stride;
    const double cum = (double)a.scores[row];
    BeamRow* out = static_cast<BeamRow*>(a.workspace) + (size_t)row * a.k;
    const bool done = a.finished && a.finished[row] != 0 && cum > -INFINITY;
    float m = -INFINITY;
    for (int i = tid; i < a.vocab; i += kBsThreads) m = fmaxf(m, beam_logit(x[i]));
    m = block_max(m, s_max);
    const bool none = done || m == -INFINITY || !(cum > -INFINITY);
    double sum = 0.0;
    if (!none)
        for (int i = tid; i < a.vocab; i += kBsThreads) sum += exp((double)beam_logit(x[i]) - (double)m);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kBsThreads / 32; ++w) sum += s_sum[w];
    if (none) {                                           // the lowest tokens, all with -inf; a finished beam's end token in front
        for (int i = tid; i < a.k; i += kBsThreads) {
            const int token = !done ? i : i == 0 ? a.eos : i - 1 < a.eos ? i - 1 : i;
            out[i] = {done && i == 0 ? cum : -(double)INFINITY, token < a.vocab ? token : -1};
        }
        return;
    }
    const double lse = (double)m + log(sum);
    unsigned long long last = ~0ull;
    for (int r = 0; r < a.k; ++r) {
        unsigned long long best = 0;
        for (int i = tid; i < a.vocab; i += kBsThreads) {
            const unsigned long long key = ((unsigned long long)beam_key(beam_logit(x[i])) << 32) | (0xffffffffu - (unsigned)i);
            if (key < last && key > best) best = key;
        }
        for (int o = 16; o > 0; o >>= 1) { const unsigned long long v = __shfl_xor_sync(0xffffffffu, best, o); best = v > best ? v : best; }
        __syncthreads();
        if (lane == 0) s_key[warp] = best;
        __syncthreads();
        for (int w = 0; w < kBsThreads / 32; ++w) best = s_key[w] > best ? s_key[w] : best;
        last = best;
        if (tid == 0) {
            const int token = best ? (int)(0xffffffffu - (unsigned)best) : -1;
            out[r] = {token < 0 ? -(double)INFINITY : cum + ((double)beam_logit(x[token]) - lse), token};
        }
        if (!best) last = 0;
    }
}

// One CTA a group: a candidate's place is the number of candidates in front of it.
__global__ void __launch_bounds__(kBsThreads) beam_groups_kernel(const tenzo_beam_select_args a) {
    const int g = blockIdx.x, n = a.beams * a.k;
    const BeamRow* in = static_cast<const BeamRow*>(a.workspace) + (size_t)g * n;
    for (int i = threadIdx.x; i < n; i += kBsThreads) {
        const BeamRow c = in[i];
        if (c.token < 0) continue;
        int before = 0;
        for (int j = 0; j < n; ++j) {
            const BeamRow o = in[j];
            if (o.token >= 0 && (o.score > c.score || (o.score == c.score && j < i))) ++before;
        }
        if (before < a.k) {
            const size_t to = (size_t)g * a.k + before;
            a.parent_out[to] = i / a.k;
            a.token_out[to] = c.token;
            a.score_out[to] = (float)c.score;
        }
    }
}

}  // namespace tz

extern "C" size_t tenzo_cuda_beam_select_workspace_bytes(int groups, int beams, int vocab, int k) {
    if (groups <= 0 || beams <= 0 || vocab <= 0 || k <= 0) return 0;
    return (size_t)groups * beams * k * sizeof(tz::BeamRow);
}

extern "C" int tenzo_cuda_beam_select(const tenzo_beam_select_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    tenzo_beam_select_args a = *args;
    if (a.groups == 0) return 0;
    if (!a.logits || !a.scores || !a.parent_out || !a.token_out || !a.score_out || !a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 15)) return -1;
    if (a.groups < 0 || a.vocab <= 0 || a.beams < 1 || a.k < 1 || a.k > (long long)a.beams * a.vocab) return -1;
    if (a.finished && (a.eos < 0 || a.eos >= a.vocab)) return -1;
    if (a.beams > TENZO_BEAMS_MOST || a.k > 2 * TENZO_BEAMS_MOST) return -5;
    if (a.row_stride == 0) a.row_stride = a.vocab;
    if (a.row_stride < a.vocab) return -1;
    if (a.workspace_bytes < tenzo_cuda_beam_select_workspace_bytes(a.groups, a.beams, a.vocab, a.k)) return -1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    beam_rows_kernel<<<a.groups * a.beams, kBsThreads, 0, st>>>(a);
    beam_groups_kernel<<<a.groups, kBsThreads, 0, st>>>(a);
    return (int)cudaGetLastError();
}
