// GQA decode attention over the 4-bit paged cache (kv4.cuh): softmax(q K^T / sqrt(128)) V over the keys 0 .. pos of a row's sequence,
// the query rotated on the way.
//
// One warp per query head and share of the keys: a lane holds four dims, the warps of a CTA join their (maximum, sum, output).
#include "kv4.cuh"

#include <cuda_fp16.h>

namespace tz {

constexpr int kA4Warps = 8, kA4Hd = 128;

__device__ int g_kv4_attention_error = 0;

__global__ void __launch_bounds__(kA4Warps * 32) attention_kv4_simple_kernel(const tenzo_attention_kv4_args a) {
    __shared__ float s_q[kA4Hd], s_o[kA4Warps][kA4Hd], s_m[kA4Warps], s_l[kA4Warps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.y, row = blockIdx.x, kvh = head / (a.n_q / a.cache.n_kv);
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const int pos = a.pos[row], seq = a.seq ? a.seq[row] : row;
    float* out = a.out + ((size_t)row * a.n_q + head) * kA4Hd;
    if (pos >= a.max_len || seq < 0 || seq >= a.cache.table_rows) {
        if (tid == 0) atomicOr(&g_kv4_attention_error, kK4ErrIndex);
        return;
    }
    const float* q = a.q + (size_t)row * a.q_stride + (size_t)head * kA4Hd;
    if (tid < 64) {
        const float x0 = q[tid], x1 = q[tid + 64];
        const bool turn = a.rope_cos && pos >= 0;
        const float c = turn ? a.rope_cos[(size_t)pos * 64 + tid] : 1.0f, s = turn ? a.rope_sin[(size_t)pos * 64 + tid] : 0.0f;
        s_q[tid] = __fmaf_rn(x0, c, -(x1 * s));
        s_q[tid + 64] = __fmaf_rn(x0, s, x1 * c);
    }
    __syncthreads();
    float qv[4], o[4] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) qv[j] = s_q[4 * lane + j] * 0.08838834764831845f;
    for (int t = warp; t <= pos; t += kA4Warps) {
        const int block = a.cache.block_table[(size_t)seq * a.cache.table_stride + t / kK4Slots];
        if (block < 0 || block >= a.cache.n_blocks) {
            if (lane == 0) atomicOr(&g_kv4_attention_error, kK4ErrIndex);
            continue;
        }
        const uint8_t* kr = a.cache.pool + kv4_page(a.cache, a.layer, kvh, block) + (size_t)(t % kK4Slots) * kK4Row;
        const uint8_t* vr = kr + kK4Half;
        const uint32_t kc = reinterpret_cast<const uint16_t*>(kr)[lane], vc = reinterpret_cast<const uint16_t*>(vr)[lane];
        const float2 kp = __half22float2(reinterpret_cast<const __half2*>(kr + kK4Codes)[lane >> 3]);
        const float2 vp = __half22float2(reinterpret_cast<const __half2*>(vr + kK4Codes)[lane >> 3]);
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) s = __fmaf_rn(qv[j], __fmaf_rn(kp.x, (float)((kc >> (4 * j)) & 15u), kp.y), s);
        s = warp_sum(s);
        const float n = fmaxf(m, s), f = expf(m - n), e = expf(s - n);
        m = n;
        l = __fmaf_rn(l, f, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __fmaf_rn(o[j], f, e * __fmaf_rn(vp.x, (float)((vc >> (4 * j)) & 15u), vp.y));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s_o[warp][4 * lane + j] = o[j];
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
    __syncthreads();
    if (tid < kA4Hd) {
        float top = -INFINITY, sum = 0.0f, v = 0.0f;
        for (int w = 0; w < kA4Warps; ++w) top = fmaxf(top, s_m[w]);
        for (int w = 0; w < kA4Warps; ++w) {
            const float f = s_m[w] == -INFINITY ? 0.0f : expf(s_m[w] - top);
            sum = __fmaf_rn(s_l[w], f, sum);
            v = __fmaf_rn(s_o[w][tid], f, v);
        }
        out[tid] = sum > 0.0f ? v / sum : 0.0f;
    }
}

int kv4_attention_take_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_kv4_attention_error, sizeof v) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_kv4_attention_error, &zero, sizeof zero);
    return v;
}
int kv4_rows_take_error();

}  // namespace tz

extern "C" size_t tenzo_cuda_attention_kv4_workspace_bytes(int rows, int n_q, int n_kv, int max_len) {
    if (rows <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_len <= 0) return 0;
    return 64;
}

extern "C" int tenzo_cuda_attention_kv4(const tenzo_attention_kv4_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    tenzo_attention_kv4_args a = *args;
    if (a.rows == 0) return 0;
    if (!kv4_cache_ok(a.cache) || !a.q || !a.out || !a.pos) return -1;
    if (a.layer < 0 || a.layer >= a.cache.n_layers || a.n_q <= 0 || a.n_q % a.cache.n_kv || a.rows < 0 || a.max_len <= 0) return -1;
    if (a.max_len > (long long)a.cache.table_stride * kK4Slots || (!a.seq && a.rows > a.cache.table_rows)) return -1;
    if ((a.rope_cos == nullptr) != (a.rope_sin == nullptr) || (a.rope_cos && a.rope_len < a.max_len)) return -1;
    if (a.split_keys < 0 || (reinterpret_cast<uintptr_t>(a.out) & 15)) return -1;
    if (a.q_stride == 0) a.q_stride = a.n_q * kA4Hd;
    if (a.q_stride < a.n_q * kA4Hd) return -1;
    return kv4_launch(attention_kv4_simple_kernel, dim3((unsigned)a.rows, (unsigned)a.n_q), kA4Warps * 32, 0, static_cast<cudaStream_t>(stream), a.use_pdl != 0, a);
}

extern "C" int tenzo_cuda_kv4_take_errors(void) {
    const int a = tz::kv4_rows_take_error(), b = tz::kv4_attention_take_error();
    return a < 0 || b < 0 ? -1 : a | b;
}
