// Attention of drafted trees over the INT8 caches (kv8.cuh), and the weight that each cached token receives.
#include "attn_common.cuh"
#include "kv8.cuh"

namespace tz {

constexpr int kTrThreads = 128;
__device__ int g_tree_error = 0;

struct TreeLaunch {
    tenzo_attention_tree_args a;
    int group;
    float* weight;
};

__device__ __forceinline__ bool tree_sees(const tenzo_attention_tree_args& a, size_t row, int i, int start, int t) {
    const int j = t - start;
    return j < 0 || (a.mask ? ld_l2(a.mask + row * a.mask_stride + (j >> 5)) >> (j & 31) & 1 : j <= i);
}

// One warp a (row, query head), a key at a time: four dims a lane.
__global__ void __launch_bounds__(kTrThreads) attention_tree_kernel(const TreeLaunch L) {
    const tenzo_attention_tree_args& a = L.a;
    const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5), kvh = head / L.group;
    const size_t row = blockIdx.x;
    const int s = (int)(row / a.nodes), i = (int)(row % a.nodes);
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    if (head >= a.n_q) return;
    const int start = ld_l2(a.start + s), count = a.count ? ld_l2(a.count + s) : a.nodes, seq = a.seq ? ld_l2(a.seq + s) : s;
    const int pos = a.rope_pos ? ld_l2(a.rope_pos + row) : start + i;
    const bool padding = start < 0 || (count >= 0 && i >= count);
    if (!padding && (count < 0 || count > a.nodes || (long long)start + count > a.max_len || seq < 0 || seq >= a.cache.table_rows || (a.rope_cos && (pos < 0 || pos >= a.rope_len)))) {
        if (lane == 0) atomicOr(&g_tree_error, kK8ErrIndex);
        return;
    }
    const float* q = a.q + row * a.q_stride + (size_t)head * kK8Hd;
    float x[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    for (int j = 0; j < 4; ++j) {
        const int d = 4 * lane + j;
        x[j] = q[d];
        if (a.rope_cos && !padding) {
            const float c = a.rope_cos[(size_t)pos * 64 + (d & 63)], sn = a.rope_sin[(size_t)pos * 64 + (d & 63)];
            x[j] = d < 64 ? __fmaf_rn(q[d], c, -(q[d + 64] * sn)) : __fmaf_rn(q[d - 64], sn, q[d] * c);
        }
    }
    for (int t = 0; !padding && t < start + count; ++t) {
        if (!tree_sees(a, row, i, start, t)) continue;
        const int block = kv8_block(a.cache, seq, t);
        if (block < 0) {
            if (lane == 0) atomicOr(&g_tree_error, kK8ErrIndex);
            continue;
        }
        const size_t at = kv8_row(a.cache, a.layer, kvh, block, t % a.cache.slots);
        const char4 k = reinterpret_cast<const char4*>(a.cache.k + at * kK8Hd)[lane], v = reinterpret_cast<const char4*>(a.cache.v + at * kK8Hd)[lane];
        const float dot = warp_sum(x[0] * k.x + x[1] * k.y + x[2] * k.z + x[3] * k.w) * a.cache.scale_k[at] * 0.08838834764831845f;
        const float now = fmaxf(m, dot), f = m == -INFINITY ? 0.0f : expf(m - now), p = expf(dot - now), w = p * a.cache.scale_v[at];
        m = now;
        l = l * f + p;
        o[0] = o[0] * f + w * v.x;
        o[1] = o[1] * f + w * v.y;
        o[2] = o[2] * f + w * v.z;
        o[3] = o[3] * f + w * v.w;
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    reinterpret_cast<float4*>(a.out + (row * a.n_q + head) * kK8Hd)[lane] = make_float4(o[0] * r, o[1] * r, o[2] * r, o[3] * r);
    if (lane == 0 && a.lse) a.lse[row * a.n_q + head] = l == 0.0f ? -INFINITY : m + logf(l);
}

// One warp a (sequence, kv head, key): all rows and heads in order.
__global__ void __launch_bounds__(kTrThreads) tree_weigh_kernel(const TreeLaunch L) {
    const tenzo_attention_tree_args& a = L.a;
    const int lane = threadIdx.x & 31, t = blockIdx.x * 4 + (threadIdx.x >> 5), kvh = blockIdx.y, s = blockIdx.z;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const int start = ld_l2(a.start + s), count = a.count ? ld_l2(a.count + s) : a.nodes, seq = a.seq ? ld_l2(a.seq + s) : s;
    if (start < 0 || count == 0) return;
    if (count < 0 || count > a.nodes || (long long)start + count > a.max_len || seq < 0 || seq >= a.cache.table_rows) {
        if (lane == 0) atomicOr(&g_tree_error, kK8ErrIndex);
        return;
    }
    if (t >= start + count) return;
    const int block = kv8_block(a.cache, seq, t);
    if (block < 0) {
        if (lane == 0) atomicOr(&g_tree_error, kK8ErrIndex);
        return;
    }
    const size_t at = kv8_row(a.cache, a.layer, kvh, block, t % a.cache.slots);
    const char4 k = reinterpret_cast<const char4*>(a.cache.k + at * kK8Hd)[lane];
    float w = 0.0f;
    for (int i = 0; i < count; ++i) {
        const size_t row = (size_t)s * a.nodes + i;
        const int pos = a.rope_pos ? ld_l2(a.rope_pos + row) : start + i;
        if (a.rope_cos && (pos < 0 || pos >= a.rope_len)) {
            if (lane == 0) atomicOr(&g_tree_error, kK8ErrIndex);
            continue;
        }
        if (!tree_sees(a, row, i, start, t)) continue;
        for (int g = 0; g < L.group; ++g) {
            const int head = kvh * L.group + g;
            const float lse = a.lse[row * a.n_q + head];
            if (!isfinite(lse)) continue;
            const float* q = a.q + row * a.q_stride + (size_t)head * kK8Hd;
            float x[4];
            for (int j = 0; j < 4; ++j) {
                const int d = 4 * lane + j;
                x[j] = q[d];
                if (a.rope_cos) {
                    const float c = a.rope_cos[(size_t)pos * 64 + (d & 63)], sn = a.rope_sin[(size_t)pos * 64 + (d & 63)];
                    x[j] = d < 64 ? __fmaf_rn(q[d], c, -(q[d + 64] * sn)) : __fmaf_rn(q[d - 64], sn, q[d] * c);
                }
            }
            w += expf(warp_sum(x[0] * k.x + x[1] * k.y + x[2] * k.z + x[3] * k.w) * a.cache.scale_k[at] * 0.08838834764831845f - lse);
        }
    }
    if (lane == 0) L.weight[at] += w;
}

int* kv8_rows_flags();
__global__ void kv8_clear_flags_kernel(int* rows, int rows_seen, int* tree, int tree_seen) {
    atomicAnd(rows, ~rows_seen);
    atomicAnd(tree, ~tree_seen);
}

// What both calls ask of their arguments; fills in what is left to the default.
static int tree_check(TreeLaunch& L) {
    tenzo_attention_tree_args& a = L.a;
    if (!kv8_cache_ok(a.cache) || !a.q || !a.start) return -1;
    if (a.layer < 0 || a.layer >= a.cache.n_layers || a.n_q <= 0 || a.n_q % a.cache.n_kv || a.sequences < 0 || a.nodes <= 0 || a.max_len <= 0) return -1;
    if (a.max_len > kv8_places(a.cache) || (!a.seq && a.sequences > a.cache.table_rows)) return -1;
    if ((a.rope_cos == nullptr) != (a.rope_sin == nullptr) || (a.rope_cos && a.rope_len <= 0)) return -1;
    if (a.nodes > TENZO_TREE_MOST) return -5;
    if (a.q_stride == 0) a.q_stride = a.n_q * kK8Hd;
    if (a.q_stride < (long long)a.n_q * kK8Hd) return -1;
    const int words = (a.nodes + 31) / 32;
    if (a.mask_stride == 0) a.mask_stride = words;
    if (a.mask_stride < words) return -1;
    L.group = a.n_q / a.cache.n_kv;
    return 0;
}

}  // namespace tz

extern "C" size_t tenzo_cuda_attention_tree_workspace_bytes(int sequences, int nodes, int n_q, int max_len) {
    if (sequences <= 0 || nodes <= 0 || n_q <= 0 || max_len <= 0) return 0;
    return (size_t)sequences * nodes * n_q * 520 * (((size_t)max_len + 127) / 128);
}

extern "C" int tenzo_cuda_attention_tree_splits(int sequences, int nodes, int n_q, int n_kv, int max_len) {
    if (sequences <= 0 || nodes <= 0 || nodes > TENZO_TREE_MOST || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_len <= 0) return 0;
    return 1;
}

extern "C" int tenzo_cuda_attention_tree(const tenzo_attention_tree_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    TreeLaunch L = {};
    L.a = *args;
    tenzo_attention_tree_args& a = L.a;
    if (a.sequences == 0) return 0;
    if (int rc = tree_check(L)) return rc;
    if (!a.out || !kv8_aligned(a.out, 16) || a.split_keys < 0) return -1;
    if (a.split_keys > 0) {
        const long long keys = ((long long)a.split_keys + 127) / 128 * 128, splits = (a.max_len + keys - 1) / keys;
        if (splits > 1 && (!a.workspace || !kv8_aligned(a.workspace, 16) || a.workspace_bytes / 520 / a.n_q / a.nodes / a.sequences < (size_t)splits)) return -1;
    }
    return kv4_launch(attention_tree_kernel, dim3((unsigned)(a.sequences * a.nodes), (unsigned)((a.n_q + 3) / 4)), kTrThreads, 0, static_cast<cudaStream_t>(stream), a.use_pdl != 0, L);
}

extern "C" int tenzo_cuda_kv8_weigh(const tenzo_attention_tree_args* args, float* weight, void* stream) {
    using namespace tz;
    if (!args) return -1;
    TreeLaunch L = {};
    L.a = *args;
    tenzo_attention_tree_args& a = L.a;
    if (a.sequences == 0) return 0;
    if (int rc = tree_check(L)) return rc;
    if (!weight || !a.lse) return -1;
    L.weight = weight;
    return kv4_launch(tree_weigh_kernel, dim3((unsigned)((a.max_len + 3) / 4), (unsigned)a.cache.n_kv, (unsigned)a.sequences), kTrThreads, 0, static_cast<cudaStream_t>(stream), a.use_pdl != 0, L);
}

// What runs on any stream is waited for, also on those that do not wait for the default one. Only bits that were seen are cleared: of what another thread's call raises
// meanwhile a bit is in the result or stays.
extern "C" int tenzo_cuda_kv8_take_errors(void) {
    using namespace tz;
    int *rows = kv8_rows_flags(), *tree = nullptr, r = 0, t = 0;
    if (!rows || cudaGetSymbolAddress(reinterpret_cast<void**>(&tree), g_tree_error) != cudaSuccess) return -1;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(&r, rows, sizeof r, cudaMemcpyDeviceToHost) != cudaSuccess ||
        cudaMemcpy(&t, tree, sizeof t, cudaMemcpyDeviceToHost) != cudaSuccess)
        return -1;
    if ((r | t) && (kv4_launch(kv8_clear_flags_kernel, dim3(1), 1, 0, cudaStreamLegacy, false, rows, r, tree, t) || cudaStreamSynchronize(cudaStreamLegacy) != cudaSuccess)) return -1;
    return r | t;
}
