// Rows of the INT8 caches (kv8.cuh): storing them at places of their own, the accepted nodes of drafted trees, and the eviction of the tokens that received
// least attention.
#include "attn_common.cuh"
#include "kv8.cuh"

namespace tz {

__device__ int g_kv8_rows_error = 0;
int* kv8_rows_flags() {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, g_kv8_rows_error) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

// ---- append ----------------------------------------------------------------------------------------------------------------
// A warp takes HB kv heads of one row: lanes 0-15 the keys, 16-31 the values, dims 4l .. 4l + 3 and 64 more a lane, so that the pairs that the rotation turns lie in one lane. Bound
// by the bytes (5 of 6 read) in long calls and by the chain of loads (place, table, row) in short ones. Four heads a warp where there are warps enough: what names the row, its place in the
// table and the rotation's coefficients are asked for once, and four times the bytes are on their way meanwhile (calls back to back in a graph; 8000 rows of 8 heads: 18.5 us by fours, 26.2 by ones; of 4 heads 10.3 and 13.9;
// 1600 rows of 8: 6.1 and 7.2; 1024: 5.3 and 5.2; 512 rows of 5 heads: 4.2 and 3.5; 9000 rows of 2 heads: 9.3 and 9.0).
constexpr int kK8RowWarps = 4;
constexpr long long kK8Many = 148 * 64;                  // (row, head) pairs from which on a warp takes four heads: as many warps as the machine holds

template <bool VEC>
__device__ __forceinline__ void k8_load4(const float* p, float* x) {
    if (VEC) {
        const float4 v = ld_l2(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = ld_l2(p + j);
    }
}

template <bool VEC, int HB>
__global__ void __launch_bounds__(kK8RowWarps * 32) kv8_append_kernel(const tenzo_kv8_append_args a) {
    const int lane = threadIdx.x & 31, is_v = lane >> 4, l = lane & 15, blocks = (a.cache.n_kv + HB - 1) / HB;
    const long long unit = (long long)blockIdx.x * kK8RowWarps + (threadIdx.x >> 5), row = unit / blocks;
    const int head0 = (int)(unit % blocks) * HB;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    if (row >= a.rows) return;
    const int place = ld_l2(a.place + row), seq = a.seq ? ld_l2(a.seq + row) : (int)row, pos = a.rope_pos ? ld_l2(a.rope_pos + row) : place;
    float x[HB][8];
    const float* p = (is_v ? a.v : a.k) + (size_t)row * a.kv_stride + 4 * l;
#pragma unroll
    for (int h = 0; h < HB; ++h) {                       // (the last block's missing heads read its first one again)
        const int head = HB == 1 || head0 + h < a.cache.n_kv ? head0 + h : head0;
        k8_load4<VEC>(p + head * kK8Hd, x[h]);
        k8_load4<VEC>(p + head * kK8Hd + 64, x[h] + 4);
    }
    if (place < 0) return;
    const bool there = seq >= 0 && seq < a.cache.table_rows && place / a.cache.slots < a.cache.table_stride && (!a.rope_cos || (pos >= 0 && pos < a.rope_len));
    const int id = there ? ld_l2(a.cache.block_table + (size_t)seq * a.cache.table_stride + place / a.cache.slots) : -1;
    float c[4] = {1, 1, 1, 1}, s[4] = {0, 0, 0, 0};
    if (a.rope_cos && there) {
        k8_load4<true>(a.rope_cos + (size_t)pos * 64 + 4 * l, c);
        k8_load4<true>(a.rope_sin + (size_t)pos * 64 + 4 * l, s);
    }
    if (id < 0 || id >= a.cache.n_blocks) {
        if (lane == 0) atomicOr(&g_kv8_rows_error, kK8ErrIndex);
        return;
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        if (a.rope_cos && !is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) rope_rotate(x[h][j], x[h][4 + j], true, c[j], s[j], x[h][j], x[h][4 + j]);
        }
        float amax = 1e-8f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[h][j]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float scale = amax * (1.0f / 127.0f), inv = 1.0f / scale;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float q = fminf(fmaxf(roundf(x[h][j] * inv), -128.0f), 127.0f);
            w[j >> 2] |= ((uint32_t)(int)q & 255u) << (8 * (j & 3));
        }
        if (HB > 1 && head0 + h >= a.cache.n_kv) break;      // (the whole warp)
        const size_t at = kv8_row(a.cache, a.layer, head0 + h, id, place % a.cache.slots);
        uint32_t* to = reinterpret_cast<uint32_t*>((is_v ? a.cache.v : a.cache.k) + at * kK8Hd);
        to[l] = w[0];
        to[16 + l] = w[1];
        if (l == 0) (is_v ? a.cache.scale_v : a.cache.scale_k)[at] = scale;
        if (lane == 1 && a.weight) a.weight[at] = 0.0f;
        if (lane == 2 && a.position) a.position[at] = pos;
    }
}

// ---- moving rows: half a warp takes one row, sixteen bytes a lane, keys and values; four lanes take what is beside them ------------------------
struct K8Row {
    uint4 code;
    uint32_t beside;
};
// What lane `which` of a row's sixteen moves beside its codes, and whether it does; those that do not read the keys' scale, for nothing.
__device__ __forceinline__ uint32_t* k8_beside(const tenzo_kv8_cache& c, float* weight, int* position, int which) {
    return which == 0 ? reinterpret_cast<uint32_t*>(c.scale_k) : which == 1 ? reinterpret_cast<uint32_t*>(c.scale_v) : which == 2 ? reinterpret_cast<uint32_t*>(weight)
         : which == 3 ? reinterpret_cast<uint32_t*>(position) : nullptr;
}
__device__ __forceinline__ void k8_take(const tenzo_kv8_cache& c, const uint32_t* beside, size_t row, int l, K8Row& r) {
    r.code = ld_l2(reinterpret_cast<const uint4*>((l & 8 ? c.v : c.k) + row * kK8Hd) + (l & 7));
    r.beside = ld_l2((beside ? beside : reinterpret_cast<const uint32_t*>(c.scale_k)) + row);
}
__device__ __forceinline__ void k8_put(const tenzo_kv8_cache& c, uint32_t* beside, size_t row, int l, const K8Row& r) {
    reinterpret_cast<uint4*>((l & 8 ? c.v : c.k) + row * kK8Hd)[l & 7] = r.code;
    if (beside) beside[row] = r.beside;
}

// ---- accepted nodes ------------------------------------------------------------------------------------------------------------
// A CTA a sequence and some of its (layer, kv head) pairs; each finds the path for itself, a chain of the tree's numbers, its walk (one thread) and the table's entries that bounds small calls (24
// nodes, 150 pairs: 4.9 us on the device). As many CTAs as eight an SM: 64 sequences of 32 nodes, 30 layers of 5 heads 12.2 us, 3.2 of which are the moved rows' bytes.
constexpr int kAcThreads = 256, kAcHalves = kAcThreads / 16, kAcBatch = 4;     // rows in flight a half warp

__global__ void __launch_bounds__(kAcThreads) kv8_accept_kernel(const tenzo_kv8_accept_args a, const int many) {
    __shared__ int s_next[TENZO_TREE_MOST], s_token[TENZO_TREE_MOST], s_chosen[TENZO_TREE_MOST], s_path[TENZO_TREE_MOST + 1];
    __shared__ int2 s_at[TENZO_TREE_MOST][2];            // (block, slot) of a row's old place and of its new one
    __shared__ int s_n;
    const int tid = threadIdx.x, s = blockIdx.y;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const int start = ld_l2(a.start + s), count = a.count ? ld_l2(a.count + s) : a.nodes, seq = a.seq ? ld_l2(a.seq + s) : s;
    const bool padding = start < 0 || count == 0;
    const bool refused = !padding && (count < 0 || count > a.nodes || seq < 0 || seq >= a.cache.table_rows || (long long)start + count > min((long long)a.cache.table_stride * a.cache.slots, 0x7fffffffLL));
    if (refused && tid == 0) atomicOr(&g_kv8_rows_error, kK8ErrIndex);
    const int n = padding || refused ? 0 : count;
    int parent = -1;
    if (tid < n) {
        s_token[tid] = ld_l2(a.token + (size_t)s * a.nodes + tid);
        s_chosen[tid] = ld_l2(a.chosen + (size_t)s * a.nodes + tid);
        parent = ld_l2(a.parent + (size_t)s * a.nodes + tid);
        s_next[tid] = 0x7fffffff;
    }
    __syncthreads();
    if (tid < n && parent >= 0 && parent < tid && s_token[tid] == s_chosen[parent]) atomicMin(&s_next[parent], tid);     // the first that fits
    __syncthreads();
    if (tid == 0) {
        int m = 0;
        for (int i = 0; m < n && i < n; i = s_next[i]) s_path[m++] = i;       // (indices grow: it ends)
        s_n = m;
    }
    __syncthreads();
    const int m = s_n;
    if (blockIdx.x == 0) {
        for (int i = tid; i < a.nodes; i += kAcThreads) a.path[(size_t)s * a.nodes + i] = i < m ? s_path[i] : -1;
        if (tid == 0) {
            a.accepted[s] = m;
            a.next[s] = m ? s_chosen[s_path[m - 1]] : -1;
        }
    }
    int first = 0;                                       // rows in front of it are in their places
    if (tid < m) {
        const int from = start + s_path[tid], to = start + tid;
        int2 x = make_int2(-1, 0), y = x;
        if (from != to) {
            x = make_int2(kv8_block(a.cache, seq, from), from % a.cache.slots);
            y = make_int2(kv8_block(a.cache, seq, to), to % a.cache.slots);
            if ((x.x < 0 || y.x < 0) && blockIdx.x == 0) atomicOr(&g_kv8_rows_error, kK8ErrIndex);
        }
        s_at[tid][0] = x;
        s_at[tid][1] = y;
    }
    first = __syncthreads_count(tid < m && s_path[tid] == tid);
    const int rows = m - first;
    if (rows == 0) return;
    // Row d goes from a node's place to one that is not behind it, and no later row comes from a place in front of its own number: rows are taken in their order,
    // kAcHalves * kAcBatch at a time, and all of those are loaded before the first is stored.
    const int unit0 = blockIdx.x * many, units = min(many, a.cache.n_layers * a.cache.n_kv - unit0), half = tid >> 4, l = tid & 15;
    uint32_t* beside = k8_beside(a.cache, a.weight, a.position, l);
    for (int e0 = 0; e0 < units * rows; e0 += kAcHalves * kAcBatch) {
        K8Row r[kAcBatch];
        size_t to[kAcBatch];
        bool moves[kAcBatch];
#pragma unroll
        for (int b = 0; b < kAcBatch; ++b) {             // (something is read, where there is none, and not stored)
            const int e = min(e0 + b * kAcHalves + half, units * rows - 1), unit = unit0 + e / rows, d = first + e % rows, layer = unit / a.cache.n_kv, kvh = unit % a.cache.n_kv;
            const int2 x = s_at[d][0], y = s_at[d][1];
            moves[b] = e0 + b * kAcHalves + half < units * rows && x.x >= 0 && y.x >= 0;
            k8_take(a.cache, beside, kv8_row(a.cache, layer, kvh, max(x.x, 0), x.y), l, r[b]);
            to[b] = kv8_row(a.cache, layer, kvh, max(y.x, 0), y.y);
        }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < kAcBatch; ++b)
            if (moves[b]) k8_put(a.cache, beside, to[b], l, r[b]);
    }
}

// ---- eviction -------------------------------------------------------------------------------------------------------------------
// One CTA a (sequence, layer, kv head). The weights become whole numbers of the same order (the protected tokens' the largest) in shared memory; the `keep`-th largest is found by
// counting, two bits a round, and only those in the range that is left once these are few; what stays is a bit a token; and the free places and the tokens that move into them are two lists, the i-th goes to the i-th.
// Nothing that moves comes from a place that another moves to (those are below `keep`, these are not), so all rows move at once.
// Bound by the chain of loads, counts and barriers where CTAs are few (150 heads of 2176 tokens: 22 us with the moves, a single call with its launch, nothing in L2; 5.6 where nothing moves, in a graph), by the
// rows' scattered pieces (128 bytes of codes twice, four of four) where they are many: 64 x 20 heads of 4224 tokens 57 us, 30 without moves, 10.4 at the memory's rate.
// T threads a CTA, 1024 / T CTAs an SM: 256, or 128 where there are more CTAs than that leaves room for at once and shared memory has room for eight an SM (64 x 20 heads of 4224 tokens: 34.5 us of
// selection by 256, 29.7 by 128; 150 heads of 2176: 5.6 and 6.7; 512 threads, cold and with the moves: 100 and 30.7 us, where 256 take 63 and 22.5). Four loads in flight of numbers and of rows
// (cold, with the moves: two of numbers 61 and 23.4, eight 72 and 26.6; two of rows 70 and 24.6, eight 71 and 24.6).
constexpr int kEvBatch = 4, kEvLoads = 4;
constexpr int kEvHeld = 48 * 1024;                       // tokens whose numbers fit in shared memory
constexpr int kEvMost = 1 << 20, kEvLists = 16 * 1024;   // tokens at most, and entries of both lists together where the numbers do not fit

// A number whose order is the weight's: NaN as -infinity, -0 as +0.
__device__ __forceinline__ uint32_t ev_number(float w) {
    w = w == w ? w + 0.0f : -INFINITY;
    const uint32_t u = __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// HELD: the numbers are kept in shared memory; otherwise they are read again each time, and the lists are made a part at a time.
template <bool HELD, int T>
__global__ void __launch_bounds__(T, 1024 / T) kv8_evict_kernel(const tenzo_kv8_evict_args a) {
    constexpr int kThreads = T, kWarps = T / 32;
    extern __shared__ __align__(16) uint32_t ev_smem[];
    __shared__ __align__(16) uint32_t s_count[2][kWarps][4];                     // (read four at a time)
    __shared__ int s_warp[3][kWarps], s_listed;
    __shared__ uint32_t s_list[2 * kThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.y, layer = blockIdx.x / a.cache.n_kv, kvh = blockIdx.x % a.cache.n_kv;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const int n = ld_l2(a.length + s), seq = a.seq ? ld_l2(a.seq + s) : s;
    const bool refused = n < 0 || n > a.max_len || seq < 0 || seq >= a.cache.table_rows;
    if (refused || n <= a.keep) {
        if (tid == 0 && blockIdx.x == 0) a.length_out[s] = n;
        if (tid == 0 && refused) atomicOr(&g_kv8_rows_error, kK8ErrIndex);
        return;
    }
    const int from = a.protect_from ? ld_l2(a.protect_from + s) : 0;
    const int words = (n + 31) / 32, chunks = (words + kWarps - 1) / kWarps;       // of the bits; a warp's share of them
    uint32_t* s_keep = ev_smem;                          // [words]: what stays
    uint32_t* s_num = ev_smem + ((a.max_len + 31) / 32 + 3) / 4 * 4;          // [n to 4], HELD only; later the two lists
    // Numbers of four tokens from 4 g on, and of so many from 4 (g + step) .., 0 behind the last; four tokens lie in one block and are one load. All loads of one kind are in front of the first
    // that is waited for, and of something where there is nothing (where two ways meet the compiler copies what was loaded, and so waits for it).
    bool bad = false;
    auto load = [&](int g, int step, uint32_t (&num)[kEvLoads][4]) {
        size_t row[kEvLoads];
        int id[kEvLoads];
        uint4 w[kEvLoads], pos[kEvLoads];
#pragma unroll
        for (int u = 0; u < kEvLoads; ++u) id[u] = ld_l2(a.cache.block_table + (size_t)seq * a.cache.table_stride + min(4 * (g + u * step), n - 1) / a.cache.slots);
#pragma unroll
        for (int u = 0; u < kEvLoads; ++u) {
            const bool there = id[u] >= 0 && id[u] < a.cache.n_blocks;
            bad |= !there;
            row[u] = kv8_row(a.cache, layer, kvh, there ? id[u] : 0, min(4 * (g + u * step), (n - 1) & ~3) % a.cache.slots);
            w[u] = ld_l2(reinterpret_cast<const uint4*>(a.weight + row[u]));
        }
#pragma unroll
        for (int u = 0; u < kEvLoads; ++u) pos[u] = ld_l2(reinterpret_cast<const uint4*>(a.position + row[u]));
#pragma unroll
        for (int u = 0; u < kEvLoads; ++u) {
            const uint32_t wx[4] = {w[u].x, w[u].y, w[u].z, w[u].w}, px[4] = {pos[u].x, pos[u].y, pos[u].z, pos[u].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                num[u][j] = 4 * (g + u * step) + j >= n ? 0u : ev_number(a.protect_from && (int)px[j] >= from ? INFINITY : __uint_as_float(wx[j]));
        }
    };
    uint32_t lo = 0xffffffffu, hi = 0;
    for (int g0 = 0; 4 * g0 < n; g0 += kEvLoads * kThreads) {
        uint32_t num[kEvLoads][4];
        load(g0 + tid, kThreads, num);
#pragma unroll
        for (int u = 0; u < kEvLoads; ++u) {
            const int g = g0 + u * kThreads + tid;
            if (4 * g >= n) break;
            if (HELD) *reinterpret_cast<uint4*>(s_num + 4 * g) = make_uint4(num[u][0], num[u][1], num[u][2], num[u][3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo = num[u][j] ? min(lo, num[u][j]) : lo;
                hi = max(hi, num[u][j]);
            }
        }
    }
    bad = __syncthreads_or(bad);
    if (tid == 0 && blockIdx.x == 0) a.length_out[s] = bad ? n : a.keep;
    if (bad) {
        if (tid == 0) atomicOr(&g_kv8_rows_error, kK8ErrIndex);
        return;
    }
    // The largest number that `keep` tokens reach: bits from the top, those that all numbers share first.
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
        s_count[0][warp][0] = lo;
        s_count[0][warp][1] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        lo = min(lo, s_count[0][w][0]);
        hi = max(hi, s_count[0][w][1]);
    }
    int bits = 32 - __clz((int)(lo ^ hi));               // (0: all are equal)
    bits += bits & 1;
    uint32_t border = bits >= 32 ? 0u : lo >> bits << bits;
    int above = 0, reach = n;                            // tokens over the border's present range, and those that are not below it
    int round = 1, base = -1;                            // once few are in the range (150 heads of 2176 tokens 5.7 us, all counted to the end 8.6): the tokens over it then,
    uint32_t mine0 = 0, mine1 = 0;                       // and the thread's two of those
    while (bits > 0) {
        if (base < 0 && reach - above <= 2 * kThreads) {
            if (tid == 0) s_listed = 0;
            __syncthreads();
            auto list = [&](uint32_t u) {
                if (u >= border && (bits >= 32 || u - border < 1u << bits) && u != 0) s_list[atomicAdd(&s_listed, 1)] = u;      // (in any order: they are only counted)
            };
            if (HELD) {
                for (int g = tid; 4 * g < n; g += kThreads) {
                    const uint4 v = *reinterpret_cast<const uint4*>(s_num + 4 * g);
                    list(v.x);
                    list(v.y);
                    list(v.z);
                    list(v.w);
                }
            } else {
                for (int g0 = 0; 4 * g0 < n; g0 += kEvLoads * kThreads) {
                    uint32_t num[kEvLoads][4];
                    load(g0 + tid, kThreads, num);
#pragma unroll
                    for (int u = 0; u < kEvLoads; ++u)
#pragma unroll
                        for (int j = 0; j < 4; ++j) list(num[u][j]);
                }
            }
            __syncthreads();
            base = above;
            mine0 = tid < s_listed ? s_list[tid] : 0u;
            mine1 = tid + kThreads < s_listed ? s_list[tid + kThreads] : 0u;
        }
        bits -= 2;
        const uint32_t t1 = border + (1u << bits), t2 = border + (2u << bits), t3 = border + (3u << bits);
        int c1 = 0, c2 = 0, c3 = 0;                      // (border > 0 or a token's number is: ev_number is never 0)
        auto count = [&](uint32_t u) {
            c1 += u >= t1;
            c2 += u >= t2;
            c3 += u >= t3;
        };
        if (base >= 0) {
            count(mine0);
            count(mine1);
        } else if (HELD) {
            for (int g = tid; 4 * g < n; g += kThreads) {
                const uint4 v = *reinterpret_cast<const uint4*>(s_num + 4 * g);
                count(v.x);
                count(v.y);
                count(v.z);
                count(v.w);
            }
        } else {
            for (int g0 = 0; 4 * g0 < n; g0 += kEvLoads * kThreads) {
                uint32_t num[kEvLoads][4];
                load(g0 + tid, kThreads, num);
#pragma unroll
                for (int u = 0; u < kEvLoads; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) count(num[u][j]);
            }
        }
        c1 = __reduce_add_sync(0xffffffffu, c1);
        c2 = __reduce_add_sync(0xffffffffu, c2);
        c3 = __reduce_add_sync(0xffffffffu, c3);
        uint32_t(*sc)[4] = s_count[round & 1];
        if (lane == 0) {
            sc[warp][0] = c1;
            sc[warp][1] = c2;
            sc[warp][2] = c3;
        }
        __syncthreads();
        c1 = c2 = c3 = max(base, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint4 v = *reinterpret_cast<const uint4*>(sc[w]);
            c1 += v.x;
            c2 += v.y;
            c3 += v.z;
        }
        if (c3 >= a.keep) border = t3, reach = c3;
        else if (c2 >= a.keep) border = t2, reach = c2, above = c3;
        else if (c1 >= a.keep) border = t1, reach = c1, above = c2;
        else above = c1;
        ++round;
    }
    // `above` are over the border; of those that equal it the first `keep - above` stay too. (With all bits found, `above` is right: it was counted in the last round
    // that had some over the border's range; before that none were.)
    const int equal = a.keep - above;
    const int w0 = warp * chunks, w1 = min(words, w0 + chunks);
    // Number of a word's token `lane` (0 behind the last). Not held, the four tokens of the lane's eighth are loaded, and the eight lanes that have the word's take turns.
    auto number = [&](int w) -> uint32_t {
        if (HELD) return 32 * w + lane < n ? s_num[32 * w + lane] : 0u;
        uint32_t num[kEvLoads][4], r = 0;
        load(8 * w + (lane & 7), 0, num);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t v = __shfl_sync(0xffffffffu, num[0][j], lane >> 2);
            if ((lane & 3) == j) r = v;
        }
        return r;
    };
    int mine = 0;                                        // equal ones in the warp's share
    for (int w = w0; w < w1; ++w) mine += __popc(__ballot_sync(0xffffffffu, number(w) == border));
    if (lane == 0) s_warp[0][warp] = mine;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < warp; ++w) before += s_warp[0][w];
    int holes = 0, far = 0;
    for (int w = w0; w < w1; ++w) {
        const int t = 32 * w + lane;
        const uint32_t u = number(w);
        const unsigned same = __ballot_sync(0xffffffffu, u == border);
        const bool stays = u > border || (u == border && before + __popc(same & ((1u << lane) - 1)) < equal);
        before += __popc(same);
        const unsigned keep = __ballot_sync(0xffffffffu, stays);
        holes += __popc(__ballot_sync(0xffffffffu, t < a.keep && !stays));
        far += __popc(__ballot_sync(0xffffffffu, t >= a.keep && stays));
        if (lane == 0) s_keep[w] = keep;
    }
    if (lane == 0) {
        s_warp[1][warp] = holes;
        s_warp[2][warp] = far;
    }
    __syncthreads();                                     // the numbers are no longer needed
    int hole_at = 0, far_at = 0, moves = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) {
            hole_at += s_warp[1][w];
            far_at += s_warp[2][w];
        }
        moves += s_warp[1][w];
    }
    const int half = tid >> 4, l = tid & 15;
    uint32_t* beside = k8_beside(a.cache, a.weight, a.position, l);
    const int room = HELD ? moves : kEvLists / 2;         // entries of a list
    uint32_t *s_hole = s_num, *s_far = s_num + room;
    for (int part = 0; part < moves; part += room) {
        int h = hole_at, f = far_at;
        for (int w = w0; w < w1; ++w) {
            const int t = 32 * w + lane;
            const bool stays = t < n && (s_keep[w] >> lane & 1);
            const unsigned hm = __ballot_sync(0xffffffffu, t < a.keep && !stays), fm = __ballot_sync(0xffffffffu, t >= a.keep && stays), below = (1u << lane) - 1;
            const int hi_ = h + __popc(hm & below) - part, fi = f + __popc(fm & below) - part;
            if ((hm >> lane & 1) && hi_ >= 0 && hi_ < room) s_hole[hi_] = t;
            if ((fm >> lane & 1) && fi >= 0 && fi < room) s_far[fi] = t;
            h += __popc(hm);
            f += __popc(fm);
        }
        __syncthreads();
        const int these = min(room, moves - part);
        for (int i0 = half; i0 < these; i0 += kThreads / 16 * kEvBatch) {
            K8Row r[kEvBatch];
            int id[kEvBatch][2], t[kEvBatch][2];
#pragma unroll
            for (int b = 0; b < kEvBatch; ++b) {         // (the last row again, where there is none)
                const int i = min(i0 + b * (kThreads / 16), these - 1);
                t[b][0] = s_far[i];
                t[b][1] = s_hole[i];
#pragma unroll
                for (int e = 0; e < 2; ++e) id[b][e] = ld_l2(a.cache.block_table + (size_t)seq * a.cache.table_stride + t[b][e] / a.cache.slots);
            }
#pragma unroll
            for (int b = 0; b < kEvBatch; ++b) k8_take(a.cache, beside, kv8_row(a.cache, layer, kvh, id[b][0], t[b][0] % a.cache.slots), l, r[b]);
#pragma unroll
            for (int b = 0; b < kEvBatch; ++b)
                if (i0 + b * (kThreads / 16) < these) k8_put(a.cache, beside, kv8_row(a.cache, layer, kvh, id[b][1], t[b][1] % a.cache.slots), l, r[b]);
        }
        __syncthreads();
    }
}

// ---- the calls ------------------------------------------------------------------------------------------------------------------
// Results that lie in what is read, anywhere in it, would be written under the eyes of CTAs that come later: such calls are refused.
struct K8Range {
    const void* at;
    size_t bytes;
};
template <int W, int N>
static bool k8_apart(const K8Range (&written)[W], const K8Range (&read)[N], const tenzo_kv8_cache& c) {
    const size_t rows = kv8_rows(c);
    const K8Range pools[4] = {{c.k, rows * kK8Hd}, {c.v, rows * kK8Hd}, {c.scale_k, rows * sizeof(float)}, {c.scale_v, rows * sizeof(float)}};
    for (int i = 0; i < W; ++i) {
        for (int j = 0; j < i; ++j)
            if (kv8_overlap(written[i].at, written[i].bytes, written[j].at, written[j].bytes)) return false;
        for (const K8Range& r : read)
            if (kv8_overlap(written[i].at, written[i].bytes, r.at, r.bytes)) return false;
        for (const K8Range& r : pools)
            if (kv8_overlap(written[i].at, written[i].bytes, r.at, r.bytes)) return false;
    }
    return true;
}

}  // namespace tz

extern "C" int tenzo_cuda_kv8_append(const tenzo_kv8_append_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    const tenzo_kv8_append_args& a = *args;
    if (!kv8_cache_ok(a.cache) || a.layer < 0 || a.layer >= a.cache.n_layers || a.rows < 0) return -1;
    if (a.rows == 0) return 0;
    if (!a.k || !a.v || !a.place || a.kv_stride < (long long)a.cache.n_kv * kK8Hd || (!a.seq && a.rows > a.cache.table_rows)) return -1;
    if ((a.rope_cos == nullptr) != (a.rope_sin == nullptr) || (a.rope_cos && (a.rope_len <= 0 || !kv8_aligned(a.rope_cos, 16) || !kv8_aligned(a.rope_sin, 16)))) return -1;
    const int hb = a.cache.n_kv > 2 && (long long)a.rows * a.cache.n_kv > kK8Many ? 4 : 1;
    const long long ctas = ((long long)a.rows * ((a.cache.n_kv + hb - 1) / hb) + kK8RowWarps - 1) / kK8RowWarps;
    if (ctas > 0x7fffffffLL) return -5;
    // Vectors of four where all rows allow it: 8000 rows of 8 heads 18.5 us, by single numbers 22.6.
    const bool vec = kv8_aligned(a.k, 16) && kv8_aligned(a.v, 16) && a.kv_stride % 4 == 0;
    auto kernel = hb == 4 ? (vec ? kv8_append_kernel<true, 4> : kv8_append_kernel<false, 4>) : (vec ? kv8_append_kernel<true, 1> : kv8_append_kernel<false, 1>);
    return kv4_launch(kernel, dim3((unsigned)ctas), kK8RowWarps * 32, 0, static_cast<cudaStream_t>(stream), a.use_pdl != 0, a);
}

extern "C" int tenzo_cuda_kv8_accept(const tenzo_kv8_accept_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    const tenzo_kv8_accept_args& a = *args;
    if (!kv8_cache_ok(a.cache) || a.sequences < 0) return -1;
    if (a.sequences == 0) return 0;
    if (!a.token || !a.parent || !a.chosen || !a.start || !a.accepted || !a.next || !a.path || a.nodes <= 0 || (!a.seq && a.sequences > a.cache.table_rows)) return -1;
    if (a.nodes > TENZO_TREE_MOST || a.sequences > 65535) return -5;
    {                                                                // results apart from each other, and from what other CTAs of the sequence still read
        const size_t one = (size_t)a.sequences * sizeof(int), all = one * a.nodes, beside = kv8_rows(a.cache) * sizeof(int);
        const K8Range written[3] = {{a.accepted, one}, {a.next, one}, {a.path, all}};
        const K8Range read[9] = {{a.token, all}, {a.parent, all}, {a.chosen, all}, {a.start, one}, {a.count, one}, {a.seq, one}, {a.cache.block_table, kv8_table_bytes(a.cache)}, {a.weight, beside}, {a.position, beside}};
        if (!k8_apart(written, read, a.cache)) return -1;
    }
    const long long units = (long long)a.cache.n_layers * a.cache.n_kv, share = (units * a.sequences + 148 * 8 - 1) / (148 * 8);
    const int many = (int)(share < units ? share : units);           // (layer, kv head) pairs a CTA takes
    if ((long long)many * a.nodes > 1 << 30) return -5;
    return kv4_launch(kv8_accept_kernel, dim3((unsigned)((units + many - 1) / many), (unsigned)a.sequences), kAcThreads, 0, static_cast<cudaStream_t>(stream), a.use_pdl != 0, a, many);
}

extern "C" int tenzo_cuda_kv8_evict(const tenzo_kv8_evict_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    const tenzo_kv8_evict_args& a = *args;
    if (!kv8_cache_ok(a.cache) || a.sequences < 0) return -1;
    if (a.sequences == 0) return 0;
    if (!a.weight || !a.position || !kv8_aligned(a.weight, 16) || !kv8_aligned(a.position, 16) || !a.length || !a.length_out) return -1;
    if (a.keep <= 0 || a.max_len <= 0 || a.max_len > kv8_places(a.cache) || (!a.seq && a.sequences > a.cache.table_rows)) return -1;
    if (a.sequences > 65535 || a.max_len > kEvMost) return -5;
    {                                                                // apart from what other CTAs still read
        const size_t one = (size_t)a.sequences * sizeof(int), beside = kv8_rows(a.cache) * sizeof(int);
        const K8Range written[1] = {{a.length_out, one}};
        const K8Range read[6] = {{a.length, one}, {a.seq, one}, {a.protect_from, one}, {a.cache.block_table, kv8_table_bytes(a.cache)}, {a.weight, beside}, {a.position, beside}};
        if (!k8_apart(written, read, a.cache)) return -1;
    }
    const bool held = a.max_len <= kEvHeld;
    const size_t smem = (((size_t)(a.max_len + 31) / 32 + 3) / 4 * 4 + (size_t)(held ? (a.max_len + 3) / 4 * 4 : kEvLists)) * 4;
    constexpr size_t most = (kEvHeld / 32 + kEvHeld) * 4;
    static_assert(most >= (kEvMost / 32 + kEvLists) * 4, "the larger of the two");
    static_assert(most <= kMaxSmem - 4096, "bits of the longest and numbers of the longest that are held");
    const long long ctas = (long long)a.cache.n_layers * a.cache.n_kv;
    if (ctas > 0x7fffffffLL) return -5;
    const bool many = ctas * a.sequences > 148 * 4 && 8 * (smem + 4096) <= kMaxSmem;
    auto kernel = many ? kv8_evict_kernel<true, 128> : held ? kv8_evict_kernel<true, 256> : kv8_evict_kernel<false, 256>;
    if (smem > 40 * 1024)
        if (cudaError_t e = allow_smem(kernel, most)) return (int)e;
    return kv4_launch(kernel, dim3((unsigned)ctas, (unsigned)a.sequences), many ? 128 : 256, smem, static_cast<cudaStream_t>(stream), a.use_pdl != 0, a);
}
