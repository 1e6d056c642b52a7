// Attention of drafted trees over the INT8 caches (kv8.cuh), and the weight that each cached token receives.
//
//   * All query vectors of a kv head (nodes x heads of the group) read the same keys, so both products are matrix products with the keys, then the dims, as rows of 128 and
//     the queries as columns: S^T = K Q^T and O^T = V^T P^T. A CTA takes 16, 32 or 64 of the queries and walks its keys in tiles of 128. With keys as rows a single
//     query fills the tensor cores as well as many do, and one kernel serves a decode step and a tree of 64 nodes.
//   * Both are products of whole numbers (tcgen05 kind::i8, sums of 32 bits), and the codes of the cache are operands as they lie: K and V tiles go from memory to shared
//     memory to the tensor cores, nothing is unpacked or converted. A query is scaled to a maximum of 2^22 - 1 and rounded; its three signed bytes are three columns. A weight, p * scale of its
//     value, is rounded to a whole number of 31 bits; its four bytes, as they lie in the register, are four columns. So P is stored as it is computed, 16 bytes for four queries, and its
//     operand and V's are both read transposed (MN-major). Sums are exact: what rounds is the query (2^-23 of its largest number), the weights (2^-28 of a row's largest) and fp32 in between.
//   * softmax: a thread has one key and sixteen queries, so a row's maximum goes across lanes; and accumulators of whole numbers cannot be scaled down.
//     Both are avoided: a row's weights are taken relative to a reference, the maximum when it was last set, and may grow to 2^4 of it. Only where a weight would pass that (one vote a
//     tile; the first tile always) the references are set anew and the accumulators moved on into fp32.
#include "attn_common.cuh"
#include "kv8.cuh"
#include "umma.cuh"

namespace tz {

constexpr int kTrTile = 128, kTrTileBytes = kTrTile * kK8Hd;          // keys a step; bytes of their codes
constexpr int kTrMask = TENZO_TREE_MOST / 32;
constexpr float kTrSlack = 4.0f, kTrOne = 134217728.0f;               // a weight of 1 is 2^27, weights up to 2^4 are let through
constexpr float kTrLow = -1e30f;                                      // a reference that is not set
constexpr uint32_t kTrShape = (2u << 4) | (1u << 7) | ((uint32_t)(kTrTile >> 4) << 24);      // of products: sums of 32 bits; codes, with a sign, as A; 128 rows
constexpr int kTrFlush = 256;                                         // tiles after which the accumulators are moved on all the same: 2^15 keys * 128 * 255 < 2^31

__device__ int g_tree_error = 0;

struct TreeLaunch {
    tenzo_attention_tree_args a;
    int group, tiles, n_splits, split_keys;              // heads a kv head; CTAs for a tree's queries; splits of the keys
    float* part_o;                                       // [row][head][split][128]
    float2* part_ml;                                     // [row][head][split]: reference (log2), sum
    float* weight;
};

// R queries a CTA.
template <int R>
struct TreeShape {
    static constexpr int warps = R / 4, threads = (warps + 3) * 32;   // four warps for sixteen queries; one that copies, two that issue products
    static constexpr int stages = R == 64 ? 3 : 2, resident = R == 64 ? 1 : 2;
    static constexpr int s_cols = 3 * R, o_cols = 4 * R, tmem_cols = R == 64 ? 512 : R == 32 ? 256 : 128;
    static constexpr int p_panels = R == 64 ? 2 : 1;                  // of 128 bytes: 32 queries
    static constexpr int q_bytes = s_cols * kK8Hd, p_bytes = p_panels * kTrTileBytes;
    static constexpr size_t smem = 1024 + (size_t)stages * 2 * kTrTileBytes + q_bytes + p_bytes + stages * 2 * kTrTile * 4;
};

__device__ __forceinline__ float tr_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float tr_lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float tr_warp_max(float x) {               // (NaN has no part)
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tr_ld8(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at) : "memory");
}
// The wait for loads of tensor memory, tied to what they load: nothing that uses these moves in front of it.
__device__ __forceinline__ void tr_wait8(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
__device__ __forceinline__ void tr_tie8(uint32_t (&r)[8]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
// Whether any of `count` threads says so.
__device__ __forceinline__ bool tr_any(int barrier, int count, bool mine) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(barrier), "r"(count), "r"((uint32_t)mine) : "memory");
    return r != 0;
}
// Operand tiles that are contiguous along M or N (rows of 128 bytes, one for each k), 128-byte swizzle: eight k are 1024 bytes, `panel` bytes from one 128 to the next.
__device__ __forceinline__ uint64_t tr_desc_mn(uint32_t saddr, uint32_t panel) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ f32x2 tr_mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 tr_fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// The accumulators of the scores start at kTrBias, the bits of 2^23 * 1.5, so that a part of a sum (below 2^21 each) is read as the float 2^23 * 1.5 + part.
// Two sums from their three parts; the lower two parts' share is rounded to 2^7 of some 2^29.
constexpr uint32_t kTrBias = 0x4B400000u;
__device__ __forceinline__ f32x2 tr_whole2(const uint32_t* high, const uint32_t* mid, const uint32_t* low) {
    auto part = [](const uint32_t* v) { return pack2(__uint_as_float(v[0]), __uint_as_float(v[1])); };
    constexpr float base = 12582912.0f;
    return add2(tr_fma2(add2(part(high), pack2(-base, -base)), pack2(65536.0f, 65536.0f), tr_fma2(part(mid), pack2(256.0f, 256.0f), part(low))), pack2(-257.0f * base, -257.0f * base));
}
// The same value in N columns of the warp's 32 lanes.
template <int N>
__device__ __forceinline__ void tr_fill(uint32_t at, uint32_t v) {
    static_assert(N % 16 == 0, "sixteen columns a store");
#pragma unroll
    for (int i = 0; i < N; i += 16)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1};" ::"r"(at + i), "r"(v) : "memory");
}

// What a sequence's numbers allow.
struct TreeSequence {
    int start, count, seq;
    bool padding, refused;
    __device__ __forceinline__ TreeSequence(const tenzo_attention_tree_args& a, int s) {
        start = ld_l2(a.start + s);
        count = a.count ? ld_l2(a.count + s) : a.nodes;
        seq = a.seq ? ld_l2(a.seq + s) : s;
        padding = start < 0 || count == 0;
        refused = !padding && (count < 0 || count > a.nodes || (long long)start + count > a.max_len || seq < 0 || seq >= a.cache.table_rows);
    }
};
__device__ __forceinline__ bool tr_position_refused(const tenzo_attention_tree_args& a, int pos) { return a.rope_cos && (pos < 0 || pos >= a.rope_len); }

// ---- the parts that both kernels have ------------------------------------------------------------------------------------------
// Query `flat` = node * group + head of the group: rotated, rounded to whole numbers of 23 bits, its bytes as rows r, R + r, 2R + r of the operand (128 bytes each, swizzled). One
// warp; returns what a unit of the products with the codes counts in the argument of 2^x (NaN for a query that is not finite).
template <int R>
__device__ __forceinline__ float tr_query(const tenzo_attention_tree_args& a, size_t row, int head, int pos, unsigned char* s_q, int r) {
    const int lane = threadIdx.x & 31;
    const float* q = a.q + row * a.q_stride + (size_t)head * kK8Hd + lane;
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = ld_l2(q + 32 * j);             // dims lane + 32 j; pairs (0, 2) and (1, 3)
    if (a.rope_cos) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float c = ld_l2(a.rope_cos + (size_t)pos * 64 + 32 * j + lane), s = ld_l2(a.rope_sin + (size_t)pos * 64 + 32 * j + lane);
            rope_rotate(x[j], x[j + 2], true, c, s, x[j], x[j + 2]);
        }
    }
    const float most = fmaxf(tr_warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])))), 1e-25f);
    const bool bad = __any_sync(0xffffffffu, !(fabsf(x[0]) < INFINITY && fabsf(x[1]) < INFINITY && fabsf(x[2]) < INFINITY && fabsf(x[3]) < INFINITY));
    const float up = 4194303.0f / most;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int v = bad ? 0 : __float2int_rn(x[j] * up), d3 = ((v + 128) & 255) - 128, m = (v - d3) >> 8, d2 = ((m + 128) & 255) - 128, d1 = (m - d2) >> 8;
        const int d = lane + 32 * j, chunk = d >> 4;
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            const int n = part * R + r;
            s_q[n * kK8Hd + ((chunk ^ (n & 7)) << 4) + (d & 15)] = (unsigned char)(part == 0 ? d1 : part == 1 ? d2 : d3);
        }
    }
    return bad ? __uint_as_float(0x7fc00000u) : most * (1.0f / 4194303.0f) * (0.08838834764831845f * 1.4426950408889634f);
}

// The warp that copies: keys c_begin .. c_end - 1 tile by tile, sixteen keys a lane of eight. A block whose table entry is out of range is left out (its bit in s_valid is 0).
template <int STAGES, bool VALUES>
struct TreeCopies {
    const tenzo_attention_tree_args& a;
    const CUtensorMap *kmap, *vmap;
    int kvh, seq, c_begin, c_end;
    unsigned char* stages;                               // [STAGES][K, V]
    float* scales;                                       // [STAGES][K, V][128]
    uint64_t *full, *empty;
    unsigned* s_valid;
    static constexpr int kPer = VALUES ? 2 : 1;
    __device__ __forceinline__ int first_row(int u) const {           // of the chunk of sixteen keys that starts at 16 u; -1: none
        if (u * kK8Chunk >= c_end) return -1;
        const int per = a.cache.slots / kK8Chunk, column = u / per;
        const int id = ld_l2(a.cache.block_table + (size_t)seq * a.cache.table_stride + column);
        if (id < 0 || id >= a.cache.n_blocks) {
            atomicOr(&g_tree_error, kK8ErrIndex);
            return -1;
        }
        return (int)kv8_row(a.cache, a.layer, kvh, id, (u - column * per) * kK8Chunk);
    }
    __device__ __forceinline__ bool run(int n_tiles, int steps) const {
        const int lane = threadIdx.x & 31;
        bool ok = true;
        int done = 0;
        // of the tile four steps share a look-up: lane / 8 of them
        auto look = [&](int i) { return i + (lane >> 3) < steps ? first_row(c_begin / kK8Chunk + (i + (lane >> 3)) % n_tiles * (kTrTile / kK8Chunk) + (lane & 7)) : -1; };
        int now = look(0), next = look(4);
        for (int i = 0; i < steps && ok; ++i) {
            const int st = i % STAGES, use = i / STAGES;
            if (i > 0 && (i & 3) == 0) {
                now = next;
                next = look(i + 4);
            }
            if (use > 0) ok = mbar_wait_bounded(&empty[st], (unsigned)(use - 1) & 1u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const unsigned there = __ballot_sync(0xffffffffu, now >= 0) >> (8 * (i & 3)) & 0xffu;
            if (lane == 0) {
                s_valid[st] = there;
                mbar_expect_tx(&full[st], (unsigned)__popc(there) * kPer * (kK8Chunk * kK8Hd + kK8Chunk * 4));
            }
            __syncwarp();
            if ((lane >> 3) == (i & 3) && now >= 0) {
                unsigned char* to = stages + (size_t)st * kPer * kTrTileBytes + (lane & 7) * kK8Chunk * kK8Hd;
                float* sc = scales + (size_t)st * kPer * kTrTile + (lane & 7) * kK8Chunk;
                tma_load_2d(to, kmap, 0, now, &full[st]);
                bulk_g2s(sc, a.cache.scale_k + now, kK8Chunk * 4, &full[st]);
                if (VALUES) {
                    tma_load_2d(to + kTrTileBytes, vmap, 0, now, &full[st]);
                    bulk_g2s(sc + kTrTile, a.cache.scale_v + now, kK8Chunk * 4, &full[st]);
                }
            }
            __syncwarp();
            done = i + 1;
        }
        if (!ok)                                         // copies in flight land before the block ends
            for (int i = max(0, done - STAGES); i < done; ++i) mbar_wait_bounded(&full[i % STAGES], (unsigned)(i / STAGES) & 1u);
        return ok;
    }
};

// For sixteen queries (columns of each part), two by two, and the lane's key, whose scale is sk: arguments of 2^x less what `down` (with its sign turned) says. The
// accumulators are left as they have to start.
template <int R>
__device__ __forceinline__ void tr_arguments(uint32_t tmem, const float* s_f, const float* s_down, float sk, f32x2 (&w)[8]) {
    const f32x2 sk2 = pack2(sk, sk);
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
        uint32_t d1[8], d2[8], d3[8];
        tr_ld8(tmem + h, d1);
        tr_ld8(tmem + R + h, d2);
        tr_ld8(tmem + 2 * R + h, d3);
        tr_wait8(d1);
        tr_tie8(d2);
        tr_tie8(d3);
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(s_f + h + j), m = *reinterpret_cast<const ulonglong2*>(s_down + h + j);
            w[(h + j) / 2] = tr_fma2(tr_whole2(d1 + j, d2 + j, d3 + j), tr_mul2(sk2, f.x), m.x);
            w[(h + j) / 2 + 1] = tr_fma2(tr_whole2(d1 + j + 2, d2 + j + 2, d3 + j + 2), tr_mul2(sk2, f.y), m.y);
        }
    }
#pragma unroll
    for (int part = 0; part < 3; ++part) tr_fill<16>(tmem + part * R, kTrBias);
    tmem_wait_st();
}

// Queries that do not see the lane's key: node j of the tree (below 0: a cached token, which all see), or `dead`, none.
__device__ __forceinline__ void tr_hide(f32x2 (&w)[8], const uint32_t (*mask)[kTrMask], int j, bool dead) {
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
        float w0, w1;
        unpack2(w[r / 2], w0, w1);
        if (dead || (j >= 0 && !(mask[r][j >> 5] >> (j & 31) & 1u))) w0 = -INFINITY;
        if (dead || (j >= 0 && !(mask[r + 1][j >> 5] >> (j & 31) & 1u))) w1 = -INFINITY;
        w[r / 2] = pack2(w0, w1);
    }
}

// ---- attention -------------------------------------------------------------------------------------------------------------------
template <int R>
__global__ void __launch_bounds__(TreeShape<R>::threads, TreeShape<R>::resident)
attention_tree_kernel(const TreeLaunch L, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using S = TreeShape<R>;
    const tenzo_attention_tree_args& a = L.a;
    extern __shared__ unsigned char tr_smem[];
    __shared__ __align__(16) float s_f[R], s_down[R], s_max[4][R], s_sum[4][R], s_scale_max[R / 16][4];      // (s_down: the references with their signs turned)
    __shared__ long long s_at[R];                        // [row][head] of a query; -1: none of this tree's, or refused; -2 - that: padding, zeros
    __shared__ uint32_t s_mask[R][kTrMask];
    __shared__ uint64_t s_full[S::stages], s_empty[S::stages], s_bar[4];
    __shared__ unsigned s_valid[S::stages];
    __shared__ uint32_t s_tmem, s_set[R / 16];           // queries that have a reference
    __shared__ float s_unit[R / 16][2];                  // values' scales count up to this power of two; what a scale is multiplied by
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tile = blockIdx.x % L.tiles, split = (int)(blockIdx.x / L.tiles) % L.n_splits, s = blockIdx.x / L.tiles / L.n_splits, kvh = blockIdx.y;
    if (a.use_pdl || L.n_splits > 1) pdl_launch_dependents();         // (the second kernel waits for this one whatever its neighbours do)
    if (a.use_pdl) pdl_wait();
    const TreeSequence q(a, s);
    if (q.refused) {
        if (tid == 0) atomicOr(&g_tree_error, kK8ErrIndex);
        return;
    }
    const int flat0 = tile * R, queries = a.nodes * L.group;
    const int total = q.padding ? 0 : q.start + q.count, c_begin = split * L.split_keys, c_end = min(total, c_begin + L.split_keys);
    const bool nothing = q.padding || flat0 / L.group >= q.count;    // rows of padding alone
    if (nothing || c_begin >= c_end) {
        if (L.n_splits == 1)
            for (int i = tid; i < R * kK8Hd; i += S::threads) {
                const int flat = flat0 + i / kK8Hd;
                if (flat >= queries) break;
                const size_t at = ((size_t)s * a.nodes + flat / L.group) * a.n_q + (size_t)kvh * L.group + flat % L.group;
                a.out[at * kK8Hd + i % kK8Hd] = 0.0f;
                if (a.lse && i % kK8Hd == 0) a.lse[at] = -INFINITY;
            }
        return;
    }
    const int n_tiles = (c_end - c_begin + kTrTile - 1) / kTrTile;
    unsigned char* base = tr_smem + (((smem_addr(tr_smem) + 1023u) & ~1023u) - smem_addr(tr_smem));
    unsigned char *s_q = base + S::stages * 2 * kTrTileBytes, *s_p = s_q + S::q_bytes;
    float* s_scales = reinterpret_cast<float*>(s_p + S::p_bytes);
    uint64_t *b_scores = s_bar, *b_free = s_bar + 1, *b_weights = s_bar + 2, *b_values = s_bar + 3;   // scores are there; were read; weights are there; their products are done
    if (tid == 0) {
        for (int i = 0; i < S::stages; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 1);
        }
        mbar_init(b_scores, 2);                          // the products, and the thread that has seen the copies land
        mbar_init(b_free, S::warps);
        mbar_init(b_weights, S::warps);
        mbar_init(b_values, 1);
        mbar_init_fence();
        for (int g = 0; g < R / 16; ++g) {
            s_unit[g][0] = s_unit[g][1] = 0.0f;
            s_set[g] = 0;
        }
    }
    if (warp == S::warps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(S::tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    constexpr int kWithQueries = (S::warps + 1) * 32;
    bool ok = true;

    if (warp == S::warps) {
        const TreeCopies<S::stages, true> copies = {a, &kmap, &vmap, kvh, q.seq, c_begin, c_end, base, s_scales, s_full, s_empty, s_valid};
        ok = copies.run(n_tiles, n_tiles);
    } else if (warp == S::warps + 1) {
        named_barrier_sync(6, kWithQueries);             // the queries are there
        if (lane == 0) {                                 // S^T = K Q^T
            constexpr uint32_t shape = kTrShape | (1u << 10) | ((uint32_t)(S::s_cols >> 3) << 17);
            const uint64_t dq = umma_desc_sw128(smem_addr(s_q));
            for (int i = 0; i < n_tiles; ++i) {
                const int st = i % S::stages;
                ok = mbar_spin_bounded(&s_full[st], (unsigned)(i / S::stages) & 1u) && (i == 0 || mbar_spin_bounded(b_free, (unsigned)(i - 1) & 1u));
                if (!ok) break;
                tc_fence_after();
                const uint64_t dk = umma_desc_sw128(smem_addr(base + (size_t)st * 2 * kTrTileBytes));
#pragma unroll
                for (int k = 0; k < kK8Hd / 32; ++k) umma_i8(tmem, dk + (uint64_t)(2 * k), dq + (uint64_t)(2 * k), shape, 1u);
                umma_commit(b_scores);
                mbar_arrive(b_scores);
            }
        }
        __syncwarp();
    } else if (warp == S::warps + 2) {
        if (lane == 0) {                                 // O^T += V^T P^T
            constexpr uint32_t shape = kTrShape | (1u << 15) | (1u << 16) | ((uint32_t)(S::o_cols >> 3) << 17);        // both operands transposed
            const uint64_t dp = tr_desc_mn(smem_addr(s_p), kTrTileBytes);
            for (int i = 0; i < n_tiles; ++i) {
                const int st = i % S::stages;
                ok = mbar_spin_bounded(&s_full[st], (unsigned)(i / S::stages) & 1u) && mbar_spin_bounded(b_weights, (unsigned)i & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dv = tr_desc_mn(smem_addr(base + (size_t)st * 2 * kTrTileBytes + kTrTileBytes), kTrTileBytes);
#pragma unroll
                for (int k = 0; k < kTrTile / 32; ++k)
                    umma_i8(tmem + S::s_cols, dv + (uint64_t)(k * (32 * kK8Hd >> 4)), dp + (uint64_t)(k * (32 * kK8Hd >> 4)), shape, 1u);
                umma_commit(b_values);
                umma_commit(&s_empty[st]);
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, group = warp >> 2, first = group * 16;      // its keys of a tile, and its queries
        constexpr int kAll = S::warps * 32, kEvery = 7;              // threads, and their barrier (1 .. 4: those of sixteen queries)
        // ---- the queries ----
        for (int r = tid; r < R; r += kAll) {
            const int flat = flat0 + r, node = flat / L.group;
            const size_t row = (size_t)s * a.nodes + node;
            long long at = -1;
            if (flat < queries) {
                at = (long long)(row * a.n_q + (size_t)kvh * L.group + flat % L.group);
                if (node >= q.count) {
                    at = -2 - at;
                } else if (tr_position_refused(a, a.rope_pos ? ld_l2(a.rope_pos + row) : q.start + node)) {
                    atomicOr(&g_tree_error, kK8ErrIndex);
                    at = -1;
                }
            }
            s_at[r] = at;
            s_down[r] = 0.0f;
            for (int w = 0; w < (a.nodes + 31) / 32; ++w)
                s_mask[r][w] = at < 0 ? 0u : a.mask ? (uint32_t)ld_l2(a.mask + row * a.mask_stride + w) : node >= 32 * w + 31 ? 0xffffffffu : node < 32 * w ? 0u : (2u << (node - 32 * w)) - 1u;
        }
        named_barrier_sync(kEvery, kAll);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = warp + j * S::warps;
            float f = 0.0f;
            if (s_at[r] >= 0) {
                const int flat = flat0 + r, node = flat / L.group;
                const size_t row = (size_t)s * a.nodes + node;
                f = tr_query<R>(a, row, kvh * L.group + flat % L.group, a.rope_pos ? ld_l2(a.rope_pos + row) : q.start + node, s_q, r);
            } else {
                for (int part = 0; part < 3; ++part) reinterpret_cast<uint32_t*>(s_q + (part * R + r) * kK8Hd)[lane] = 0;
            }
            if (lane == 0) s_f[r] = f;
        }
        const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16), t_scores = t_lane + (uint32_t)first, t_values = t_lane + (uint32_t)(S::s_cols + 4 * first);
        tr_fill<64>(t_values, 0u);
#pragma unroll
        for (int part = 0; part < 3; ++part) tr_fill<16>(t_scores + part * R, kTrBias);
        tmem_wait_st();
        tc_fence_before();
        fence_proxy_async_smem();
        named_barrier_sync(6, kWithQueries);
        const int key = 32 * quarter + lane;
        float o[16];                                     // of dim `key`: outputs that were moved on
        f32x2 l[8];                                      // of key `key`: sums
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; ++r) l[r] = 0;
        // Adds the accumulators to o.
        auto move_on = [&](float unit) {
#pragma unroll
            for (int h = 0; h < 16; h += 2) {
                uint32_t v[8];
                tr_ld8(t_values + 4 * h, v);
                tr_wait8(v);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float hi = __fmaf_rn((float)(int)v[4 * j + 3], 256.0f, (float)(int)v[4 * j + 2]), lo = __fmaf_rn((float)(int)v[4 * j + 1], 256.0f, (float)(int)v[4 * j]);
                    o[h + j] = __fmaf_rn(__fmaf_rn(hi, 65536.0f, lo), unit, o[h + j]);
                }
            }
        };
        for (int i = 0; i < n_tiles; ++i) {
            const int st = i % S::stages, t = c_begin + i * kTrTile + key;
            ok = ok && mbar_wait_bounded(b_scores, (unsigned)i & 1u);
            __syncwarp();
            const unsigned valid = s_valid[st];
            const bool ragged = c_begin + (i + 1) * kTrTile > min(c_end, q.start) || valid != 0xffu;
            const bool dead = ragged && (t >= c_end || !(valid >> (key >> 4) & 1u));
            float sv = dead ? 0.0f : s_scales[(2 * st + 1) * kTrTile + key], sk = dead ? 0.0f : s_scales[2 * st * kTrTile + key];
            if (!(sv < INFINITY)) {                      // the value of a key that is no number: it spoils the rows that see it by way of their sums
                sv = 0.0f;
                sk = __uint_as_float(0x7fc00000u);
            }
            tc_fence_after();
            f32x2 w[8];
            tr_arguments<R>(t_scores, s_f + first, s_down + first, sk, w);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_free);
            if (ragged) tr_hide(w, s_mask + first, t - q.start, dead);
            float over = -INFINITY;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float w0, w1;
                unpack2(w[r], w0, w1);
                over = fmaxf(fmaxf(over, w0), w1);
            }
            const uint32_t set = s_set[group];
            const bool anew = tr_any(1 + group, 128, over > kTrSlack || sv > s_unit[group][0] || set != 0xffffu || (i + 1) % kTrFlush == 0);
            if (anew) {
                // ---- references of these sixteen queries anew, and their accumulators moved on ----
                const float unit = s_unit[group][0];
                float top = -INFINITY;                   // lane r: of query `first` + r, less the reference
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    float w0, w1;
                    unpack2(w[r / 2], w0, w1);
                    w0 = tr_warp_max(w0);
                    w1 = tr_warp_max(w1);
                    if (lane == r) top = w0;
                    if (lane == r + 1) top = w1;
                }
                if (lane < 16) s_max[quarter][first + lane] = top;
                const float most = tr_warp_max(sv);
                if (lane == 0) s_scale_max[group][quarter] = most;
                if (i > 0) {
                    ok = ok && mbar_wait_bounded(b_values, (unsigned)(i - 1) & 1u);
                    __syncwarp();
                    tc_fence_after();
                    move_on(unit * (1.0f / kTrOne));
                    tr_fill<64>(t_values, 0u);
                    tmem_wait_st();
                    tc_fence_before();
                }
                named_barrier_sync(1 + group, 128);
                const float4 scales = *reinterpret_cast<const float4*>(s_scale_max[group]);
                const float scale_most = fmaxf(fmaxf(scales.x, scales.y), fmaxf(scales.z, scales.w));
                float up, by;                            // of query `first` + lane % 16: how far its reference goes up (the first one may go down), and what that leaves of its sums
                {
                    const int r = lane & 15;
                    const bool was = set >> r & 1u;
                    top = fmaxf(fmaxf(s_max[0][first + r], s_max[1][first + r]), fmaxf(s_max[2][first + r], s_max[3][first + r]));
                    up = was ? fmaxf(top, 0.0f) : top == -INFINITY ? 0.0f : top;
                    by = was ? tr_ex2(-up) : 0.0f;       // (there is nothing yet)
                }
                const uint32_t now_set = set | (__ballot_sync(0xffffffffu, top != -INFINITY) & 0xffffu);
                if (quarter == 0) {
                    if (lane < 16) s_down[first + lane] -= up;
                    if (lane == 0) {
                        // a power of two above the largest scale, at least 2^-60
                        const float now = scale_most > unit ? __uint_as_float(min(max((__float_as_uint(scale_most) >> 23) + 1u, 67u), 254u) << 23) : unit;
                        s_unit[group][0] = now;
                        s_unit[group][1] = now > 0.0f ? kTrOne / now : 0.0f;
                        s_set[group] = now_set;
                    }
                }
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float u0 = __shfl_sync(0xffffffffu, up, r), u1 = __shfl_sync(0xffffffffu, up, r + 1);
                    const float b0 = __shfl_sync(0xffffffffu, by, r), b1 = __shfl_sync(0xffffffffu, by, r + 1);
                    o[r] *= b0;
                    o[r + 1] *= b1;
                    l[r / 2] = tr_mul2(l[r / 2], pack2(b0, b1));
                    w[r / 2] = add2(w[r / 2], pack2(-u0, -u1));
                }
                named_barrier_sync(1 + group, 128);
            }
            const float by = sv * s_unit[group][1];
            const f32x2 by2 = pack2(by, by);
            uint32_t word[16];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float p0, p1;
                unpack2(w[r], p0, p1);
                const f32x2 p = pack2(tr_ex2(p0), tr_ex2(p1));
                l[r] = add2(l[r], p);
                unpack2(tr_mul2(p, by2), p0, p1);
                word[2 * r] = __float2uint_rn(p0);
                word[2 * r + 1] = __float2uint_rn(p1);
            }
            if (i > 0 && !anew) ok = ok && mbar_wait_bounded(b_values, (unsigned)(i - 1) & 1u);        // (the weights in front were read)
            __syncwarp();
            unsigned char* to = s_p + (first >> 5) * kTrTileBytes + key * kK8Hd;
            const int chunk = (first & 31) >> 2;
#pragma unroll
            for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(to + (((chunk + c) ^ (key & 7)) << 4)) = make_uint4(word[4 * c], word[4 * c + 1], word[4 * c + 2], word[4 * c + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_weights);
        }
        // ---- the outputs ----
        ok = ok && mbar_wait_bounded(b_values, (unsigned)(n_tiles - 1) & 1u);
        __syncwarp();
        tc_fence_after();
        move_on(s_unit[group][0] * (1.0f / kTrOne));
        tc_fence_before();
        float mine = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            float l0, l1;
            unpack2(l[r / 2], l0, l1);
            l0 = warp_sum(l0);
            l1 = warp_sum(l1);
            if (lane == r) mine = l0;
            if (lane == r + 1) mine = l1;
        }
        if (lane < 16) s_sum[quarter][first + lane] = mine;
        named_barrier_sync(1 + group, 128);
        const uint32_t set = s_set[group];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const long long at = s_at[first + r];
            const float sum = (s_sum[0][first + r] + s_sum[1][first + r]) + (s_sum[2][first + r] + s_sum[3][first + r]);
            if (L.n_splits > 1) {
                if (at >= 0) {
                    L.part_o[((size_t)at * L.n_splits + split) * kK8Hd + key] = o[r];
                    if (key == 0) L.part_ml[(size_t)at * L.n_splits + split] = make_float2(set >> r & 1u ? -s_down[first + r] : kTrLow, sum);
                }
            } else if (at != -1) {
                const size_t to = (size_t)(at >= 0 ? at : -2 - at);
                const bool none = at < 0 || sum == 0.0f;
                a.out[to * kK8Hd + key] = none ? 0.0f : o[r] / sum;
                if (a.lse && key == 0) a.lse[to] = none ? -INFINITY : (tr_lg2(sum) - s_down[first + r]) * 0.6931471805599453f;
            }
        }
    }
    if (!ok) atomicOr(&g_tree_error, kK8ErrWait);
    tc_fence_before();
    __syncthreads();
    if (warp == S::warps) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::tmem_cols) : "memory");
    }
}

// The splits of a (row, head): one warp each, four dims a lane.
constexpr int kTrMergeWarps = 4;
__global__ void __launch_bounds__(kTrMergeWarps * 32) attention_tree_merge_kernel(const TreeLaunch L) {
    const tenzo_attention_tree_args& a = L.a;
    const int lane = threadIdx.x & 31, head = blockIdx.y * kTrMergeWarps + (threadIdx.x >> 5);
    const size_t row = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    if (head >= a.n_q) return;
    const int s = (int)(row / a.nodes), node = (int)(row % a.nodes);
    const TreeSequence q(a, s);
    if (q.refused) return;
    const bool padding = q.padding || node >= q.count;
    if (!padding && tr_position_refused(a, a.rope_pos ? ld_l2(a.rope_pos + row) : q.start + node)) return;
    const int n = padding ? 0 : (q.start + q.count + L.split_keys - 1) / L.split_keys;
    const size_t at = (row * a.n_q + head) * L.n_splits;
    const float2* ml = L.part_ml + at;
    const float4* po = reinterpret_cast<const float4*>(L.part_o) + at * (kK8Hd / 4) + lane;
    float m = -INFINITY;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, ld_l2(ml + i).x);
    m = warp_max(m);
    const float use = m == -INFINITY ? 0.0f : m;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    constexpr int kBatch = 8;                            // loads in flight
    for (int i0 = 0; i0 < n; i0 += kBatch) {
        float2 v[kBatch];
        float4 p[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            v[u] = i0 + u < n ? ld_l2(ml + i0 + u) : make_float2(kTrLow, 0.0f);
            p[u] = i0 + u < n ? ld_l2(po + (size_t)(i0 + u) * (kK8Hd / 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const float x = tr_ex2(v[u].x - use);
            o.x = __fmaf_rn(p[u].x, x, o.x);
            o.y = __fmaf_rn(p[u].y, x, o.y);
            o.z = __fmaf_rn(p[u].z, x, o.z);
            o.w = __fmaf_rn(p[u].w, x, o.w);
            l = __fmaf_rn(v[u].y, x, l);
        }
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;         // (a query with a NaN has a NaN here)
    reinterpret_cast<float4*>(a.out + (row * a.n_q + head) * kK8Hd)[lane] = make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
    if (lane == 0 && a.lse) a.lse[row * a.n_q + head] = l == 0.0f ? -INFINITY : (use + tr_lg2(l)) * 0.6931471805599453f;
}

// ---- the weight that keys receive -------------------------------------------------------------------------------------------------
// The same scores, for up to kTwTiles tiles of keys a CTA and all queries of the kv head, R at a time (a pass): a thread has one key, so its sum over sixteen queries needs no other
// lane, and the sums lie in shared memory, each thread's own, until all passes are done. No key has two CTAs: one order of summation, no atomics.
constexpr int kTwTiles = 8;

template <int R>
struct WeighShape {
    static constexpr int groups = R / 16, warps = R / 4, threads = (warps + 2) * 32, stages = 4, resident = R == 64 ? 1 : 2;
    static constexpr int s_cols = 3 * R, tmem_cols = R == 64 ? 512 : R == 32 ? 256 : 128;        // two sets of scores
    static constexpr int q_bytes = s_cols * kK8Hd;
    static constexpr size_t smem = 1024 + (size_t)stages * kTrTileBytes + q_bytes + stages * kTrTile * 4 + groups * kTwTiles * kTrTile * 4;
};

template <int R>
__global__ void __launch_bounds__(WeighShape<R>::threads, WeighShape<R>::resident) tree_weigh_kernel(const TreeLaunch L, const __grid_constant__ CUtensorMap kmap) {
    using S = WeighShape<R>;
    const tenzo_attention_tree_args& a = L.a;
    extern __shared__ unsigned char tr_smem[];
    __shared__ __align__(16) float s_f[R], s_down[R];    // (the log-sum-exp with its sign turned)
    __shared__ uint32_t s_mask[R][kTrMask];
    __shared__ uint64_t s_full[S::stages], s_empty[S::stages], s_scores[2], s_free[2], s_query;
    __shared__ unsigned s_valid[S::stages];
    __shared__ uint32_t s_tmem;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int split = (int)blockIdx.x % L.n_splits, s = (int)blockIdx.x / L.n_splits, kvh = blockIdx.y;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const TreeSequence q(a, s);
    if (q.refused) {
        if (tid == 0) atomicOr(&g_tree_error, kK8ErrIndex);
        return;
    }
    if (q.padding) return;
    const int total = q.start + q.count, c_begin = split * L.split_keys, c_end = min(total, c_begin + L.split_keys);
    if (c_begin >= c_end) return;
    const int n_tiles = (c_end - c_begin + kTrTile - 1) / kTrTile, queries = q.count * L.group, passes = (queries + R - 1) / R, steps = n_tiles * passes;
    unsigned char* base = tr_smem + (((smem_addr(tr_smem) + 1023u) & ~1023u) - smem_addr(tr_smem));
    unsigned char* s_q = base + S::stages * kTrTileBytes;
    float *s_scales = reinterpret_cast<float*>(s_q + S::q_bytes), *s_sum = s_scales + S::stages * kTrTile;
    if (tid == 0) {
        for (int i = 0; i < S::stages; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], S::warps + 1);        // the products, and the warps that read the scales
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_scores[i], 2);                  // the products, and the thread that has seen the copies land
            mbar_init(&s_free[i], S::warps);
        }
        mbar_init(&s_query, S::warps);
        mbar_init_fence();
    }
    if (warp == S::warps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(S::tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    bool ok = true;

    if (warp == S::warps) {
        const TreeCopies<S::stages, false> copies = {a, &kmap, nullptr, kvh, q.seq, c_begin, c_end, base, s_scales, s_full, s_empty, s_valid};
        ok = copies.run(n_tiles, steps);
    } else if (warp == S::warps + 1) {
        if (lane == 0) {
            constexpr uint32_t d_scores = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(S::s_cols >> 3) << 17) | ((uint32_t)(kTrTile >> 4) << 24);
            const uint64_t dq = umma_desc_sw128(smem_addr(s_q));
            for (int n = 0; n < steps && ok; ++n) {
                const int st = n % S::stages, half = n & 1;
                if (n % n_tiles == 0) ok = mbar_spin_bounded(&s_query, (unsigned)(n / n_tiles) & 1u);
                ok = ok && mbar_spin_bounded(&s_full[st], (unsigned)(n / S::stages) & 1u) && (n < 2 || mbar_spin_bounded(&s_free[half], (unsigned)(n / 2 - 1) & 1u));
                if (!ok) break;
                tc_fence_after();
                const uint64_t dk = umma_desc_sw128(smem_addr(base + (size_t)st * kTrTileBytes));
#pragma unroll
                for (int k = 0; k < kK8Hd / 32; ++k) umma_i8(tmem + half * S::s_cols, dk + (uint64_t)(2 * k), dq + (uint64_t)(2 * k), d_scores, 1u);
                umma_commit(&s_scores[half]);
                mbar_arrive(&s_scores[half]);
                umma_commit(&s_empty[st]);
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, first = (warp >> 2) * 16, key = 32 * quarter + lane;
        constexpr int kAll = S::warps * 32;
        const uint32_t t_scores = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)first;
        float* sums = s_sum + (warp >> 2) * kTwTiles * kTrTile + key;
#pragma unroll
        for (int part = 0; part < 6; ++part) tr_fill<16>(t_scores + part * R, kTrBias);
        tmem_wait_st();
        tc_fence_before();
        for (int n = 0; n < steps; ++n) {
            const int i = n % n_tiles, pass = n / n_tiles, st = n % S::stages, half = n & 1;
            if (i == 0) {                                // the next queries; the products with the ones in front are done
                named_barrier_sync(1, kAll);
                for (int r = tid; r < R; r += kAll) {
                    const int flat = pass * R + r, node = flat / L.group;
                    const size_t row = (size_t)s * a.nodes + node;
                    float lse = INFINITY;                // of a query that does not count
                    if (flat < queries) {
                        if (tr_position_refused(a, a.rope_pos ? ld_l2(a.rope_pos + row) : q.start + node)) {
                            atomicOr(&g_tree_error, kK8ErrIndex);
                        } else {
                            lse = ld_l2(a.lse + row * a.n_q + (size_t)kvh * L.group + flat % L.group) * 1.4426950408889634f;
                            if (!(fabsf(lse) < INFINITY)) lse = INFINITY;
                        }
                    }
                    s_down[r] = -lse;
                    for (int w = 0; w < (a.nodes + 31) / 32; ++w)
                        s_mask[r][w] = flat >= queries ? 0u : a.mask ? (uint32_t)ld_l2(a.mask + row * a.mask_stride + w) : node >= 32 * w + 31 ? 0xffffffffu : node < 32 * w ? 0u : (2u << (node - 32 * w)) - 1u;
                }
                named_barrier_sync(1, kAll);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = warp + j * S::warps, flat = pass * R + r, node = flat / L.group;
                    const size_t row = (size_t)s * a.nodes + node;
                    float f = 0.0f;
                    if (s_down[r] > -INFINITY) {
                        f = tr_query<R>(a, row, kvh * L.group + flat % L.group, a.rope_pos ? ld_l2(a.rope_pos + row) : q.start + node, s_q, r);
                    } else {
                        for (int part = 0; part < 3; ++part) reinterpret_cast<uint32_t*>(s_q + (part * R + r) * kK8Hd)[lane] = 0;
                    }
                    if (lane == 0) s_f[r] = f;
                }
                fence_proxy_async_smem();
                named_barrier_sync(1, kAll);
                if (lane == 0) mbar_arrive(&s_query);
            }
            ok = ok && mbar_wait_bounded(&s_scores[half], (unsigned)(n / 2) & 1u);
            __syncwarp();
            const int t = c_begin + i * kTrTile + key;
            const unsigned valid = s_valid[st];
            const bool ragged = c_begin + (i + 1) * kTrTile > min(c_end, q.start) || valid != 0xffu, dead = ragged && (t >= c_end || !(valid >> (key >> 4) & 1u));
            float sk = dead ? 0.0f : s_scales[st * kTrTile + key];
            if (!(fabsf(sk) < INFINITY)) sk = 0.0f;      // (no query that sees it has a finite lse)
            tc_fence_after();
            f32x2 w[8];
            tr_arguments<R>(t_scores + half * S::s_cols, s_f + first, s_down + first, sk, w);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_free[half]);
                mbar_arrive(&s_empty[st]);
            }
            if (ragged) tr_hide(w, s_mask + first, t - q.start, dead);
            f32x2 sum2 = 0;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float w0, w1;
                unpack2(w[r], w0, w1);
                sum2 = add2(sum2, pack2(tr_ex2(w0), tr_ex2(w1)));
            }
            float sum, other;
            unpack2(sum2, sum, other);
            sum += other;
            sums[i * kTrTile] = pass == 0 ? sum : sums[i * kTrTile] + sum;
        }
        named_barrier_sync(1, kAll);
        for (int k = tid; k < c_end - c_begin; k += kAll) {
            const int t = c_begin + k, id = kv8_block(a.cache, q.seq, t);
            if (id < 0) continue;
            float sum = 0.0f;
#pragma unroll
            for (int g = 0; g < S::groups; ++g) sum += s_sum[g * kTwTiles * kTrTile + k];
            float* w = L.weight + kv8_row(a.cache, a.layer, kvh, id, t % a.cache.slots);
            *w = ld_l2(w) + sum;
        }
    }
    if (!ok) atomicOr(&g_tree_error, kK8ErrWait);
    tc_fence_before();
    __syncthreads();
    if (warp == S::warps) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::tmem_cols) : "memory");
    }
}

// ---- the calls ---------------------------------------------------------------------------------------------------------------------
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
    if (a.nodes > TENZO_TREE_MOST || a.n_q > 1 << 20 || a.cache.n_kv > 65535 || a.max_len > 1 << 30) return -5;
    if (a.q_stride == 0) a.q_stride = a.n_q * kK8Hd;
    if (a.q_stride < a.n_q * kK8Hd) return -1;
    const int words = (a.nodes + 31) / 32;
    if (a.mask_stride == 0) a.mask_stride = words;
    if (a.mask_stride < words) return -1;
    L.group = a.n_q / a.cache.n_kv;
    return 0;
}

static int tree_map(CUtensorMap* map, const tenzo_kv8_cache& c, const int8_t* codes) {
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, kK8Hd, (uint64_t)c.n_blocks * c.n_layers * c.n_kv * c.slots, kK8Hd, kK8Hd, kK8Chunk, CU_TENSOR_MAP_SWIZZLE_128B);
}

static int tree_queries_a_cta(long long queries) { return queries <= 16 ? 16 : queries <= 32 ? 32 : 64; }

// Keys a CTA takes: the number of splits whose rounds of CTAs take least at the longest length, a CTA's own cost counted as some hundred keys.
static void tree_pick_split(TreeLaunch& L, int resident, long long most) {
    const tenzo_attention_tree_args& a = L.a;
    const long long items = (long long)a.sequences * a.cache.n_kv * L.tiles, places = 148 * resident;
    double best = 0.0;
    for (int want = 1; want <= most; ++want) {
        const int keys = ((a.max_len + want - 1) / want + kTrTile - 1) / kTrTile * kTrTile, splits = (a.max_len + keys - 1) / keys;
        if (splits > most) continue;
        const long long ctas = items * splits;
        const double rounds = ctas <= 3 * places ? (double)((ctas + places - 1) / places) : (double)ctas / places + 0.5;
        const double cost = rounds * (keys + 500.0) + (splits > 1 ? 400.0 + 16.0 * (splits - 1) : 0.0);
        if (want == 1 || cost < best) {
            best = cost;
            L.split_keys = keys;
            L.n_splits = splits;
        }
        if (keys == kTrTile) break;
    }
}
constexpr int kTrMostSplits = 64;

static void tree_plan(TreeLaunch& L, long long room) {
    const tenzo_attention_tree_args& a = L.a;
    const long long queries = (long long)a.nodes * L.group;
    const int r = tree_queries_a_cta(queries);
    L.tiles = (int)((queries + r - 1) / r);
    if (a.split_keys > 0) {
        const long long keys = ((long long)a.split_keys + kTrTile - 1) / kTrTile * kTrTile, all = ((long long)a.max_len + kTrTile - 1) / kTrTile * kTrTile;
        L.split_keys = (int)(keys < all ? keys : all);
        L.n_splits = (a.max_len + L.split_keys - 1) / L.split_keys;
        return;
    }
    tree_pick_split(L, r == 64 ? 1 : 2, room < 1 ? 1 : room < kTrMostSplits ? room : kTrMostSplits);
}

template <int R>
static int tree_run(const TreeLaunch& L, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t st) {
    if (cudaError_t e = allow_smem(attention_tree_kernel<R>, TreeShape<R>::smem)) return (int)e;
    const dim3 grid((unsigned)((long long)L.a.sequences * L.n_splits * L.tiles), (unsigned)L.a.cache.n_kv);
    return kv4_launch(attention_tree_kernel<R>, grid, TreeShape<R>::threads, TreeShape<R>::smem, st, L.a.use_pdl != 0, L, kmap, vmap);
}
template <int R>
static int weigh_run(const TreeLaunch& L, const CUtensorMap& kmap, cudaStream_t st) {
    if (cudaError_t e = allow_smem(tree_weigh_kernel<R>, WeighShape<R>::smem)) return (int)e;
    const dim3 grid((unsigned)((long long)L.a.sequences * L.n_splits), (unsigned)L.a.cache.n_kv);
    return kv4_launch(tree_weigh_kernel<R>, grid, WeighShape<R>::threads, WeighShape<R>::smem, st, L.a.use_pdl != 0, L, kmap);
}
static size_t tree_part_bytes(const tenzo_attention_tree_args& a) { return (size_t)a.sequences * a.nodes * a.n_q * (kK8Hd + 2) * sizeof(float); }

}  // namespace tz

extern "C" size_t tenzo_cuda_attention_tree_workspace_bytes(int sequences, int nodes, int n_q, int max_len) {
    if (sequences <= 0 || nodes <= 0 || n_q <= 0 || max_len <= 0) return 0;
    return (size_t)sequences * nodes * n_q * 520 * (((size_t)max_len + 127) / 128);     // the finest split that may be asked for
}

extern "C" int tenzo_cuda_attention_tree_splits(int sequences, int nodes, int n_q, int n_kv, int max_len) {
    using namespace tz;
    if (sequences <= 0 || nodes <= 0 || nodes > TENZO_TREE_MOST || n_q <= 0 || n_kv <= 0 || n_q % n_kv || n_q > 1 << 20 || n_kv > 65535 || max_len <= 0 || max_len > 1 << 30) return 0;
    TreeLaunch L = {};
    L.a.sequences = sequences; L.a.nodes = nodes; L.a.n_q = n_q; L.a.cache.n_kv = n_kv; L.a.max_len = max_len;
    L.group = n_q / n_kv;
    tree_plan(L, kTrMostSplits);
    return L.n_splits;
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
    const bool ws_ok = a.workspace && kv8_aligned(a.workspace, 16);
    const long long room = ws_ok ? (long long)(a.workspace_bytes / tree_part_bytes(a)) : 0;
    tree_plan(L, room);
    if (L.n_splits > 1 && room < L.n_splits) return -1;
    if ((long long)a.sequences * L.n_splits * L.tiles > 0x7fffffffLL || (long long)a.sequences * a.nodes > 0x7fffffffLL) return -5;
    L.part_o = static_cast<float*>(a.workspace);
    L.part_ml = reinterpret_cast<float2*>(L.part_o + (size_t)a.sequences * a.nodes * a.n_q * L.n_splits * kK8Hd);
    CUtensorMap kmap, vmap;
    if (int rc = tree_map(&kmap, a.cache, a.cache.k)) return rc;
    if (int rc = tree_map(&vmap, a.cache, a.cache.v)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int r = tree_queries_a_cta((long long)a.nodes * L.group);
    if (int rc = r == 16 ? tree_run<16>(L, kmap, vmap, st) : r == 32 ? tree_run<32>(L, kmap, vmap, st) : tree_run<64>(L, kmap, vmap, st)) return rc;
    if (L.n_splits == 1) return 0;
    return kv4_launch(attention_tree_merge_kernel, dim3((unsigned)(a.sequences * a.nodes), (unsigned)((a.n_q + kTrMergeWarps - 1) / kTrMergeWarps)), kTrMergeWarps * 32, 0, st, true, L);
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
    const int r = tree_queries_a_cta((long long)a.nodes * L.group);
    // Keys a CTA takes: as few as give every SM some CTAs, at most what it has sums for.
    const long long heads = (long long)a.sequences * a.cache.n_kv, want = (148LL * (r == 64 ? 2 : 4) + heads - 1) / heads;
    long long keys = ((a.max_len + want - 1) / want + kTrTile - 1) / kTrTile * kTrTile;
    L.split_keys = (int)(keys < kTwTiles * kTrTile ? keys : kTwTiles * kTrTile);
    L.n_splits = (a.max_len + L.split_keys - 1) / L.split_keys;
    if ((long long)a.sequences * L.n_splits > 0x7fffffffLL) return -5;
    CUtensorMap kmap;
    if (int rc = tree_map(&kmap, a.cache, a.cache.k)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return r == 16 ? weigh_run<16>(L, kmap, st) : r == 32 ? weigh_run<32>(L, kmap, st) : weigh_run<64>(L, kmap, st);
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
