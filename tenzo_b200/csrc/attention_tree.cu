// Attention of drafted trees over the INT8 caches (kv8.cuh), and the weight that each cached token receives.
//
//   * All query vectors of a kv head (nodes x heads of the group) read the same keys, so both products are matrix products with the keys, then the dims, as rows of 128 and
//     the queries as columns: S^T = K Q^T and O^T = V^T P^T. A CTA takes 16, 32, 48 or 64 of the queries and walks its keys in tiles of 128. With keys as rows a single
//     query fills the tensor cores as well as many do, and one kernel serves a decode step and a tree of 64 nodes.
//   * Both are products of whole numbers (tcgen05 kind::i8, sums of 32 bits), and the codes of the cache are operands as they lie: K and V tiles go from memory to shared
//     memory to the tensor cores, nothing is unpacked or converted. A query is scaled to a maximum of 2^29 to 2^30 and rounded; its four signed bytes are four columns. A weight, p * scale of its
//     value, is rounded to a whole number of 31 bits; its four bytes, as they lie in the register, are four columns. So P is stored as it is computed, 16 bytes for four queries, and its
//     operand and V's are both read transposed (MN-major). Sums are exact: what rounds is the query (2^-30 of its largest number; with three bytes, 2^-22, a query with one large dim lost its others, and 16 trees of 64 nodes took 231 us instead of 235), the products of weight and scale (2^-27 of a row's largest) and fp32 in between.
//   * softmax: a thread has one key and sixteen queries, so a row's maximum goes across lanes; and accumulators of whole numbers cannot be scaled down.
//     Both are avoided: a row's weights are taken relative to a reference, set so that the largest product of weight and scale is 1, and these products may grow to 2^5. Only where one would pass
//     that (one vote a tile; the first tile always) the references are set anew and the accumulators moved on into fp32. The reference goes by the product, which a thread has as a sum with its scale's
//     logarithm, and by the row's own keys: neither a key of most weight and small values, as a first token often is, nor one of large values that others see leaves a row fewer bits.
//   * Bound (times of calls back to back in a graph): single tokens by the bytes (64 sequences of 8192 keys, 20 heads over 5: 120 us, 106 at the memory's measured rate), trees by the instructions of the
//     warps that make weights, some 470 for 32 keys and sixteen queries with all that lies around them (16 trees of 64 nodes, 8192 keys: 235 us, 66 % of the issue slots; tensor cores 36 %, memory 11 %);
//     small calls by the chain share, queries, tile, outputs, join (8 nodes, 1000 keys: 12.7 us). Going on to the next pair takes some 9000 cycles, half of them 64 queries'.
//     With queries of three bytes, 227 us then: the same 64 queries as one line of 64, whose products wait for all warps, 282, plain fp32 instead of packed pairs 248.
#include "attn_common.cuh"
#include "kv8.cuh"
#include "umma.cuh"
#include "weigh_sums.cuh"

namespace tz {

constexpr int kTrTile = 128, kTrTileBytes = kTrTile * kK8Hd;          // keys a step; bytes of their codes
constexpr int kTrMask = TENZO_TREE_MOST / 32;
constexpr int kTrOne = 26;                                            // a row's largest product of weight and scale is 2^26
constexpr float kTrSlack = 5.0f;                                      // when it was looked for; up to 2^5 of that is let through
constexpr float kTrScales = 60.0f;                                    // a scale below 2^-60 of the others is taken as that where references are set
constexpr float kTrLow = -1e30f;                                      // a reference that is not set
constexpr uint32_t kTrShape = (2u << 4) | (1u << 7) | ((uint32_t)(kTrTile >> 4) << 24);      // of products: sums of 32 bits; codes, with a sign, as A; 128 rows
constexpr int kTrFlush = 256;                                         // tiles after which the accumulators are moved on all the same: 2^15 keys * 128 * 255 < 2^31

__device__ int g_tree_error = 0;

// How the work is shared out: the keys of all (sequence, kv head) pairs, one pair behind the other, are cut into equal shares of whole tiles, whatever the lengths are, and `tiles` CTAs
// with R of the queries each walk a share. A pair that a cut goes through leaves partial results, two a CTA at most (of the pair that its share begins in, and of the one it
// ends in), which a second kernel joins.
struct TreeLaunch {
    tenzo_attention_tree_args a;
    int group, tiles, shares;                            // heads a kv head; CTAs for a tree's queries; shares of the keys
    int cut;                                             // shares end anywhere; otherwise with a pair
    int aligned;                                         // queries and tables, to 16 bytes
    int2* head;                                          // [pair]: the share that its first tile is in, and the shares that it has a part of; 0 where no cut goes through it
    float* part_o;                                       // [share][tile][2][R][128]
    float2* part_ml;                                     // [share][tile][2][R]: reference (log2), sum
    float* weight;
};

// R queries a CTA.
template <int R>
struct TreeShape {
    static constexpr int groups = R / 16, warps = R / 4, threads = (warps + 4) * 32;      // four warps for sixteen queries; two that copy, one or two that issue products, four of these in all
    // 64 queries are two lines of 32, which have the tiles in common and wait for nothing else of each other: the tensor cores work for the one while the other's warps make weights.
    static constexpr int lines = R == 64 ? 2 : 1, line = R / lines, line_warps = line / 4;
    static constexpr int stages = R > 32 ? 3 : 2, resident = R > 32 ? 1 : 2;
    static constexpr int s_cols = 4 * line, o_cols = 4 * line, all_s = 4 * R, all_o = 4 * R, tmem_cols = R > 32 ? 512 : R == 32 ? 256 : 128;
    static_assert(all_s + all_o <= tmem_cols, "tensor memory: scores, products with the values");
    // Registers a thread: as the block is launched, and after the warps of the second line have given some to those of the first.
    static constexpr int launched = R == 64 ? 96 : R == 48 ? 128 : R == 32 ? 80 : 128, most = R == 64 ? 112 : R == 48 ? 144 : R == 32 ? 104 : 168, least = R == 48 ? 40 : R == 16 ? 64 : 32;
    static_assert(warps * most + 4 * least <= (warps + 4) * launched, "what is taken is there");
    static_assert(launched == 65536 / (threads * resident) / 8 * 8, "as many as the launch bounds leave, which the compiler takes where warps hand registers on; the build checks that it has");
    static constexpr int p_panels = R > 32 ? 2 : 1;                   // of 128 bytes: 32 queries
    static constexpr int q_bytes = all_s * kK8Hd, p_bytes = p_panels * kTrTileBytes;
    static constexpr bool kept_shared = R != 32;                      // outputs that were moved on lie in shared memory; of two CTAs of 32 queries there is no room for them, and they are the threads' own
    static constexpr size_t smem = 1024 + (size_t)stages * 2 * kTrTileBytes + q_bytes + p_bytes + stages * 2 * kTrTile * 4 + (kept_shared ? R * kTrTile * 4 : 0);
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
// What one lane of a warp does that is together: which, and a product and a commit of it. (From a branch that one lane takes, the same products start 93 cycles apart and those of 256
// columns take 169; like this 77 and 128, which is what the multiplications take.)
__device__ __forceinline__ uint32_t tr_elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void tr_mma(uint32_t elected, uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
__device__ __forceinline__ void tr_commit(uint32_t elected, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)), "r"(elected) : "memory");
}
// Operand tiles that are contiguous along M or N (rows of 128 bytes, one for each k), 128-byte swizzle: eight k are 1024 bytes, `panel` bytes from one 128 to the next.
__device__ __forceinline__ uint64_t tr_desc_mn(uint32_t saddr, uint32_t panel) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ f32x2 tr_mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 tr_fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// Two sums from the four parts of whole numbers (below 2^21 each), highest first.
__device__ __forceinline__ f32x2 tr_whole(const uint32_t* a, const uint32_t* b, const uint32_t* c, const uint32_t* d) {
    const f32x2 high = pack2((float)((int)a[0] * 256 + (int)b[0]), (float)((int)a[1] * 256 + (int)b[1]));
    return tr_fma2(high, pack2(65536.0f, 65536.0f), pack2((float)((int)c[0] * 256 + (int)d[0]), (float)((int)c[1] * 256 + (int)d[1])));
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
__device__ __forceinline__ int tr_tiles(const TreeSequence& q) { return q.padding || q.refused ? 0 : (int)(((long long)q.start + q.count + kTrTile - 1) / kTrTile); }

// Where the block's share begins, found by all of its threads.
struct TreeShareAt {
    long long tiles, all, first;                         // a share; all of them; the first tile of this one
    int s;                                               // its sequence,
    long long before;                                    // whose first tile is this
};
template <int THREADS>
__device__ __forceinline__ TreeShareAt tr_share(const TreeLaunch& L, int share, long long (&s_scan)[THREADS / 32 + 2], int& s_found) {
    static_assert(THREADS % 32 == 0, "whole warps");
    const tenzo_attention_tree_args& a = L.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    TreeShareAt at = {0, 0, 0, 0, 0};
    // Sum of the tiles in front of sequence base + tid, counted from `base`; `sum`: of all THREADS.
    auto scan = [&](int base, long long& mine, long long& sum) {
        mine = base + tid < a.sequences ? (long long)tr_tiles(TreeSequence(a, base + tid)) * a.cache.n_kv : 0;
        long long up = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += v;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp] = up;
        __syncthreads();
        long long front = 0;
        sum = 0;
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) front += s_scan[w];
            sum += s_scan[w];
        }
        return front + up - mine;
    };
    long long mine = 0, sum = 0, front = scan(0, mine, sum);
    at.all = sum;
    for (int base = THREADS; base < a.sequences; base += THREADS) {
        long long m, n;
        scan(base, m, n);
        at.all += n;
    }
    at.tiles = (at.all + L.shares - 1) / L.shares;
    if (at.tiles < 1) at.tiles = 1;
    at.first = share * at.tiles;
    if (at.first >= at.all) return at;
    long long before = 0;
    for (int base = 0; base < a.sequences; base += THREADS) {
        if (base > 0) front = scan(base, mine, sum);
        const long long b = before + front;
        if (mine > 0 && b <= at.first && at.first < b + mine) {      // one thread
            s_found = base + tid;
            s_scan[THREADS / 32] = b;
        }
        before += sum;
        if (before > at.first) break;
    }
    __syncthreads();
    at.s = s_found;
    at.before = s_scan[THREADS / 32];
    return at;
}

// The pieces of a share, one after the other: tiles t0 .. t1 - 1 of a pair. Every role of a block walks them for itself.
struct TreeWalk {
    const TreeLaunch& L;
    long long u, end;                                    // the tile to go on with, and the end of the share
    int s, kvh, t0, t1, tiles;                           // tiles of the pair
    int start, count, seq;
    __device__ __forceinline__ TreeWalk(const TreeLaunch& launch, const TreeShareAt& at) : L(launch), u(at.first), end(min(at.all, at.first + at.tiles)), s(at.s), t1(0) {
        load();
        const long long in = at.first - at.before;
        kvh = (int)(in / tiles);
        t1 = (int)(in % tiles);                          // (next() goes on from here)
        if (!L.cut && t1 > 0) {                          // the pair is another share's
            u += tiles - t1;
            t1 = tiles;
        }
    }
    __device__ __forceinline__ void load() {
        const TreeSequence q(L.a, s);
        start = q.start;
        count = q.count;
        seq = q.seq;
        tiles = tr_tiles(q);
    }
    __device__ __forceinline__ bool next() {
        if (u >= end) return false;
        if (t1 == tiles) {
            t1 = 0;
            if (++kvh == L.a.cache.n_kv) {
                kvh = 0;
                do {
                    ++s;
                    load();
                } while (tiles == 0);                    // (there is a tile to go on with, so there is a sequence)
            }
        }
        t0 = t1;
        t1 = L.cut ? (int)min((long long)tiles, t0 + (end - u)) : tiles;
        u += t1 - t0;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == tiles; }
};

// ---- the parts that both kernels have ------------------------------------------------------------------------------------------
// R queries of a block on their way to the operand, four by each of its R / 4 warps. A lane has dims 4 lane .. 4 lane + 3, and the lane sixteen on, or back, those that they are turned
// with. A vector is turned, scaled by a power of two to a maximum between 2^29 and 2^30 and rounded; its signed bytes are rows r, LINE + r, .., 3 LINE + r of its line's operand (128 bytes each, swizzled).
// s_f: what a unit of the products with the codes counts in the argument of 2^x (NaN for a query that is not finite). from[r]: the vector in q, -1: none, zeros.
// (Every load is made, of something, without a branch around it: where two ways meet the compiler copies what was loaded, and so waits for it. Bytes cut off one after another, by shifts, made the
// weights of 4 x 250 nodes, which are mostly this, 178 us, like this 168, with three bytes; with four 180.)
template <int R, int LINE, bool VEC>
__device__ __forceinline__ void tr_queries(const TreeLaunch& L, const long long* from, const int* pos, unsigned char* s_q, float* s_f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool rotate = L.a.rope_cos != nullptr;
    auto load4 = [](const float* p, float (&v)[4]) {
        if (VEC) {
            const float4 w = ld_l2(reinterpret_cast<const float4*>(p));
            v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = ld_l2(p + j);
        }
    };
    float x[4][4], c[4][4], s[4][4];
    long long at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = from[warp + i * (R / 4)];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float* q = L.a.q + max(at[i], 0LL);
        const size_t turn = (size_t)(at[i] < 0 ? 0 : pos[warp + i * (R / 4)]) * 64 + 4 * (lane & 15);
        load4(q + 4 * lane, x[i]);
        load4(rotate ? (lane < 16 ? L.a.rope_cos : L.a.rope_sin) + turn : q, c[i]);
        load4(rotate ? (lane < 16 ? L.a.rope_sin : L.a.rope_cos) + turn : q, s[i]);
    }
    if (rotate) {                                        // x c - other s in the lower half, other s + x c in the upper one, whose tables were taken the other way round
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float other = __shfl_xor_sync(0xffffffffu, x[i][j], 16);
                x[i][j] = __fmaf_rn(lane < 16 ? x[i][j] : other, c[i][j], (lane < 16 ? -other : x[i][j]) * s[i][j]);
            }
    }
    uint32_t most[4];                                    // bits of the largest magnitude: infinity's and above where one is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t m = 0x15f79688u;                        // (1e-25)
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7fffffffu);
        most[i] = __reduce_max_sync(0xffffffffu, m);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = warp + i * (R / 4);
        const bool bad = most[i] >= 0x7f800000u;         // (its bytes are anything, as those of a vector that is not there)
        const uint32_t e = most[i] >> 23;                // 43 .. 254
        const float up = bad || at[i] < 0 ? 0.0f : __uint_as_float((283u - e) << 23);
        uint32_t v[4];                                   // with 128 added to every byte, carries and all, the bytes are the four signed ones and 128 each
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (uint32_t)__float2int_rn(x[i][j] * up) + 0x80808080u;
        const uint32_t low0 = prmt(v[0], v[1], 0x5140u), low1 = prmt(v[2], v[3], 0x5140u), top0 = prmt(v[0], v[1], 0x7362u), top1 = prmt(v[2], v[3], 0x7362u);
        const uint32_t part[4] = {prmt(top0, top1, 0x7632u), prmt(top0, top1, 0x5410u), prmt(low0, low1, 0x7632u), prmt(low0, low1, 0x5410u)};
        static_assert(LINE % 8 == 0, "the parts of a vector are swizzled alike");
        unsigned char* to = s_q + (r / LINE * (4 * LINE) + r % LINE) * kK8Hd + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(to + k * LINE * kK8Hd) = part[k] ^ 0x80808080u;
        if (lane == 0) s_f[r] = at[i] < 0 ? 0.0f : bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((e - 29u) << 23) * (0.08838834764831845f * 1.4426950408889634f);
    }
}

// A warp that copies keys, or values: a tile after the other into a ring of stages, the codes by tensor copies of sixteen rows, a lane of eight each, the scales by sixteen bytes a lane. A block
// whose table entry is out of range is left out (its bit in s_valid is 0). (A warp issues its lanes' copies one by one: with both rings and the scales' copies, four a lane, in one warp 64 queries'
// tiles took 3500 cycles and were waited for.)
template <int STAGES>
struct TreeCopies {
    const tenzo_attention_tree_args& a;
    const CUtensorMap* map;
    const float *scale_k, *scale_v;                      // (those of the values come with the keys; null: none)
    unsigned char* stages;                               // [STAGES]
    float* scales;                                       // [STAGES][2][128]
    uint64_t *full, *empty;                              // [STAGES]; full: 33 arrivals and the copies' bytes
    unsigned* s_valid;                                   // [STAGES], or null
    int *rows, rows_most;                                // null, or where the rows of the last tiles' chunks are remembered: [tile % rows_most][8]
    int n;                                               // tiles that were asked for
    // Tiles t0 .. t1 - 1 of a pair, `passes` times.
    __device__ __forceinline__ bool run(int seq, int kvh, int total, int t0, int t1, int passes) {
        const int lane = threadIdx.x & 31, n_tiles = t1 - t0, steps = n_tiles * passes, per = a.cache.slots / kK8Chunk;
        auto first_row = [&](int i) -> int {             // of the sixteen keys that lane copies in step i + lane / 8; -1: none
            i += lane >> 3;
            const int u = (t0 + i % n_tiles) * (kTrTile / kK8Chunk) + (lane & 7);
            if (i >= steps || (long long)u * kK8Chunk >= total) return -1;
            const int column = u / per, id = ld_l2(a.cache.block_table + (size_t)seq * a.cache.table_stride + column);
            if (id < 0 || id >= a.cache.n_blocks) {
                atomicOr(&g_tree_error, kK8ErrIndex);
                return -1;
            }
            return (int)kv8_row(a.cache, a.layer, kvh, id, (u - column * per) * kK8Chunk);
        };
        int now = first_row(0), next = first_row(4);
        for (int i = 0; i < steps; ++i, ++n) {
            const int st = n % STAGES, use = n / STAGES;
            if (i > 0 && (i & 3) == 0) {
                now = next;
                next = first_row(i + 4);
            }
            const int mine = __shfl_sync(0xffffffffu, now, 8 * (i & 3) + (lane >> 2));           // row of the chunk whose scales 4 (lane % 4) .. the lane copies
            const unsigned there = __ballot_sync(0xffffffffu, now >= 0) >> (8 * (i & 3)) & 0xffu;
            const bool ok = use == 0 || mbar_wait_bounded(&empty[st], (unsigned)(use - 1) & 1u);
            if (!__all_sync(0xffffffffu, ok)) return false;
            auto copy = [&](const float* from, float* to) {
                if (from && mine >= 0) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to + 4 * lane)), "l"(from + mine + 4 * (lane & 3)) : "memory");
            };
            copy(scale_k, scales + 2 * st * kTrTile);
            copy(scale_v, scales + (2 * st + 1) * kTrTile);
            if (rows && (lane >> 3) == (i & 3)) rows[n % rows_most * 8 + (lane & 7)] = now;
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(&full[st])) : "memory");
            __syncwarp();                                // (lane 0's arrival says that the rows are written)
            if (lane == 0) {
                if (s_valid) s_valid[st] = there;
                mbar_expect_tx(&full[st], (unsigned)__popc(there) * (kK8Chunk * kK8Hd));
            }
            __syncwarp();
            if ((lane >> 3) == (i & 3) && now >= 0) tma_load_2d(stages + (size_t)st * kTrTileBytes + (lane & 7) * kK8Chunk * kK8Hd, map, 0, now, &full[st]);
            __syncwarp();
        }
        return true;
    }
    // After a wait that was given up: copies in flight land before the block ends.
    __device__ __forceinline__ void drain() const {
        for (int i = max(0, n - STAGES); i < n; ++i) mbar_wait_bounded(&full[i % STAGES], (unsigned)(i / STAGES) & 1u);
    }
};

// What a row sees of its tree, word by word; nothing where it is not there.
struct TreeMask {
    uint32_t word[kTrMask];
    __device__ __forceinline__ void load(const tenzo_attention_tree_args& a, size_t row, int node) {
#pragma unroll
        for (int w = 0; w < kTrMask; ++w)
            if (32 * w < a.nodes) word[w] = a.mask ? (uint32_t)ld_l2(a.mask + row * a.mask_stride + w) : node >= 32 * w + 31 ? 0xffffffffu : node < 32 * w ? 0u : (2u << (node - 32 * w)) - 1u;
    }
    __device__ __forceinline__ void store(const tenzo_attention_tree_args& a, bool there, uint32_t (&mask)[kTrMask]) const {
#pragma unroll
        for (int w = 0; w < kTrMask; ++w)
            if (32 * w < a.nodes) mask[w] = there ? word[w] : 0u;
    }
};

// For sixteen queries (columns of each part, R apart), two by two, and the lane's key, whose scale is sk: arguments of 2^x less what `down` (with its sign turned) says.
template <int R>
__device__ __forceinline__ void tr_arguments(uint32_t tmem, const float* s_f, const float* s_down, float sk, f32x2 (&w)[8]) {
    const f32x2 sk2 = pack2(sk, sk);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t part[4][8];
#pragma unroll
        for (int k = 0; k < 4; ++k) tr_ld8(tmem + k * R + 8 * h, part[k]);
        tr_wait8(part[0]);
        tr_tie8(part[1]); tr_tie8(part[2]); tr_tie8(part[3]);
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(s_f + 8 * h + j), m = *reinterpret_cast<const ulonglong2*>(s_down + 8 * h + j);
            w[4 * h + j / 2] = tr_fma2(tr_whole(part[0] + j, part[1] + j, part[2] + j, part[3] + j), tr_mul2(sk2, f.x), m.x);
            w[4 * h + j / 2 + 1] = tr_fma2(tr_whole(part[0] + j + 2, part[1] + j + 2, part[2] + j + 2, part[3] + j + 2), tr_mul2(sk2, f.y), m.y);
        }
    }
}

// Sums over the warp of sixteen numbers a lane: that of number lane / 2.
__device__ __forceinline__ float tr_sums(const f32x2 (&l)[8]) {
    float v[16];
#pragma unroll
    for (int r = 0; r < 8; ++r) unpack2(l[r], v[2 * r], v[2 * r + 1]);
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o > 1; o >>= 1) {                   // half of the numbers go to the other half of the lanes
#pragma unroll
        for (int r = 0; r < o / 2; ++r) {
            const float keep = lane & o ? v[r + o / 2] : v[r], give = lane & o ? v[r] : v[r + o / 2];
            v[r] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
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
    __shared__ __align__(16) float s_f[R];
    __shared__ __align__(16) float s_down[R];            // the references with their signs turned
    __shared__ __align__(16) float s_max[4][R], s_sum[4][R], s_scale_max[S::groups][4];
    __shared__ __align__(16) float4 s_unit[S::groups];   // of these queries' weights: log2 of a scale that is as good as 1, that and the slack, 2^26 over it, it over 2^26
    __shared__ long long s_at[R], s_from[R];             // [row][head] of a query, and its vector in q; -1: none of this tree's, or refused
    __shared__ __align__(16) uint32_t s_mask[R][kTrMask];
    __shared__ int s_pos[R];
    __shared__ uint64_t s_full[2 * S::stages], s_empty[2 * S::stages], s_bar[S::lines][4];     // rings of keys and of values
    __shared__ unsigned s_valid[S::stages];
    __shared__ uint32_t s_tmem, s_set[S::groups];        // queries that have a reference
    __shared__ int s_vote[S::groups][2], s_found;
    __shared__ long long s_scan[S::threads / 32 + 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, tile = (int)blockIdx.x % L.tiles, share = (int)blockIdx.x / L.tiles, flat0 = tile * R;
    unsigned char* base = tr_smem + (((smem_addr(tr_smem) + 1023u) & ~1023u) - smem_addr(tr_smem));
    unsigned char *s_q = base + S::stages * 2 * kTrTileBytes, *s_p = s_q + S::q_bytes;
    float *s_scales = reinterpret_cast<float*>(s_p + S::p_bytes), *s_kept = s_scales + S::stages * 2 * kTrTile;
    enum { kScores, kFree, kWeights, kValues };          // a line's scores are there; were read; weights are there; their products are done
    if (tid == 0) {
        for (int i = 0; i < 2 * S::stages; ++i) {
            mbar_init(&s_full[i], 33);
            mbar_init(&s_empty[i], i < S::stages ? S::lines + S::warps : S::lines);       // products, and for the keys the warps that read the scales
        }
        for (int i = 0; i < S::lines; ++i) {
            mbar_init(&s_bar[i][kScores], 2);            // the products, and the thread that has seen the copies land
            mbar_init(&s_bar[i][kFree], S::line_warps);
            mbar_init(&s_bar[i][kWeights], S::line_warps);
            mbar_init(&s_bar[i][kValues], 1);
        }
        mbar_init_fence();
        for (int g = 0; g < S::groups; ++g) s_vote[g][0] = s_vote[g][1] = 0;
    }
    if (warp == S::warps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(S::tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        // Kernels behind this one may come in only when the block has its tensor memory: one that allocates all of it, and then waits for this one, would otherwise be waited for by the allocation above
        // where the kernel in front still holds some. (The second kernel waits for this one whatever its neighbours do.)
        if (a.use_pdl || L.cut) pdl_launch_dependents();
    }
    if (a.use_pdl) pdl_wait();
    tc_fence_before();
    const TreeShareAt at = tr_share<S::threads>(L, share, s_scan, s_found);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    const bool idle = at.first >= at.all;
    constexpr int kWithQueries = (S::warps + S::lines) * 32, kQueries = 6;       // threads that wait for a pair's queries, and their barrier
    bool ok = true;

    if (!idle && warp >= S::warps) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::least));
    if (idle || warp > S::warps + 1 + S::lines) {
    } else if (warp >= S::warps && warp <= S::warps + 1) {         // keys; values
        const int ring = warp - S::warps;
        TreeCopies<S::stages> copies = {a, ring ? &vmap : &kmap, ring ? nullptr : a.cache.scale_k, ring ? nullptr : a.cache.scale_v, base + (size_t)ring * S::stages * kTrTileBytes, s_scales,
                                        s_full + ring * S::stages, s_empty + ring * S::stages, ring ? nullptr : s_valid, nullptr, 0, 0};
        for (TreeWalk walk(L, at); ok && walk.next();) {
            if (flat0 >= walk.count * L.group) continue;             // rows of padding alone
            ok = copies.run(walk.seq, walk.kvh, walk.start + walk.count, walk.t0, walk.t1, 1);
        }
        if (!ok) copies.drain();
    } else if (warp > S::warps + 1) {                    // the products of a line
        constexpr uint32_t d_scores = kTrShape | (1u << 10) | ((uint32_t)(S::s_cols >> 3) << 17);                             // S^T = K Q^T
        constexpr uint32_t d_values = kTrShape | (1u << 15) | (1u << 16) | ((uint32_t)(S::o_cols >> 3) << 17);                 // O^T += V^T P^T, both operands transposed
        const int line = warp - S::warps - 2;
        uint64_t* bar = s_bar[line];
        const uint32_t t_scores = tmem + line * S::s_cols, t_values = tmem + S::all_s + line * S::o_cols;
        const uint64_t dq = umma_desc_sw128(smem_addr(s_q) + line * S::s_cols * kK8Hd), dp = tr_desc_mn(smem_addr(s_p) + line * kTrTileBytes, kTrTileBytes);
        const uint32_t one = tr_elect();
        int n = 0;                                       // tiles so far
        auto wait = [&](uint64_t* b, int k) { ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(b, (unsigned)k & 1u)); };
        auto scores = [&](int k) {                       // of the k-th tile
            const int st = k % S::stages;
            wait(&s_full[st], k / S::stages);
            if (k > 0) wait(&bar[kFree], k - 1);
            if (!ok) return;
            tc_fence_after();
            const uint64_t dk = umma_desc_sw128(smem_addr(base + (size_t)st * kTrTileBytes));
#pragma unroll
            for (int i = 0; i < kK8Hd / 32; ++i) tr_mma(one, t_scores, dk + (uint64_t)(2 * i), dq + (uint64_t)(2 * i), d_scores, i > 0);
            tr_commit(one, &bar[kScores]);
            tr_commit(one, &s_empty[st]);
            if (one) mbar_arrive(&bar[kScores]);
        };
        for (TreeWalk walk(L, at); walk.next();) {
            if (flat0 >= walk.count * L.group) continue;
            __syncwarp();
            named_barrier_sync(kQueries, kWithQueries);
            if (!ok) continue;
            scores(n);
            for (int i = walk.t0; ok && i < walk.t1; ++i, ++n) {
                if (i + 1 < walk.t1) scores(n + 1);
                const int st = n % S::stages;
                wait(&s_full[S::stages + st], n / S::stages);
                wait(&bar[kWeights], n);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dv = tr_desc_mn(smem_addr(base + (size_t)(S::stages + st) * kTrTileBytes), kTrTileBytes);
#pragma unroll
                for (int k = 0; k < kTrTile / 32; ++k) tr_mma(one, t_values, dv + (uint64_t)(k * (32 * kK8Hd >> 4)), dp + (uint64_t)(k * (32 * kK8Hd >> 4)), d_values, 1u);
                tr_commit(one, &bar[kValues]);
                tr_commit(one, &s_empty[S::stages + st]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::most));
        const int quarter = warp & 3, group = warp >> 2, first = group * 16, key = 32 * quarter + lane;      // its keys of a tile, and its queries
        constexpr int kAll = S::warps * 32, kEvery = 7;              // threads, and their barrier (1 .. 4: those of sixteen queries)
        const int line = first / S::line, in_line = first % S::line;
        uint64_t* bar = s_bar[line];
        const uint32_t t_lane = tmem + ((uint32_t)(32 * quarter) << 16), t_scores = t_lane + (uint32_t)(line * S::s_cols + in_line),
                       t_values = t_lane + (uint32_t)(S::all_s + 4 * first);
        // Outputs of dim `key` that were moved on, seldom looked at.
        float* kept = s_kept + first * kTrTile + key;
        volatile float kept_own[S::kept_shared ? 1 : 16];
        tr_fill<64>(t_values, 0u);
        tmem_wait_st();
        tc_fence_before();
        int n = 0;                                       // tiles so far
        for (TreeWalk walk(L, at); walk.next();) {
            if (flat0 >= walk.count * L.group) continue;
            // ---- the queries ----
            named_barrier_sync(kEvery, kAll);            // (those in front are done with)
            if (tid < R) {
                const int flat = flat0 + tid, node = flat / L.group;
                const size_t row = (size_t)walk.s * a.nodes + node;
                long long to = -1;
                int pos = -1;
                TreeMask mask = {};
                if (flat < walk.count * L.group) {
                    pos = a.rope_pos ? ld_l2(a.rope_pos + row) : walk.start + node;
                    mask.load(a, row, node);
                    to = (long long)(row * a.n_q + (size_t)walk.kvh * L.group + flat - node * L.group);
                    if (tr_position_refused(a, pos)) {
                        atomicOr(&g_tree_error, kK8ErrIndex);
                        to = -1;
                    }
                }
                s_at[tid] = to;
                s_pos[tid] = pos;
                s_from[tid] = to < 0 ? -1 : (long long)(row * a.q_stride + ((size_t)walk.kvh * L.group + flat - node * L.group) * kK8Hd);
                s_down[tid] = 0.0f;
                mask.store(a, to >= 0, s_mask[tid]);
            }
            if (lane == 0 && quarter == 0) {
                s_unit[group] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                s_set[group] = 0;
            }
            named_barrier_sync(kEvery, kAll);
            if (L.aligned) tr_queries<R, S::line, true>(L, s_from, s_pos, s_q, s_f);
            else tr_queries<R, S::line, false>(L, s_from, s_pos, s_q, s_f);
            fence_proxy_async_smem();
            named_barrier_sync(kQueries, kWithQueries);
            f32x2 l[8];                                  // of key `key`: sums
#pragma unroll
            for (int r = 0; r < 8; ++r) l[r] = 0;
            bool has = false;                            // kept_own has something
            if (S::kept_shared) {
#pragma unroll
                for (int j = 0; j < 16; ++j) kept[j * kTrTile] = 0.0f;
            }
            // Eight queries' outputs of dim `key`: what was moved on, and the accumulators.
            auto moved = [&](int h, float unit, float (&o)[8]) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    uint32_t v[8];
                    tr_ld8(t_values + 4 * (h + j), v);
                    tr_wait8(v);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float hi = __fmaf_rn((float)(int)v[4 * k + 3], 256.0f, (float)(int)v[4 * k + 2]), lo = __fmaf_rn((float)(int)v[4 * k + 1], 256.0f, (float)(int)v[4 * k]);
                        o[j + k] = __fmaf_rn(__fmaf_rn(hi, 65536.0f, lo), unit, S::kept_shared ? kept[(h + j + k) * kTrTile] : 0.0f);
                    }
                }
                if (has) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] += kept_own[S::kept_shared ? 0 : h + j];
                }
            };
            const int total = walk.start + walk.count;
            bool early = false;                          // the next scores were seen to be there
            for (int i = walk.t0; i < walk.t1; ++i, ++n) {
                const int st = n % S::stages, t = i * kTrTile + key;
                if (!early) ok = ok && mbar_wait_bounded(&bar[kScores], (unsigned)n & 1u);
                __syncwarp();
                const unsigned valid = s_valid[st];
                const bool ragged = (i + 1) * kTrTile > walk.start || valid != 0xffu;
                const bool dead = ragged && (t >= total || !(valid >> (key >> 4) & 1u));
                float sv = dead ? 0.0f : s_scales[(2 * st + 1) * kTrTile + key], sk = dead ? 0.0f : s_scales[2 * st * kTrTile + key];
                if (!(sv < INFINITY)) {                  // the value of a key that is no number: it spoils the rows that see it by way of their sums
                    sv = 0.0f;
                    sk = __uint_as_float(0x7fc00000u);
                }
                tc_fence_after();
                f32x2 w[8];
                tr_arguments<S::line>(t_scores, s_f + first, s_down + first, sk, w);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bar[kFree]);
                    mbar_arrive(&s_empty[st]);
                }
                const bool values_early = n == 0 || mbar_test(&bar[kValues], (unsigned)(n - 1) & 1u);     // (looked at when the weights are ready to be stored)
                if (ragged) tr_hide(w, s_mask + first, t - walk.start, dead);
                float over = -INFINITY;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float w0, w1;
                    unpack2(w[r], w0, w1);
                    over = fmaxf(fmaxf(over, w0), w1);
                }
                const uint32_t set = s_set[group];
                const float4 unit = s_unit[group];
                const float log_scale = fmaxf(tr_lg2(sv), unit.x - kTrScales);
                if (over + log_scale > unit.y || set != 0xffffu || (n + 1) % kTrFlush == 0) s_vote[group][n & 1] = n + 1;
                named_barrier_sync(1 + group, 128);
                const int vote = *reinterpret_cast<volatile int*>(&s_vote[group][n & 1]);
                f32x2 p[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float w0, w1;
                    unpack2(w[r], w0, w1);
                    p[r] = pack2(tr_ex2(w0), tr_ex2(w1));
                }
                if (vote == n + 1) {
                    // ---- references of these sixteen queries anew, and their accumulators moved on ----
                    float top = -INFINITY;               // lane r: of query `first` + r, less the reference
#pragma unroll
                    for (int r = 0; r < 16; r += 2) {
                        float w0, w1;
                        unpack2(w[r / 2], w0, w1);
                        w0 = tr_warp_max(w0 + log_scale);
                        w1 = tr_warp_max(w1 + log_scale);
                        if (lane == r) top = w0;
                        if (lane == r + 1) top = w1;
                    }
                    if (lane < 16) s_max[quarter][first + lane] = top;
                    const float most = tr_warp_max(over > -INFINITY ? sv : 0.0f);      // (a key that none of these queries sees does not count)
                    if (lane == 0) s_scale_max[group][quarter] = most;
                    named_barrier_sync(1 + group, 128);
                    const float4 scales = *reinterpret_cast<const float4*>(s_scale_max[group]);
                    // The unit is set with the first references: a power of two above the largest scale there, 2^-60 to 2^30 (1, where all of them are 0).
                    const float scale_most = fmaxf(fmaxf(scales.x, scales.y), fmaxf(scales.z, scales.w));
                    const int bits = scale_most > 0.0f ? (int)min(max((__float_as_uint(scale_most) >> 23) + 1u, 67u), 157u) : 127;
                    const float log_unit = set ? unit.x : (float)(bits - 127);
                    float up, by;                        // of query `first` + lane % 16: how far its reference goes up (the first one may go down), and what that leaves of its sums
                    {
                        const int r = lane & 15;
                        const bool was = set >> r & 1u;
                        top = fmaxf(fmaxf(s_max[0][first + r], s_max[1][first + r]), fmaxf(s_max[2][first + r], s_max[3][first + r])) - log_unit;
                        up = was ? fmaxf(top, 0.0f) : top == -INFINITY ? 0.0f : top;
                        by = was ? tr_ex2(-up) : 0.0f;   // (there is nothing yet)
                    }
                    const uint32_t now_set = set | (__ballot_sync(0xffffffffu, top != -INFINITY) & 0xffffu);
                    if (quarter == 0) {
                        if (lane < 16) s_down[first + lane] -= up;
                        if (lane == 0) {
                            if (!set && now_set) s_unit[group] = make_float4(log_unit, log_unit + kTrSlack, __uint_as_float((uint32_t)(254 + kTrOne - bits) << 23), __uint_as_float((uint32_t)(bits - kTrOne) << 23));
                            s_set[group] = now_set;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; r += 2) {
                        const float u0 = __shfl_sync(0xffffffffu, up, r), u1 = __shfl_sync(0xffffffffu, up, r + 1);
                        const float b0 = __shfl_sync(0xffffffffu, by, r), b1 = __shfl_sync(0xffffffffu, by, r + 1);
                        float w0, w1;
                        unpack2(w[r / 2], w0, w1);
                        l[r / 2] = tr_mul2(l[r / 2], pack2(b0, b1));
                        p[r / 2] = pack2(tr_ex2(w0 - u0), tr_ex2(w1 - u1));
                    }
                    if (i > walk.t0) {
                        ok = ok && mbar_wait_bounded(&bar[kValues], (unsigned)(n - 1) & 1u);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll
                        for (int h = 0; h < 16; h += 8) {
                            float o[8];
                            moved(h, unit.w, o);
#pragma unroll
                            for (int r = 0; r < 8; ++r) {
                                o[r] *= __shfl_sync(0xffffffffu, by, h + r);
                                if (S::kept_shared) kept[(h + r) * kTrTile] = o[r]; else kept_own[S::kept_shared ? 0 : h + r] = o[r];
                            }
                        }
                        has = !S::kept_shared;
                        tr_fill<64>(t_values, 0u);
                        tmem_wait_st();
                        tc_fence_before();
                    }
                    named_barrier_sync(1 + group, 128);
                }
                const float by = sv * s_unit[group].z;
                const f32x2 by2 = pack2(by, by);
                uint32_t word[16];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float p0, p1;
                    l[r] = add2(l[r], p[r]);
                    unpack2(tr_mul2(p[r], by2), p0, p1);
                    word[2 * r] = __float2uint_rn(p0);
                    word[2 * r + 1] = __float2uint_rn(p1);
                }
                if (!values_early) ok = ok && mbar_wait_bounded(&bar[kValues], (unsigned)(n - 1) & 1u);    // (the weights in front were read)
                __syncwarp();
                unsigned char* to = s_p + (first >> 5) * kTrTileBytes + key * kK8Hd;
                const int chunk = (first & 31) >> 2;
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(to + (((chunk + c) ^ (key & 7)) << 4)) = make_uint4(word[4 * c], word[4 * c + 1], word[4 * c + 2], word[4 * c + 3]);
                early = i + 1 < walk.t1 && mbar_test(&bar[kScores], (unsigned)(n + 1) & 1u);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar[kWeights]);
            }
            // ---- the outputs ----
            ok = ok && mbar_wait_bounded(&bar[kValues], (unsigned)(n - 1) & 1u);
            __syncwarp();
            tc_fence_after();
            const float mine = tr_sums(l);
            if (!(lane & 1)) s_sum[quarter][first + (lane >> 1)] = mine;
            named_barrier_sync(1 + group, 128);
            const bool whole = walk.whole();
            const size_t part = (((size_t)share * L.tiles + tile) * 2 + (walk.t0 > 0 ? 0 : 1)) * R + first;
            const uint32_t set = s_set[group];
            float inv, log_sum;                          // lane r: of query `first` + r
            {
                const int r = lane & 15;
                const float sum = (s_sum[0][first + r] + s_sum[1][first + r]) + (s_sum[2][first + r] + s_sum[3][first + r]);
                inv = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
                log_sum = sum == 0.0f ? -INFINITY : (tr_lg2(sum) - s_down[first + r]) * 0.6931471805599453f;
                const long long to = s_at[first + r];
                if (quarter == 0 && lane < 16 && to >= 0) {
                    if (!whole) L.part_ml[part + r] = make_float2(set >> r & 1u ? -s_down[first + r] : kTrLow, sum);
                    else if (a.lse) a.lse[to] = log_sum;
                }
            }
            if (L.cut && tile == 0 && walk.t0 == 0 && tid == 0)      // (what this share leaves goes to the next ones, at.tiles each)
                L.head[(size_t)walk.s * a.cache.n_kv + walk.kvh] = make_int2(share, whole ? 0 : 1 + (int)((walk.tiles - walk.t1 + at.tiles - 1) / at.tiles));
#pragma unroll
            for (int h = 0; h < 16; h += 8) {
                float o[8];
                moved(h, s_unit[group].w, o);
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const long long to = s_at[first + h + r];
                    const float by = __shfl_sync(0xffffffffu, inv, h + r);
                    float* out = whole ? a.out + (size_t)to * kK8Hd : L.part_o + (part + h + r) * kK8Hd;
                    if (to >= 0) out[key] = o[r] * by;
                }
            }
            tr_fill<64>(t_values, 0u);                   // for the next pair
            tmem_wait_st();
            tc_fence_before();
        }
    }
    // Rows of padding, and sequences that are refused: a share of them to each block.
    for (int s = (int)blockIdx.x; s < a.sequences; s += (int)gridDim.x) {
        const TreeSequence q(a, s);
        if (q.refused) {
            if (tid == 0) atomicOr(&g_tree_error, kK8ErrIndex);
            continue;
        }
        const int there = q.padding ? 0 : q.count;
        const size_t from = ((size_t)s * a.nodes + there) * a.n_q, rest = (size_t)(a.nodes - there) * a.n_q;
        for (size_t i = tid; i < rest * (kK8Hd / 4); i += S::threads) reinterpret_cast<float4*>(a.out)[from * (kK8Hd / 4) + i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (a.lse)
            for (size_t i = tid; i < rest; i += S::threads) a.lse[from + i] = -INFINITY;
    }
    if (!ok) atomicOr(&g_tree_error, kK8ErrWait);
    tc_fence_before();
    __syncthreads();
    if (warp == S::warps) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::tmem_cols) : "memory");
    }
}

// The parts of a (row, head) that cuts go through: one warp each, four dims a lane.
constexpr int kTrMergeWarps = 4;
__global__ void __launch_bounds__(kTrMergeWarps * 32) attention_tree_merge_kernel(const TreeLaunch L, const int queries) {
    const tenzo_attention_tree_args& a = L.a;
    const int lane = threadIdx.x & 31, head = blockIdx.y * kTrMergeWarps + (threadIdx.x >> 5);
    const size_t row = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    if (head >= a.n_q) return;
    const int s = (int)blockIdx.x / a.nodes, node = (int)blockIdx.x - s * a.nodes, kvh = head / L.group, flat = node * L.group + head - kvh * L.group;
    // (Everything is asked for that does not hang on something else, then the first eight parts and what they count: two ways to memory. One after the other these were 4.6 us of tree 1 x 8's 14.)
    const unsigned long long pair = ld_l2(reinterpret_cast<const unsigned long long*>(L.head) + (size_t)s * a.cache.n_kv + kvh);
    const int given = ld_l2(a.rope_pos ? a.rope_pos + row : a.start + s);
    const TreeSequence q(a, s);
    const int first = (int)(uint32_t)pair, parts = (int)(pair >> 32), pos = a.rope_pos ? given : given + node;
    if (q.refused || q.padding || node >= q.count || tr_position_refused(a, pos) || parts == 0) return;
    // part i is of share first + i: its second, for the first of them (the pair begins in that share, or at its begin), the first one of the others
    const size_t at = ((size_t)first * L.tiles + flat / queries) * 2 * queries + flat % queries, step = (size_t)L.tiles * 2 * queries;
    auto where = [&](int i) { return at + i * step + (i == 0 ? queries : 0); };
    constexpr int kBatch = 8;                            // loads in flight
    float2 v[kBatch];
    float4 p[kBatch];
    auto load = [&](int i0) {                            // (the last part again, where there is none)
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const size_t from = where(min(i0 + u, parts - 1));
            v[u] = ld_l2(L.part_ml + from);
            p[u] = ld_l2(reinterpret_cast<const float4*>(L.part_o + from * kK8Hd) + lane);
        }
    };
    load(0);
    float m = -INFINITY;
    for (int i = kBatch + lane; i < parts; i += 32) m = fmaxf(m, ld_l2(L.part_ml + where(i)).x);
    m = warp_max(m);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) m = fmaxf(m, v[u].x);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    for (int i0 = 0; i0 < parts; i0 += kBatch) {
        if (i0 > 0) load(i0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (i0 + u >= parts) break;
            const float x = tr_ex2(v[u].x - m);
            o.x = __fmaf_rn(p[u].x, x, o.x);
            o.y = __fmaf_rn(p[u].y, x, o.y);
            o.z = __fmaf_rn(p[u].z, x, o.z);
            o.w = __fmaf_rn(p[u].w, x, o.w);
            l = __fmaf_rn(v[u].y, x, l);
        }
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;         // (a query with a NaN has a NaN here)
    reinterpret_cast<float4*>(a.out + (row * a.n_q + head) * kK8Hd)[lane] = make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
    if (lane == 0 && a.lse) a.lse[row * a.n_q + head] = l == 0.0f ? -INFINITY : (m + tr_lg2(l)) * 0.6931471805599453f;
}

// ---- the weight that keys receive -------------------------------------------------------------------------------------------------
// The same scores, R queries a pass: a thread has one key, so its sum over sixteen queries needs no other lane. With sixteen a CTA it is added to the key's weight at once, without a wait (one
// tile belongs to one CTA, a second pass's addition comes from the same thread behind the first: one order of summation). With more, four warps' sums of a key have to come together: they lie in
// shared memory, for as many tiles at a time as there is room for, until all passes over these are done. Nothing holds the warps together but the scores, of which there are two sets.
// Bound by the bytes of the keys for single tokens (64 sequences of 8192 keys, 5 kv heads: 69 us, 54 at the memory's rate), behind a start of some 14000 cycles; for trees by the
// chain of a pass's queries (5000 cycles, which a CTA's few tiles do not hide: 7 x 33 nodes, 8 x 4 heads, 6001 keys: 52 us) and 1200 cycles a tile of 48 queries.
// Measured, with queries of three bytes: sums of single tokens in shared memory as well 42.5 us (64 x 4096 keys; at once 40.0, with four bytes 38.8); two CTAs an SM of 16 queries and four stages 70.5 (64 x 24 queries; three of three stages 67.2);
// 64 tiles a block instead of 128 at 48 queries 41.6 (32 x 48; 40.1); eight of sixteen queries left out where there are four: no difference.
template <int R>
struct WeighShape {
    static constexpr int groups = R / 16, warps = R / 4, threads = (warps + 2) * 32, stages = R == 16 ? 3 : 4, resident = R == 16 ? 3 : 1;
    static constexpr bool direct = groups == 1;                       // a key has one thread: its sums go to its weight at once
    static constexpr int most = direct ? 1 << 30 : 128 / groups, rows_most = direct ? stages : most + 2 * stages;
    static constexpr int s_cols = 4 * R, tmem_cols = R > 32 ? 512 : R == 32 ? 256 : 128;         // two sets of scores
    static constexpr int q_bytes = s_cols * kK8Hd;
    static constexpr size_t smem = 1024 + (size_t)stages * kTrTileBytes + q_bytes + stages * 2 * kTrTile * 4 + (direct ? 0 : groups * most * kTrTile * 4);
};

template <int R>
__global__ void __launch_bounds__(WeighShape<R>::threads, WeighShape<R>::resident) tree_weigh_kernel(const TreeLaunch L, const __grid_constant__ CUtensorMap kmap) {
    using S = WeighShape<R>;
    const tenzo_attention_tree_args& a = L.a;
    extern __shared__ unsigned char tr_smem[];
    __shared__ __align__(16) float s_f[R];
    __shared__ __align__(16) float s_down[R];            // log-sum-exps with their signs turned
    __shared__ long long s_from[R];
    __shared__ __align__(16) uint32_t s_mask[R][kTrMask];
    __shared__ int s_pos[R];
    __shared__ uint64_t s_full[S::stages], s_empty[S::stages], s_scores[2], s_free[2];
    __shared__ unsigned s_valid[S::stages];
    __shared__ uint32_t s_tmem;
    __shared__ int s_found, s_given_up, s_rows[S::rows_most * 8];    // (s_rows: rows of the chunks of the last tiles)
    __shared__ long long s_scan[S::threads / 32 + 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned char* base = tr_smem + (((smem_addr(tr_smem) + 1023u) & ~1023u) - smem_addr(tr_smem));
    unsigned char* s_q = base + S::stages * kTrTileBytes;
    float *s_scales = reinterpret_cast<float*>(s_q + S::q_bytes), *s_sum = s_scales + 2 * S::stages * kTrTile;
    if (tid == 0) {
        s_given_up = 0;
        for (int i = 0; i < S::stages; ++i) {
            mbar_init(&s_full[i], 33);
            mbar_init(&s_empty[i], S::warps + 1);        // the products, and the warps that read the scales
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_scores[i], 2);                  // the products, and the thread that has seen the copies land
            mbar_init(&s_free[i], S::warps);
        }
        mbar_init_fence();
    }
    if (warp == S::warps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(S::tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        if (a.use_pdl) pdl_launch_dependents();          // (as in the attention: only with the block's tensor memory)
    }
    if (a.use_pdl) pdl_wait();
    tc_fence_before();
    const TreeShareAt at = tr_share<S::threads>(L, (int)blockIdx.x, s_scan, s_found);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    constexpr int kWithQueries = (S::warps + 1) * 32, kQueries = 6;
    bool ok = true;

    if (at.first >= at.all) {
    } else if (warp == S::warps) {
        TreeCopies<S::stages> copies = {a, &kmap, a.cache.scale_k, nullptr, base, s_scales, s_full, s_empty, s_valid, s_rows, S::rows_most, 0};
        for (TreeWalk walk(L, at); ok && walk.next();)
            for (int t0 = walk.t0; ok && t0 < walk.t1; t0 += S::most)
                ok = copies.run(walk.seq, walk.kvh, walk.start + walk.count, t0, min(walk.t1, t0 + S::most), (walk.count * L.group + R - 1) / R);
        if (!ok) copies.drain();
    } else if (warp == S::warps + 1) {
        constexpr uint32_t shape = kTrShape | (1u << 10) | ((uint32_t)(S::s_cols >> 3) << 17);
        const uint64_t dq = umma_desc_sw128(smem_addr(s_q));
        const uint32_t one = tr_elect();
        int n = 0;
        for (TreeWalk walk(L, at); walk.next();)
            for (int t0 = walk.t0; t0 < walk.t1; t0 += S::most)
                for (int flat0 = 0; flat0 < walk.count * L.group; flat0 += R) {
                    __syncwarp();
                    named_barrier_sync(kQueries, kWithQueries);
                    for (int i = t0; ok && i < min(walk.t1, t0 + S::most); ++i, ++n) {
                        const int st = n % S::stages, half = n & 1;
                        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[st], (unsigned)(n / S::stages) & 1u) && (n < 2 || mbar_wait_bounded(&s_free[half], (unsigned)(n / 2 - 1) & 1u)));
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dk = umma_desc_sw128(smem_addr(base + (size_t)st * kTrTileBytes));
#pragma unroll
                        for (int k = 0; k < kK8Hd / 32; ++k) tr_mma(one, tmem + half * S::s_cols, dk + (uint64_t)(2 * k), dq + (uint64_t)(2 * k), shape, k > 0);
                        tr_commit(one, &s_scores[half]);
                        tr_commit(one, &s_empty[st]);
                        if (one) mbar_arrive(&s_scores[half]);
                    }
                }
    } else {
        const int quarter = warp & 3, group = warp >> 2, first = group * 16, key = 32 * quarter + lane;
        constexpr int kAll = S::warps * 32, kEvery = 7;
        const uint32_t t_scores = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)first;
        float* sums = s_sum + group * S::most * kTrTile + key;
        int n = 0;
        for (TreeWalk walk(L, at); walk.next();)
            for (int t0 = walk.t0; t0 < walk.t1; t0 += S::most) {
                const int t1 = min(walk.t1, t0 + S::most), queries = walk.count * L.group, total = walk.start + walk.count;
                for (int flat0 = 0; flat0 < queries; flat0 += R) {
                    named_barrier_sync(kEvery, kAll);    // (the queries in front, and the sums, are done with)
                    if (tid < R) {
                        const int flat = flat0 + tid, node = flat / L.group;
                        const size_t row = (size_t)walk.s * a.nodes + node;
                        float lse = INFINITY;            // of a query that does not count
                        int pos = -1;
                        TreeMask mask = {};
                        if (flat < queries) {
                            pos = a.rope_pos ? ld_l2(a.rope_pos + row) : walk.start + node;
                            lse = ld_l2(a.lse + row * a.n_q + (size_t)walk.kvh * L.group + flat - node * L.group) * 1.4426950408889634f;
                            mask.load(a, row, node);
                            if (!(fabsf(lse) < INFINITY)) lse = INFINITY;
                            if (tr_position_refused(a, pos)) {
                                atomicOr(&g_tree_error, kK8ErrIndex);
                                lse = INFINITY;
                            }
                        }
                        s_down[tid] = -lse;
                        s_pos[tid] = pos;
                        s_from[tid] = lse < INFINITY ? (long long)(row * a.q_stride + ((size_t)walk.kvh * L.group + flat - node * L.group) * kK8Hd) : -1;
                        mask.store(a, lse < INFINITY, s_mask[tid]);
                    }
                    named_barrier_sync(kEvery, kAll);
                    if (L.aligned) tr_queries<R, R, true>(L, s_from, s_pos, s_q, s_f);
                    else tr_queries<R, R, false>(L, s_from, s_pos, s_q, s_f);
                    fence_proxy_async_smem();
                    named_barrier_sync(kQueries, kWithQueries);
                    for (int i = t0; i < t1; ++i, ++n) {
                        const int st = n % S::stages, half = n & 1, t = i * kTrTile + key;
                        ok = ok && mbar_wait_bounded(&s_scores[half], (unsigned)(n / 2) & 1u);
                        __syncwarp();
                        const unsigned valid = s_valid[st];
                        const int direct = S::direct ? s_rows[n % S::rows_most * 8 + (key >> 4)] : -1;
                        if (!S::direct && ok && flat0 == 0 && group == 0 && (lane & 15) == 0) {     // the weights, which are wanted when the last pass is done
                            const int row = s_rows[n % S::rows_most * 8 + (key >> 4)];
                            if (row >= 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(L.weight + row));
                        }
                        const bool ragged = (i + 1) * kTrTile > walk.start || valid != 0xffu, dead = ragged && (t >= total || !(valid >> (key >> 4) & 1u));
                        float sk = dead ? 0.0f : s_scales[2 * st * kTrTile + key];
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
                        if (ragged) tr_hide(w, s_mask + first, t - walk.start, dead);
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
                        if (!S::direct) sums[(i - t0) * kTrTile] = flat0 == 0 ? sum : sums[(i - t0) * kTrTile] + sum;
                        else if (ok && !dead) atomicAdd(L.weight + direct + (key & (kK8Chunk - 1)), sum);      // (sums below 2^-126 are 0)
                    }
                }
                if (S::direct) continue;
                if (!ok) s_given_up = 1;
                named_barrier_sync(kEvery, kAll);
                // (behind n the copies are at most `stages` tiles)
                weigh_add<S::groups, S::most, S::rows_most, kAll, kTrTile, kK8Chunk>(*reinterpret_cast<volatile int*>(&s_given_up) != 0, tid, n, t0, t1, total, s_rows, s_sum, L.weight);
            }
    }
    if (blockIdx.x == 0)
        for (int s = tid; s < a.sequences; s += S::threads)
            if (TreeSequence(a, s).refused) atomicOr(&g_tree_error, kK8ErrIndex);
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
    if (a.nodes > TENZO_TREE_MOST || a.n_q > 1 << 17 || a.cache.n_kv > 65535 || a.max_len > 1 << 30) return -5;
    if (a.q_stride == 0) a.q_stride = a.n_q * kK8Hd;
    if (a.q_stride < a.n_q * kK8Hd) return -1;
    const int words = (a.nodes + 31) / 32;
    if (a.mask_stride == 0) a.mask_stride = words;
    if (a.mask_stride < words) return -1;
    L.group = a.n_q / a.cache.n_kv;
    // (Vectors of four where all rows allow it: 16 trees of 64 nodes, 8192 keys, 234 us, by single numbers 250; their weights 162 and 202.)
    L.aligned = kv8_aligned(a.q, 16) && a.q_stride % 4 == 0 && kv8_aligned(a.rope_cos, 16) && kv8_aligned(a.rope_sin, 16);
    return 0;
}

static int tree_map(CUtensorMap* map, const tenzo_kv8_cache& c, const int8_t* codes) {
    return encode_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, kK8Hd, (uint64_t)c.n_blocks * c.n_layers * c.n_kv * c.slots, kK8Hd, kK8Hd, kK8Chunk, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Queries a CTA of the attention: the width at which the CTAs that a tree's queries take cost least, one of 16, 32 and 48 as this much of one of 64. Measured, sequences x 4096 keys:
// 64 x 24 queries 91 us at 32, 103 at 16, 117 at 48; 32 x 48: 69 at 48, 80 at 64, 90 at 32; 32 x 64: 82 at 64, 92 at 32; 32 x 80: 123 at 48, 129 at 32, 142 at 64; 16 x 128: 79 at
// 64, 89 at 32; 16 x 144: 95 at 48, 109 at 32 and 64; 4 x 1000: 144 at 64, 152 at 48, 163 at 32; and 64 x 4 queries of 8192 keys 121 at 16, 144 at 32. (80 queries take 32: short
// sequences pay for a change of pair, 26 x 270 queries of 51 keys 14.3 at 32, 18.6 at 48.)
static int tree_queries_a_cta(long long queries) {
    constexpr int width[4] = {64, 48, 32, 16};
    constexpr double cost[4] = {1.0, 0.80, 0.53, 0.32};
    int best = 0;
    for (int i = 1; i < 4; ++i)
        if (cost[i] * (double)((queries + width[i] - 1) / width[i]) < cost[best] * (double)((queries + width[best] - 1) / width[best])) best = i;
    return width[best];
}
// Queries a pass over the keys whose weights are summed, of which a CTA makes as many as there are: 16, twice if that is enough (64 sequences of 20 or 32 queries, 4096 keys: 63 and 64 us; in one of
// 48, 78); then 48 (32 x 48: 43 us, three of 16 48, one of 64 50; 32 x 80: 73, 75 and 88) or 64, of which a pass of 48 costs 0.87 (32 x 64: 51 us at 64, 62 at 16, 73 at 48; 16 x 128: 50 at 64,
// 61 at 48; 4 x 1000: 180 and 195).
static int weigh_queries_a_pass(long long queries) {
    if (queries <= 32) return 16;
    return 0.87 * (double)((queries + 47) / 48) < (double)((queries + 63) / 64) ? 48 : 64;
}

// Shares of the keys, with CTAs for every SM.
static void tree_plan(TreeLaunch& L) {
    const tenzo_attention_tree_args& a = L.a;
    const long long queries = (long long)a.nodes * L.group;
    const int r = tree_queries_a_cta(queries), places = 148 * (r > 32 ? 1 : 2);
    L.tiles = (int)((queries + r - 1) / r);
    L.shares = a.shares > 0 ? a.shares : L.tiles < places ? places / L.tiles : 1;
}
// Bytes for what cuts leave: nothing is cut where there is one share, as with queries for half of the SMs and more (a few bytes all the same: 0 is the answer to arguments that are refused).
static size_t tree_room(const TreeLaunch& L) {
    const int r = tree_queries_a_cta((long long)L.a.nodes * L.group);
    const size_t head = ((size_t)L.a.sequences * L.a.cache.n_kv * sizeof(int2) + 15) & ~(size_t)15;
    return head + (L.shares == 1 ? 16 : (size_t)L.shares * L.tiles * 2 * r * (kK8Hd + 2) * sizeof(float));
}

template <int R>
static int tree_run(const TreeLaunch& L, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t st) {
    if (cudaError_t e = allow_smem(attention_tree_kernel<R>, TreeShape<R>::smem)) return (int)e;
    // With fewer registers than the warps ask of one another they would wait for good; the kernel's number is the compiler's. (Registers are given out by eights.)
    static const bool registers_ok = [] {
        cudaFuncAttributes f = {};
        return cudaFuncGetAttributes(&f, attention_tree_kernel<R>) == cudaSuccess && (f.numRegs + 7) / 8 * 8 >= TreeShape<R>::launched && f.numRegs <= TreeShape<R>::most;
    }();
    if (!registers_ok) return (int)cudaErrorLaunchOutOfResources;
    return kv4_launch(attention_tree_kernel<R>, dim3((unsigned)(L.shares * L.tiles)), TreeShape<R>::threads, TreeShape<R>::smem, st, L.a.use_pdl != 0, L, kmap, vmap);
}
template <int R>
static int weigh_run(TreeLaunch L, const CUtensorMap& kmap, cudaStream_t st) {
    if (cudaError_t e = allow_smem(tree_weigh_kernel<R>, WeighShape<R>::smem)) return (int)e;
    L.shares = 148 * WeighShape<R>::resident;
    L.cut = 1;
    return kv4_launch(tree_weigh_kernel<R>, dim3((unsigned)L.shares), WeighShape<R>::threads, WeighShape<R>::smem, st, L.a.use_pdl != 0, L, kmap);
}

static bool tree_sizes_ok(int sequences, int nodes, int n_q, int n_kv) {
    return sequences > 0 && nodes > 0 && nodes <= TENZO_TREE_MOST && n_q > 0 && n_kv > 0 && n_q % n_kv == 0 && n_q <= 1 << 17 && n_kv <= 65535;
}

}  // namespace tz

extern "C" size_t tenzo_cuda_attention_tree_workspace_bytes(int sequences, int nodes, int n_q, int n_kv, int shares) {
    using namespace tz;
    if (!tree_sizes_ok(sequences, nodes, n_q, n_kv) || shares < 0 || shares > 65535) return 0;
    TreeLaunch L = {};
    L.a.sequences = sequences; L.a.nodes = nodes; L.a.n_q = n_q; L.a.cache.n_kv = n_kv; L.a.shares = shares;
    L.group = n_q / n_kv;
    tree_plan(L);
    return tree_room(L);
}

extern "C" int tenzo_cuda_attention_tree(const tenzo_attention_tree_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    TreeLaunch L = {};
    L.a = *args;
    tenzo_attention_tree_args& a = L.a;
    if (a.sequences == 0) return 0;
    if (int rc = tree_check(L)) return rc;
    if (!a.out || !kv8_aligned(a.out, 16) || a.shares < 0 || a.shares > 65535) return -1;
    {                                                    // (a query, and what names it, is read by every CTA that has some of its keys)
        const size_t row = (size_t)a.n_q * kK8Hd, rows = (size_t)a.sequences * a.nodes, q_bytes = ((rows - 1) * a.q_stride + row) * sizeof(float);
        const size_t out_bytes = rows * row * sizeof(float), lse_bytes = rows * a.n_q * sizeof(float);
        if (kv8_overlap(a.q, q_bytes, a.out, out_bytes) || kv8_overlap(a.q, q_bytes, a.lse, lse_bytes) || kv8_overlap(a.out, out_bytes, a.lse, lse_bytes)) return -1;
    }
    tree_plan(L);
    L.cut = a.workspace && kv8_aligned(a.workspace, 16) && a.workspace_bytes >= tree_room(L);
    if (a.shares > 0 && !L.cut) return -1;
    // Up to four tiles are not cut, and the call is one launch: what the cut saves the second kernel takes again. Whole and cut, 20 heads over 5, us: 8 nodes, 500 keys, one sequence 13.4 and 12.4, 16
    // sequences 18.2 and 19.6, 64 33.3 and 37.2; 64 nodes 17.2 and 17.8, 41.6 and 49.5, 120 and 157. Beyond that the rule goes by one sequence, which gains most (1000 keys: 19.6 and 12.7, 22.6 and 19.4);
    // many sequences of some eight tiles are slower cut (8 nodes: 16 sequences 25.2 and 28.6, 64 46.5 and 45.9; 64 nodes: 58.5 and 61.9, 168 and 204; of 2000 keys 38.2 and 32.4, 72.1 and 62.5, 91.2
    // and 90.6, 265 and 298): a call without a workspace leaves them whole.
    if (L.shares == 1 || (a.shares == 0 && a.max_len <= 4 * kTrTile)) L.cut = 0;
    if ((long long)L.shares * L.tiles > 0x7fffffffLL || (long long)a.sequences * a.nodes > 0x7fffffffLL) return -5;
    const int r = tree_queries_a_cta((long long)a.nodes * L.group);
    L.head = static_cast<int2*>(a.workspace);
    L.part_o = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + (((size_t)a.sequences * a.cache.n_kv * sizeof(int2) + 15) & ~(size_t)15));
    L.part_ml = reinterpret_cast<float2*>(L.part_o + (size_t)L.shares * L.tiles * 2 * r * kK8Hd);
    CUtensorMap kmap, vmap;
    if (int rc = tree_map(&kmap, a.cache, a.cache.k)) return rc;
    if (int rc = tree_map(&vmap, a.cache, a.cache.v)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (int rc = r == 16 ? tree_run<16>(L, kmap, vmap, st) : r == 32 ? tree_run<32>(L, kmap, vmap, st) : r == 48 ? tree_run<48>(L, kmap, vmap, st) : tree_run<64>(L, kmap, vmap, st))
        return rc;
    if (!L.cut) return 0;
    return kv4_launch(attention_tree_merge_kernel, dim3((unsigned)(a.sequences * a.nodes), (unsigned)((a.n_q + kTrMergeWarps - 1) / kTrMergeWarps)), kTrMergeWarps * 32, 0, st, true, L, r);
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
    CUtensorMap kmap;
    if (int rc = tree_map(&kmap, a.cache, a.cache.k)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int r = weigh_queries_a_pass((long long)a.nodes * L.group);
    return r == 16 ? weigh_run<16>(L, kmap, st) : r == 48 ? weigh_run<48>(L, kmap, st) : weigh_run<64>(L, kmap, st);
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
