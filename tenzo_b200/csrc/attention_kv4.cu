// GQA decode attention over the 4-bit paged cache (kv4.cuh): softmax(q K^T / sqrt(128)) V over the keys 0 .. pos of a row's sequence,
// the query rotated on the way.
//
//   * The keys of a (row, kv head) are split over CTAs and, inside a CTA, over four warps that never wait for one another: each streams
//     steps of 32 keys, two pages of 2560 bytes by one bulk copy each, through a ring of its own and keeps a running
//     (maximum, sum, output) per query head. The triples meet by log-sum-exp, first the warps', then the splits': in shared memory of a
//     thread-block cluster, or in a second kernel where there are too many.
//   * With value = minimum + scale * code per group of 32 dims,
//       q.k   = sum_g scale_g (q_g . c_g) + minimum_g (sum of q over g)
//       p.v_d = sum_t (p_t scale_tg) (c_td - 8) + sum_t p_t (minimum_tg + 8 scale_tg)
//     the products with codes run on the tensor cores, which see nothing but codes as they lie, and the scales go in fp32 to the sums (keys) or to the
//     weights (values); the other terms are one MMA more, over the parameters.
//   * Keys: whole numbers. A head's query is scaled to a maximum of 2^22 - 1 and rounded, and its three signed bytes are rows of the A operand (products of bytes and
//     codes, 32 dims a chain: exact in 32 bits). Up to four heads a kv head, rows 0-3 have the first bytes, 4-7 the second and 8-11 the third, so one MMA does; with
//     more a second one.
//   * Values: fp16. A nibble in the low bits of a 16-bit word is the number code * 2^-24, one field further up code * 2^-20; one packed fused
//     multiplication makes two of them normal numbers (code - 8) * 2^-9. (The tensor cores take subnormal operands too, exactly, but line the products up by the
//     exponent they are written with: sums lose the leading zeros' bits, 1e-5 instead of 4e-7 over 100 keys. And they cut off what a sum's last bit
//     does not hold, always towards zero: hence codes around zero, and accumulators of 32 keys that are added up in fp32.) The weights, up to 2^14 with the largest
//     scale of the values seen so far, enter as two parts of eleven bits.
//   * S = Q K^T has heads as rows, and its accumulators are, lane by lane, the weights' B operand of O^T = V^T P^T, whose columns are heads. Up to four heads a kv
//     head, columns 4-7 carry the weights' second parts; with five to eight a second MMA does.
// In fewer bits than fp32: the query (whole numbers of 23 bits of its head's largest), the weights (two parts of eleven bits, cut off) and the centres of the values (two fp16 parts).
// Outputs differ from 64 bits by 5e-7 to 1e-6 of their norm (1 x 1000 keys 4.7e-7, 256 ragged 6.3e-7, 64 x 8192 8.0e-7, 4 x 16000 9.9e-7; plain fp32 7.5e-7, 1.2e-6, 1.8e-6, 7.9e-7).
//
// 64 x 8192 keys of 20/5 heads: 114 us, 420 MB at 3.7 TB/s or 0.56 of the memory's rate. What takes its time is instructions: some 1100 slots for a step of 32 keys,
// three quarters of them unpacking, scaling and converting around the 38 MMAs (110 us without the copies, 78 without the MMAs and what they need, 44 without either); 56 % of
// the issue slots are used, the rest is fixed latencies that three or four warps a scheduler do not cover.
#include "attn_common.cuh"
#include "kv4.cuh"

#include <cuda_fp16.h>

namespace tz {

constexpr int kA4Hd = 128, kA4Warps = 4, kA4Threads = kA4Warps * 32;
constexpr int kA4Step = 32;                              // keys a warp takes at a time
constexpr int kA4Stages = 2, kA4StepBytes = 2 * kK4Page;
constexpr int kA4Resident = 4;                           // CTAs an SM
constexpr int kA4Cluster = 8;                            // splits that a cluster may take
constexpr int kA4MostSplits = 64;                        // and a choice of its own, at most

__device__ int g_kv4_attention_error = 0;

struct A4Launch {
    tenzo_attention_kv4_args a;
    int n_splits, split_keys, group, head_blocks;        // query heads a kv head, and blocks of them that a CTA takes
    int cluster;                                         // the splits of an item are a thread-block cluster, which joins them itself
    float* part_o;                                       // [row][head][split][128]
    float2* part_ml;                                     // [row][head][split]: maximum (log2), sum
};

__device__ __forceinline__ float a4_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t a4_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float a4_low(uint32_t pair) { return __low2float(*reinterpret_cast<const __half2*>(&pair)); }
__device__ __forceinline__ float a4_high(uint32_t pair) { return __high2float(*reinterpret_cast<const __half2*>(&pair)); }
// D = A B (+ D); the accumulators of the first form start at zero.
__device__ __forceinline__ void a4_mma16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void a4_mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void a4_mma8_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
__device__ __forceinline__ f32x2 a4_mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 a4_fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// The eleven leading bits of two numbers as fp16 (towards zero).
__device__ __forceinline__ uint32_t a4_pack_cut(float lo, float hi) {
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Codes of a word as two fp16 numbers (code - 8) * 2^-9: nibbles 0 and 4, nibbles 1 and 5.
__device__ __forceinline__ uint32_t a4_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
constexpr uint32_t kMinus8 = 0xa400a400u;                                                     // -2^-6
__device__ __forceinline__ uint32_t a4_even(uint32_t w) { return a4_fma(w & 0x000f000fu, 0x78007800u, kMinus8); }    // code * 2^-24, times 2^15
__device__ __forceinline__ uint32_t a4_odd(uint32_t w) { return a4_fma(w & 0x00f000f0u, 0x68006800u, kMinus8); }     // code * 2^-20, times 2^11

// Rows that are left alone (a position or a sequence out of range); the same rule in both kernels.
__device__ __forceinline__ bool a4_refused(const tenzo_attention_kv4_args& a, int pos, int seq) { return pos >= a.max_len || seq < 0 || seq >= a.cache.table_rows; }

// D = A B, signed bytes times codes.
__device__ __forceinline__ void a4_imma(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(0));
}

template <int HB>
__global__ void __launch_bounds__(kA4Threads, kA4Resident) attention_kv4_kernel(const A4Launch L) {
    static_assert(HB == 4 || HB == 8, "heads a CTA takes");
    const tenzo_attention_kv4_args& a = L.a;
    extern __shared__ __align__(128) unsigned char a4_smem[];
    __shared__ float s_q[HB][kA4Hd], s_qsum[HB][4], s_f[HB], s_ml[kA4Warps][HB][2];
    __shared__ uint64_t s_bar[kA4Warps][kA4Stages];
    __shared__ __align__(16) float s_scale[kA4Warps][2][kA4Step / 2][4][2];      // a step's scales, keys and values: [pair of keys][group][key]
    __shared__ __align__(16) uint4 s_centre[kA4Warps][kA4Step];                  // minimum + 8 scale of the values: four first parts, four second ones
    __shared__ __align__(16) uint4 s_qa[4][HB == 8 ? 2 : 1][32];      // the queries' A fragments, the same in every warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int row = blockIdx.x / L.n_splits, split = blockIdx.x % L.n_splits;
    const int kvh = blockIdx.y / L.head_blocks, head0 = blockIdx.y % L.head_blocks * HB, heads = min(HB, L.group - head0);
    if (lane == 0)
        for (int s = 0; s < kA4Stages; ++s) mbar_init(&s_bar[warp][s], 2);
    mbar_init_fence();
    if (a.use_pdl || (L.n_splits > 1 && !L.cluster)) pdl_launch_dependents();       // the second kernel waits for this one whatever its neighbours do
    if (a.use_pdl) pdl_wait();
    const int pos = ld_l2(a.pos + row), seq = a.seq ? ld_l2(a.seq + row) : row;
    if (a4_refused(a, pos, seq)) {
        if (tid == 0) atomicOr(&g_kv4_attention_error, kK4ErrIndex);
        return;
    }
    const int c_begin = split * L.split_keys, c_end = min(pos + 1, c_begin + L.split_keys);
    float* out = a.out + ((size_t)row * a.n_q + (size_t)kvh * L.group + head0) * kA4Hd;
    if (c_begin >= c_end && (!L.cluster || pos < 0)) {   // the second kernel knows which splits there are
        if (L.n_splits == 1 || (L.cluster && split == 0))
            for (int i = tid; i < heads * kA4Hd; i += kA4Threads) out[i] = 0.0f;
        return;
    }
    // (a cluster's CTAs without keys go the same way, with no step: 0 outputs, a maximum of -infinity)
    const int steps = max(0, c_end - c_begin + kA4Step - 1) / kA4Step;
    const int my_steps = warp < steps ? (steps - warp + kA4Warps - 1) / kA4Warps : 0;
    const int* table = a.cache.block_table + (size_t)seq * a.cache.table_stride + c_begin / kK4Slots;
    const int pages = max(0, c_end - c_begin + kK4Slots - 1) / kK4Slots;
    unsigned char* ring = a4_smem + (size_t)warp * kA4Stages * kA4StepBytes;
    uint64_t* bar = s_bar[warp];

    // A lane has the address of one page of sixteen of the warp's steps (null: no such page, or a table entry out of range) and copies it when its step's turn comes.
    auto page_at = [&](int k0) -> const uint8_t* {
        const int page = 2 * (warp + (k0 + (lane >> 1)) * kA4Warps) + (lane & 1);
        if (page >= pages) return nullptr;
        const int id = ld_l2(table + page);
        if (id < 0 || id >= a.cache.n_blocks) {
            atomicOr(&g_kv4_attention_error, kK4ErrIndex);
            return nullptr;
        }
        return a.cache.pool + kv4_page(a.cache, a.layer, kvh, id);
    };
    __syncwarp();                                        // (the barriers)
    const uint8_t *from = page_at(0), *from_next = my_steps > 16 ? page_at(16) : nullptr;
    unsigned there = __ballot_sync(0xffffffffu, from != nullptr), there_before = 0;       // of the pages: of these sixteen steps, of those before
    auto issue = [&](int k) {                            // the warp's k-th step into stage k % kA4Stages
        const int st = k % kA4Stages;
        if ((lane >> 1) == (k & 15)) {
            if (from) {
                mbar_expect_tx(&bar[st], (unsigned)kK4Page);
                bulk_g2s(ring + (size_t)st * kA4StepBytes + (lane & 1) * kK4Page, from, kK4Page, &bar[st]);
            } else {
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&bar[st])) : "memory");
            }
        }
        if ((k & 15) == 15) {
            from = from_next;
            there_before = there;
            there = __ballot_sync(0xffffffffu, from != nullptr);
            from_next = page_at(k + 17);
        }
    };
    for (int k = 0; k < kA4Stages && k < my_steps; ++k) issue(k);

    // ---- the heads' queries: rotated, scaled to a maximum of 2^22 - 1 and rounded, and their sums over each group of dims ----
    const float* q = a.q + (size_t)row * a.q_stride + ((size_t)kvh * L.group + head0) * kA4Hd;
    for (int i = tid; i < HB * 64; i += kA4Threads) {
        const int h = i >> 6, d = i & 63;
        float r0 = 0.0f, r1 = 0.0f;
        if (h < heads) {
            const float x0 = ld_l2(q + h * kA4Hd + d), x1 = ld_l2(q + h * kA4Hd + d + 64);
            r0 = x0;
            r1 = x1;
            if (a.rope_cos) {
                const float c = ld_l2(a.rope_cos + (size_t)pos * 64 + d), s = ld_l2(a.rope_sin + (size_t)pos * 64 + d);
                r0 = __fmaf_rn(x0, c, -(x1 * s));
                r1 = __fmaf_rn(x0, s, x1 * c);
            }
        }
        s_q[h][d] = r0;
        s_q[h][d + 64] = r1;
    }
    __syncthreads();
    for (int h = warp; h < HB; h += kA4Warps) {
        float4 v = *reinterpret_cast<const float4*>(&s_q[h][4 * lane]);
        const float m = warp_max(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        const float most = fmaxf(m, 1e-25f), up = 4194303.0f / most, down = most / 4194303.0f;
        v.x = rintf(v.x * up); v.y = rintf(v.y * up); v.z = rintf(v.z * up); v.w = rintf(v.w * up);
        *reinterpret_cast<float4*>(&s_q[h][4 * lane]) = v;
        float sum = (v.x + v.y) + (v.z + v.w);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if ((lane & 7) == 0) s_qsum[h][lane >> 3] = sum;
        if (lane == 0) s_f[h] = down * (0.08838834764831845f * 1.4426950408889634f);           // (the unit of the products), 1/sqrt(128) and log2(e)
    }
    __syncthreads();
    const int mine = g & (HB - 1);                       // the head of a lane's scores
    {                                                    // group `warp`: byte i of a word is dim 8t + 2i, of the other word 8t + 2i + 1
        uint32_t w[4] = {0, 0, 0, 0}, w2[2] = {0, 0};    // rows g, rows g + 8 (see above)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int x = (int)s_q[mine][32 * warp + 8 * t + i];
            const int d3 = ((x + 128) & 255) - 128, r = (x - d3) >> 8, d2 = ((r + 128) & 255) - 128, d1 = (r - d2) >> 8;
            const int up = HB == 8 || g < 4 ? d1 : d2, down = HB == 8 || g < 4 ? d3 : 0, at = 2 * (i & 1), by = 8 * (i >> 1);
            w[at] |= (uint32_t)(up & 255) << by;
            w[at + 1] |= (uint32_t)(down & 255) << by;
            w2[i & 1] |= (uint32_t)(d2 & 255) << by;
        }
        s_qa[warp][0][lane] = make_uint4(w[0], w[1], w[2], w[3]);
        if (HB == 8) s_qa[warp][HB == 8 ? 1 : 0][lane] = make_uint4(w2[0], 0, w2[1], 0);
    }
    uint32_t qm[2] = {0, 0};                             // beside the minimum (the scale has 0); 2^-18 of the products' unit
    if (HB == 8 || g < 4) {
        const float sum = s_qsum[mine][t] * 3.814697265625e-6f, first = __half2float(__float2half_rn(sum));
        qm[0] = a4_pack(0.0f, first);
        qm[1] = a4_pack(0.0f, sum - first);
    }
    const float f = s_f[mine];
    __syncthreads();

    float m_run = -INFINITY, top = 0.0f;                 // head `mine`: largest product so far, its score (log2) less 14
    f32x2 l_pair = 0;                                    // this lane's share of the sum
    float vs = 1.0f;                                     // values' scales are multiplied by this power of two, to at most 1
    uint32_t v_most = 0;                                 // the largest exponent of a scale so far, as fp16 bits
    f32x2 acc[8][2], accm = 0;                           // group i / 2: dims 4g + 2 (i % 2), and + 1; heads 2t, 2t + 1
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = 0;
    const uint32_t cut = HB == 8 || g >= 4 ? 0xffffe000u : 0u;                                  // columns 4-7: what the first eleven bits leave
    const f32x2 minus = pack2(-1.0f, -1.0f), f2 = pack2(f, f), qm_unit = pack2(262144.0f, 262144.0f);
    const int shifted = HB == 8 || g < 4 ? 65536 : 256;  // what the row's digits count
    bool gave_up = false;

    for (int k = 0; k < my_steps; ++k) {
        const int st = k % kA4Stages, t0 = c_begin + (warp + k * kA4Warps) * kA4Step;
        unsigned char* step = ring + (size_t)st * kA4StepBytes;
        if (!mbar_wait_bounded(&bar[st], (unsigned)(k / kA4Stages) & 1u)) gave_up = true;
        // (copies run ahead of the products, so `there` may be of the next sixteen steps already)
        const unsigned copied = ((min(k + kA4Stages, my_steps) >> 4) == (k >> 4) ? there : there_before) >> (2 * (k & 15)) & 3u;
        const bool ragged = t0 + kA4Step > c_end || copied != 3u;
        unsigned char* own = step + (lane >> 4) * kK4Page + (lane & 15) * kK4Row + kK4Codes;    // the parameters of key t0 + lane
        if (ragged) {                                    // keys that do not count: parameters of zero, whatever lies there
            if (t0 + lane >= c_end || !((copied >> (lane >> 4)) & 1u)) {
                *reinterpret_cast<uint4*>(own) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(own + kK4Half) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                   // a later copy into the stage comes after these
            }
            __syncwarp();
        }
        // ---- the step's scales in fp32, one key a lane ---------------------------------------------------------------------
        bool v_grown;
        float ratio = 1.0f;
        {
            const uint4 pk = *reinterpret_cast<const uint4*>(own), pv = *reinterpret_cast<const uint4*>(own + kK4Half);
            const uint32_t v_max = max(max(pv.x & 0x7c00u, pv.y & 0x7c00u), max(pv.z & 0x7c00u, pv.w & 0x7c00u));
            v_grown = __any_sync(0xffffffffu, v_max > v_most) || k == 0;
            if (v_grown) {                               // a scale below 2^(e - 14) times 2^(14 - e) is below 1
                v_most = __reduce_max_sync(0xffffffffu, v_max);
                const float now = __uint_as_float((127u + 14u - max(v_most >> 10, 1u)) << 23);
                ratio = k == 0 ? 1.0f : now / vs;
                vs = now;
            }
            float* ks = &s_scale[warp][0][lane >> 1][0][lane & 1];
            float* vt = &s_scale[warp][1][lane >> 1][0][lane & 1];
            ks[0] = a4_low(pk.x); ks[2] = a4_low(pk.y); ks[4] = a4_low(pk.z); ks[6] = a4_low(pk.w);
            const float sv[4] = {a4_low(pv.x), a4_low(pv.y), a4_low(pv.z), a4_low(pv.w)};
            vt[0] = sv[0] * vs; vt[2] = sv[1] * vs; vt[4] = sv[2] * vs; vt[6] = sv[3] * vs;
            const float c[4] = {__fmaf_rn(8.0f, sv[0], a4_high(pv.x)), __fmaf_rn(8.0f, sv[1], a4_high(pv.y)), __fmaf_rn(8.0f, sv[2], a4_high(pv.z)),
                                __fmaf_rn(8.0f, sv[3], a4_high(pv.w))};
            const uint32_t c01 = a4_pack(c[0], c[1]), c23 = a4_pack(c[2], c[3]);
            s_centre[warp][lane] = make_uint4(c01, c23, a4_pack(c[0] - a4_low(c01), c[1] - a4_high(c01)), a4_pack(c[2] - a4_low(c23), c[3] - a4_high(c23)));
            __syncwarp();
        }
        // ---- products with the keys: columns are eight keys a tile ----------------------------------------------------------
        f32x2 x[4] = {0, 0, 0, 0};
        const unsigned char* kr = step + g * kK4Row + 4 * t;
        auto tile = [](int nt) { return (nt >> 1) * kK4Page + (nt & 1) * 8 * kK4Row; };
#pragma unroll
        for (int gr = 0; gr < 4; ++gr) {
            const uint4 qa = s_qa[gr][0][lane], qb = s_qa[gr][HB == 8 ? 1 : 0][lane];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(kr + tile(nt) + 16 * gr), even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
                int c[4], d[4];
                a4_imma(c, qa, even, odd);               // 32 codes times 22 bits and a sign: 31 bits at most
                c[0] = c[0] * shifted + c[2];
                c[1] = c[1] * shifted + c[3];
                if (HB == 8) {
                    a4_imma(d, qb, even, odd);
                    c[0] += d[0] * 256;
                    c[1] += d[1] * 256;
                }
                x[nt] = a4_fma2(*reinterpret_cast<const f32x2*>(&s_scale[warp][0][4 * nt + t][gr][0]), pack2((float)c[0], (float)c[1]), x[nt]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            float c[4];
            a4_mma8_new(c, qm[0], qm[1], *reinterpret_cast<const uint32_t*>(kr + tile(nt) + kK4Codes));
            x[nt] = a4_fma2(add2(pack2(c[0], c[1]), pack2(c[2], c[3])), qm_unit, x[nt]);
            if (HB == 4) x[nt] = add2(x[nt], __shfl_xor_sync(0xffffffffu, x[nt], 16));
        }
        float s[4][2];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) unpack2(x[nt], s[nt][0], s[nt][1]);
        if (ragged) {
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (t0 + nt * 8 + 2 * t + j >= c_end || !((copied >> (nt >> 1)) & 1u)) s[nt][j] = -INFINITY;
                x[nt] = pack2(s[nt][0], s[nt][1]);
            }
        }
        // ---- the running maximum ---------------------------------------------------------------------------------------------
        float mx = s[0][0];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) mx = fmaxf(mx, fmaxf(s[nt][0], s[nt][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (__any_sync(0xffffffffu, mx > m_run || v_grown)) {
            float alpha = 1.0f;
            if (mx > m_run) {
                const float now = __fmaf_rn(mx, f, -14.0f);
                alpha = m_run == -INFINITY ? 0.0f : a4_ex2(top - now);
                m_run = mx;
                top = now;
            }
            l_pair = a4_mul2(l_pair, pack2(alpha, alpha));
            const f32x2 a01 = pack2(__shfl_sync(0xffffffffu, alpha, 8 * t), __shfl_sync(0xffffffffu, alpha, 8 * t + 4));
            accm = a4_mul2(accm, a01);
            const f32x2 scaled = a4_mul2(a01, pack2(ratio, ratio));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[i][0] = a4_mul2(acc[i][0], scaled);
                acc[i][1] = a4_mul2(acc[i][1], scaled);
            }
        }
        // ---- weights (2^14-fold) and O^T += V^T P^T --------------------------------------------------------------------------
        const f32x2 down = pack2(-top, -top);
        f32x2 e[4];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            float e0, e1;
            unpack2(a4_fma2(x[nt], f2, down), e0, e1);
            e[nt] = pack2(a4_ex2(e0), a4_ex2(e1));
            l_pair = add2(l_pair, e[nt]);
        }
        // The two fp16 parts of a pair of weights: the first eleven bits, and what they leave (cut off in turn: 2^-22 less on average,
        // in all products alike).
        auto parts = [&](f32x2 w, uint32_t& first, uint32_t& second) {
            float w0, w1, r0, r1;
            unpack2(w, w0, w1);
            unpack2(a4_fma2(pack2(__uint_as_float(__float_as_uint(w0) & cut), __uint_as_float(__float_as_uint(w1) & cut)), minus, w), r0, r1);
            if (HB == 8) {
                first = a4_pack_cut(w0, w1);
                second = a4_pack_cut(r0, r1);
            } else {
                first = a4_pack_cut(r0, r1);             // columns 0-3 nothing was taken off, columns 4-7 the first part
            }
        };
        uint32_t b[4], c[4];
        auto product = [&](float (&o)[4], const uint32_t (&v0)[4], const uint32_t (&v1)[4]) {       // the step's 32 keys
            a4_mma16_new(o, v0, b[0], b[1]);
            a4_mma16(o, v1, b[2], b[3]);
            if (HB == 8) {
                a4_mma16(o, v0, c[0], c[1]);
                a4_mma16(o, v1, c[2], c[3]);
            }
        };
        {
            uint32_t v0[4] = {}, v1[4] = {};
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v0[0]), "=r"(v0[2]), "=r"(v1[0]), "=r"(v1[2]) : "r"(smem_addr(&s_centre[warp][lane])) : "memory");
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) parts(e[nt], b[nt], c[nt]);
            float m[4];
            product(m, v0, v1);
            accm = add2(accm, pack2(m[0], m[1]));
        }
        const uint32_t at = smem_addr(step) + (uint32_t)((lane >> 4) * kK4Page + kK4Half + (8 * ((lane >> 3) & 1) + (lane & 7)) * kK4Row);
#pragma unroll
        for (int gr = 0; gr < 4; ++gr) {
            uint32_t r[4];                               // the tiles' keys; dims 32 gr + 4g ..
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at + 16 * gr) : "memory");
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) parts(a4_mul2(e[nt], *reinterpret_cast<const f32x2*>(&s_scale[warp][1][4 * nt + t][gr][0])), b[nt], c[nt]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t v0[4] = {a4_even(r[0]), a4_odd(r[0]), a4_even(r[1]), a4_odd(r[1])};
                const uint32_t v1[4] = {a4_even(r[2]), a4_odd(r[2]), a4_even(r[3]), a4_odd(r[3])};
                float o[4];                              // added in fp32: the tensor cores' own sums are cut off, not rounded
                product(o, v0, v1);
                acc[2 * gr + i][0] = add2(acc[2 * gr + i][0], pack2(o[0], o[1]));
                acc[2 * gr + i][1] = add2(acc[2 * gr + i][1], pack2(o[2], o[3]));
#pragma unroll
                for (int n = 0; n < 4; ++n) r[n] >>= 8;
            }
        }
        __syncwarp();                                    // every lane is done with the stage and the scales
        if (k + kA4Stages < my_steps) issue(k + kA4Stages);
    }
    if (gave_up) atomicOr(&g_kv4_attention_error, kK4ErrWait);                                // (any lane: each waits for itself)
    float l_run, l_other;
    unpack2(l_pair, l_run, l_other);
    l_run += l_other;
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
    l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);

    // ---- the warps' outputs in one unit, then their triples into one --------------------------------------------------------
    __syncthreads();                                     // all rings are idle: reuse them
    float* w_o = reinterpret_cast<float*>(a4_smem);      // [warp][HB][128]
    float am[2];
    unpack2(accm, am[0], am[1]);
    const float unit = 512.0f / vs;
#pragma unroll
    for (int gr = 0; gr < 4; ++gr) {
        const float m0 = __shfl_sync(0xffffffffu, am[0], 4 * gr + t) + __shfl_sync(0xffffffffu, am[0], 16 + 4 * gr + t);
        const float m1 = __shfl_sync(0xffffffffu, am[1], 4 * gr + t) + __shfl_sync(0xffffffffu, am[1], 16 + 4 * gr + t);
        float o[2][4];                                   // [head 2t, 2t + 1][dims 32 gr + 4g ..]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float c[4];
            unpack2(acc[2 * gr + i][0], c[0], c[1]);
            unpack2(acc[2 * gr + i][1], c[2], c[3]);
            o[0][2 * i] = __fmaf_rn(c[0], unit, m0);
            o[1][2 * i] = __fmaf_rn(c[1], unit, m1);
            o[0][2 * i + 1] = __fmaf_rn(c[2], unit, m0);
            o[1][2 * i + 1] = __fmaf_rn(c[3], unit, m1);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (HB == 4) {
#pragma unroll
                for (int d = 0; d < 4; ++d) o[h][d] += __shfl_xor_sync(0xffffffffu, o[h][d], 2);
            }
            if (HB == 8 || t < 2) *reinterpret_cast<float4*>(w_o + ((size_t)warp * HB + 2 * t + h) * kA4Hd + 32 * gr + 4 * g) = make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
        }
    }
    if (t == 0 && g < HB) {
        s_ml[warp][g][0] = m_run == -INFINITY ? -INFINITY : top;
        s_ml[warp][g][1] = l_run;
    }
    __syncthreads();
    float* part = w_o + kA4Warps * HB * kA4Hd;            // the CTA's outputs and (maximum, sum), for the cluster
    float2* part_ml = reinterpret_cast<float2*>(part + HB * kA4Hd);
    for (int i = tid; i < heads * kA4Hd; i += kA4Threads) {
        const int h = i / kA4Hd, d = i % kA4Hd;
        float m = -INFINITY, o = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kA4Warps; ++w) m = fmaxf(m, s_ml[w][h][0]);
        const float m_use = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < kA4Warps; ++w) {
            const float x = a4_ex2(s_ml[w][h][0] - m_use);
            o = __fmaf_rn(w_o[((size_t)w * HB + h) * kA4Hd + d], x, o);
            l = __fmaf_rn(s_ml[w][h][1], x, l);
        }
        if (L.n_splits == 1) {
            out[i] = l == 0.0f ? 0.0f : o / l;
        } else if (L.cluster) {
            part[i] = o;
            if (d == 0) part_ml[h] = make_float2(m, l);
        } else {
            const size_t at = ((size_t)row * a.n_q + (size_t)kvh * L.group + head0 + h) * L.n_splits + split;
            L.part_o[at * kA4Hd + d] = o;
            if (d == 0) L.part_ml[at] = make_float2(m, l);
        }
    }
    if (L.cluster) {                                     // each CTA joins a share of the outputs, from all of the cluster's shared memory
        // (not .aligned: a share's last round leaves lanes out, and nothing says that a warp is together again after a loop)
        auto cluster_sync = [] { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); };
        cluster_sync();
        auto of = [](uint32_t at, int rank) {
            uint32_t r;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
            return v;
        };
        const int share = (heads * kA4Hd + L.n_splits - 1) / L.n_splits;
        for (int i = split * share + tid; i < min(heads * kA4Hd, (split + 1) * share); i += kA4Threads) {
            const uint32_t ml = smem_addr(part_ml + i / kA4Hd), at = smem_addr(part + i);
            float m = -INFINITY, o = 0.0f, l = 0.0f, pm[kA4Cluster];
#pragma unroll
            for (int r = 0; r < kA4Cluster; ++r) {
                pm[r] = r < L.n_splits ? of(ml, r) : -INFINITY;
                m = fmaxf(m, pm[r]);
            }
#pragma unroll
            for (int r = 0; r < kA4Cluster; ++r) {
                const float x = a4_ex2(pm[r] - (m == -INFINITY ? 0.0f : m));
                if (r < L.n_splits) {
                    o = __fmaf_rn(of(at, r), x, o);
                    l = __fmaf_rn(of(ml + 4, r), x, l);
                }
            }
            out[i] = l == 0.0f ? 0.0f : o / l;
        }
        cluster_sync();                                  // until all have read
    }
}

// The splits of a (row, head): one warp each, four dims a lane.
__global__ void __launch_bounds__(kA4Threads) attention_kv4_merge_kernel(const A4Launch L) {
    const tenzo_attention_kv4_args& a = L.a;
    const int lane = threadIdx.x & 31, head = blockIdx.y * kA4Warps + (threadIdx.x >> 5), row = blockIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    if (head >= a.n_q) return;
    const int pos = ld_l2(a.pos + row), seq = a.seq ? ld_l2(a.seq + row) : row;
    if (a4_refused(a, pos, seq)) return;
    const int n = pos < 0 ? 0 : pos / L.split_keys + 1;
    const size_t at = ((size_t)row * a.n_q + head) * L.n_splits;
    const float2* ml = L.part_ml + at;
    const float4* po = reinterpret_cast<const float4*>(L.part_o) + at * (kA4Hd / 4) + lane;
    float m = -INFINITY;
    for (int s = lane; s < n; s += 32) m = fmaxf(m, ld_l2(ml + s).x);
    m = warp_max(m);
    const float m_use = m == -INFINITY ? 0.0f : m;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    constexpr int kBatch = 8;                            // loads in flight
    for (int s0 = 0; s0 < n; s0 += kBatch) {
        float2 v[kBatch];
        float4 p[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            v[u] = s0 + u < n ? ld_l2(ml + s0 + u) : make_float2(-INFINITY, 0.0f);
            p[u] = s0 + u < n ? ld_l2(po + (size_t)(s0 + u) * (kA4Hd / 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const float x = a4_ex2(v[u].x - m_use);
            o.x = __fmaf_rn(p[u].x, x, o.x);
            o.y = __fmaf_rn(p[u].y, x, o.y);
            o.z = __fmaf_rn(p[u].z, x, o.z);
            o.w = __fmaf_rn(p[u].w, x, o.w);
            l = __fmaf_rn(v[u].y, x, l);
        }
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;         // (a query with a NaN has a NaN here)
    reinterpret_cast<float4*>(a.out + ((size_t)row * a.n_q + head) * kA4Hd)[lane] = make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
}

static size_t a4_part_bytes(int rows, int n_q) { return (size_t)rows * n_q * (kA4Hd + 2) * sizeof(float); }

// Keys a CTA takes: the number of splits whose rounds of CTAs take least at the longest length, a CTA's own cost counted as some
// hundred keys. `most`: as many splits as there is room for partial results; `join`: what joining them costs, in keys.
// Against every split by hand: 1 x 16384 keys of 20/5 heads 17.6 us (best 17.6, whole 168), 64 x 8192 114 (114, whole 143, by 512 keys 138), 256 x 4095 ragged 175 (176, by 512
// 209), 4 x 16001 of 32/8 31.4 (31.3), 128 x 1000 41.8 (41.4), 1 x 4000 of 16/16 12.4 (12.1).
static double a4_pick_split(long long items, int max_len, int most, double join, int* n_splits, int* split_keys) {
    const long long places = 148 * kA4Resident;
    double best = 0.0;
    for (int want = 1; want <= most; ++want) {
        const int keys = ((max_len + want - 1) / want + 127) / 128 * 128, splits = (max_len + keys - 1) / keys;
        if (splits > most) continue;
        const long long ctas = items * splits;
        const double rounds = ctas <= 3 * places ? (double)((ctas + places - 1) / places) : (double)ctas / places + 0.5;
        const double cost = rounds * (keys + 500.0) + (splits > 1 ? join + 16.0 * (splits - 1) : 0.0);
        if (want == 1 || cost < best) {
            best = cost;
            *split_keys = keys;
            *n_splits = splits;
        }
        if (keys == 128) break;
    }
    return best;
}

// Splits, and who joins them, for CTAs of `hb` heads.
static void a4_plan(A4Launch& L, int hb, size_t room) {
    const tenzo_attention_kv4_args& a = L.a;
    L.head_blocks = (L.group + hb - 1) / hb;
    L.cluster = 0;
    if (a.split_keys > 0) {
        const long long keys = ((long long)a.split_keys + 127) / 128 * 128, all = ((long long)a.max_len + 127) / 128 * 128;
        L.split_keys = (int)(keys < all ? keys : all);
        L.n_splits = (a.max_len + L.split_keys - 1) / L.split_keys;
        return;
    }
    const long long items = (long long)a.rows * a.cache.n_kv * L.head_blocks;
    const double apart = a4_pick_split(items, a.max_len, room > 1 ? (int)(room < kA4MostSplits ? room : kA4MostSplits) : 1, 300.0, &L.n_splits, &L.split_keys);
    // Joined by clusters: 1 x 1000 keys 7.0 us and 9.2 by a second kernel, 12 x 8192 of 40/5 heads 36.3 and 38.1; but where CTAs come in several rounds
    // a cluster waits for room for all of its own (256 x 4095 ragged: 218 and 174).
    int splits, keys;
    if (a4_pick_split(items, a.max_len, kA4Cluster, 100.0, &splits, &keys) < apart && splits > 1 && items * splits <= 148 * kA4Resident) {
        L.n_splits = splits;
        L.split_keys = keys;
        L.cluster = 1;
    }
}

template <int HB>
static int a4_run(const A4Launch& L, cudaStream_t st) {
    const size_t smem = (size_t)kA4Warps * kA4Stages * kA4StepBytes;
    static_assert(kA4Warps * HB * kA4Hd * 4 + HB * (kA4Hd + 2) * 4 <= kA4Warps * kA4Stages * kA4StepBytes, "outputs where the rings were");
    if (cudaError_t e = allow_smem(attention_kv4_kernel<HB>, smem)) return (int)e;
    const dim3 grid((unsigned)L.a.rows * (unsigned)L.n_splits, (unsigned)(L.a.cache.n_kv * L.head_blocks));
    return kv4_launch_cluster(attention_kv4_kernel<HB>, grid, kA4Threads, L.cluster ? L.n_splits : 1, smem, st, L.a.use_pdl != 0, L);
}

int* kv4_rows_flags();
__global__ void kv4_clear_flags_kernel(int* rows, int rows_seen, int* attention, int attention_seen) {
    atomicAnd(rows, ~rows_seen);
    atomicAnd(attention, ~attention_seen);
}

}  // namespace tz

extern "C" size_t tenzo_cuda_attention_kv4_workspace_bytes(int rows, int n_q, int n_kv, int max_len) {
    if (rows <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_len <= 0) return 0;
    const size_t splits = ((size_t)max_len + 127) / 128;     // the finest split that may be asked for
    return tz::a4_part_bytes(rows, n_q) * splits;
}

extern "C" int tenzo_cuda_attention_kv4_splits(int rows, int n_q, int n_kv, int max_len) {
    using namespace tz;
    if (rows <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || n_q > 4 * 65535 || n_kv > 65535 || max_len <= 0 || max_len > 1 << 30) return 0;
    A4Launch L = {};
    L.a.rows = rows; L.a.n_q = n_q; L.a.cache.n_kv = n_kv; L.a.max_len = max_len;
    L.group = n_q / n_kv;
    int splits = 1;                                      // of the two plans that the call compares
    for (int hb = 4; hb <= (L.group > 4 ? 8 : 4); hb += 4) {
        a4_plan(L, hb, kA4MostSplits);
        if (!L.cluster && L.n_splits > splits) splits = L.n_splits;
    }
    return splits;
}

extern "C" int tenzo_cuda_attention_kv4(const tenzo_attention_kv4_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    A4Launch L = {};
    L.a = *args;
    tenzo_attention_kv4_args& a = L.a;
    if (a.rows == 0) return 0;
    if (!kv4_cache_ok(a.cache) || !a.q || !a.out || !a.pos) return -1;
    if (a.layer < 0 || a.layer >= a.cache.n_layers || a.n_q <= 0 || a.n_q % a.cache.n_kv || a.rows < 0 || a.max_len <= 0) return -1;
    if (a.max_len > (long long)a.cache.table_stride * kK4Slots || (!a.seq && a.rows > a.cache.table_rows)) return -1;
    if ((a.rope_cos == nullptr) != (a.rope_sin == nullptr) || (a.rope_cos && a.rope_len < a.max_len)) return -1;
    if (a.max_len > 1 << 30 || a.n_q > 4 * 65535) return -1;
    if (a.split_keys < 0 || (reinterpret_cast<uintptr_t>(a.out) & 15)) return -1;
    if (a.q_stride == 0) a.q_stride = a.n_q * kA4Hd;
    if (a.q_stride < a.n_q * kA4Hd) return -1;
    L.group = a.n_q / a.cache.n_kv;
    const bool ws_ok = a.workspace && !(reinterpret_cast<uintptr_t>(a.workspace) & 15);
    const size_t room = ws_ok ? a.workspace_bytes / a4_part_bytes(a.rows, a.n_q) : 0;
    // Heads a CTA takes: four, whose two parts of a weight share an MMA (64 x 8192 keys of 20/5 heads: 114 us, by eights 137); more than four heads a kv head by
    // eights, so that fewer CTAs copy and unpack a key (64 x 4096 of 40/5: 86 us, by fours 118), unless by fours there are no more than two or three CTAs an
    // SM, where an eight's longer way counts (1 x 1000 of 40/5: by fours 7.2 us, by eights 9.0; 4 x 1000: 9.4 and 10.2; but 16 x 1000: 16.9 and 15.0).
    int hb = 4;
    a4_plan(L, hb, room);
    if (L.group > 4 && (long long)a.rows * a.cache.n_kv * L.head_blocks * L.n_splits > 148 * 5 / 2) a4_plan(L, hb = 8, room);
    if (a.split_keys > 0 && L.n_splits > 1 && room < (size_t)L.n_splits) return -1;
    if ((long long)a.cache.n_kv * L.head_blocks > 65535) return -1;
    if ((long long)a.rows * L.n_splits > 0x7fffffffLL) return -1;
    L.part_o = static_cast<float*>(a.workspace);
    L.part_ml = reinterpret_cast<float2*>(L.part_o + (size_t)a.rows * a.n_q * L.n_splits * kA4Hd);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (int rc = hb == 4 ? a4_run<4>(L, st) : a4_run<8>(L, st)) return rc;
    if (L.n_splits == 1 || L.cluster) return 0;
    return kv4_launch(attention_kv4_merge_kernel, dim3((unsigned)a.rows, (unsigned)((a.n_q + kA4Warps - 1) / kA4Warps)), kA4Threads, 0, st, true, L);
}

// What runs on any stream is waited for, also on those that do not wait for the default one. Only bits that were seen are cleared: of what another thread's call raises
// meanwhile a bit is in the result or stays.
extern "C" int tenzo_cuda_kv4_take_errors(void) {
    using namespace tz;
    int *rows = kv4_rows_flags(), *attention = nullptr, r = 0, a = 0;
    if (!rows || cudaGetSymbolAddress(reinterpret_cast<void**>(&attention), g_kv4_attention_error) != cudaSuccess) return -1;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(&r, rows, sizeof r, cudaMemcpyDeviceToHost) != cudaSuccess ||
        cudaMemcpy(&a, attention, sizeof a, cudaMemcpyDeviceToHost) != cudaSuccess)
        return -1;
    if ((r | a) && (kv4_launch(kv4_clear_flags_kernel, dim3(1), 1, 0, cudaStreamLegacy, false, rows, r, attention, a) || cudaStreamSynchronize(cudaStreamLegacy) != cudaSuccess)) return -1;
    return r | a;
}
