// Rows of the 4-bit paged cache (kv4.cuh): appending them, reading them back, and handing the tables of parents on to the beams that
// continue them.
//
// A warp takes one kv head of one row (or of two), lanes 0-15 the key, 16-31 the value, dims 4l .. 4l + 3 and 64 more a lane: the pairs that the
// rotation turns lie in one lane, and every load and store is of whole sectors. Neighbouring warps take neighbouring heads. Every step is rounded to
// fp32 in the order the header gives (a code next to a border must not depend on who computes it); only the two parameters are
// rounded further, to fp16: at 32 dims a pair a third format of 32 bits would cost 10 % of the cache's bytes.
// 1024 bytes in and 160 out a row and head: 8 x 1000 ragged rows of 8 heads 20.6 us, 14 of which are the loads alone; the quantiser's 150 instructions a row are the rest, the
// stores cost nothing. (Registers for ten CTAs an SM: 20.6 us, as many as the compiler likes 21.3.) Read: 16.9 us, 0.6 of the memory's rate, nearly all of it stores.
#include "kv4.cuh"

#include <cuda_fp16.h>

namespace tz {

constexpr int kRowWarps = 4;                             // warps a CTA; a warp takes R consecutive rows of one kv head
constexpr float kFp16Most = 65504.0f;

__device__ int g_kv4_rows_error = 0;

struct RowsArgs {
    tenzo_kv4_cache c;
    int layer, rows, kv_stride, rope_len, use_pdl;
    const int *pos, *seq;
    const float *cs, *sn;
};

template <bool VEC>
__device__ __forceinline__ void load4(const float* p, float* x) {
    if (VEC) {
        const float4 v = ld_l2(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = ld_l2(p + j);
    }
}

// Lane r < R looks up the warp's r-th row: the position (-1: padding) and the table's entry are asked for at once, the place comes from them. Null for padding
// and for an index outside its range, which is flagged.
template <int R>
struct RowPlaces {
    const RowsArgs& a;
    int kvh, pos, block;
    __device__ __forceinline__ RowPlaces(const RowsArgs& args, int row0, int head, int rope_len) : a(args), kvh(head), pos(-1), block(-1) {
        const int lane = threadIdx.x & 31, row = row0 + lane;
        if (lane < R && row < a.rows) {
            pos = ld_l2(a.pos + row);
            const int seq = a.seq ? ld_l2(a.seq + row) : row;
            if (pos >= 0) {
                const bool there = seq >= 0 && seq < a.c.table_rows && pos / kK4Slots < a.c.table_stride && pos < rope_len;
                if (there) block = ld_l2(a.c.block_table + (size_t)seq * a.c.table_stride + pos / kK4Slots);
            }
        }
    }
    __device__ __forceinline__ int position(int r) const { return __shfl_sync(0xffffffffu, pos, r); }
    __device__ __forceinline__ uint8_t* finish(int r) const {
        const int p = __shfl_sync(0xffffffffu, pos, r), b = __shfl_sync(0xffffffffu, block, r);
        if (p < 0) return nullptr;
        if (b < 0 || b >= a.c.n_blocks) {
            if ((threadIdx.x & 31) == 0) atomicOr(&g_kv4_rows_error, kK4ErrIndex);
            return nullptr;
        }
        return a.c.pool + kv4_page(a.c, a.layer, kvh, b) + (size_t)(p % kK4Slots) * kK4Row;
    }
};

// The four codes of x, a nibble each.
__device__ __forceinline__ uint32_t row_codes(const float* x, float m, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w += __float_as_uint(fminf(fmaxf((x[j] - m) * inv, 0.0f), 15.0f) + 12582912.0f) << (4 * j);      // 1.5 2^23: nearest, ties to even
    return w & 0xffffu;
}

template <bool VEC, bool ROPE, int R>
__global__ void __launch_bounds__(kRowWarps * 32, 10) kv4_append_kernel(const RowsArgs a, const float* k, const float* v) {
    const int lane = threadIdx.x & 31, unit = blockIdx.x * kRowWarps + (threadIdx.x >> 5), kvh = unit % a.c.n_kv, row0 = unit / a.c.n_kv * R;
    const int is_v = lane >> 4, l = lane & 15;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    if (row0 >= a.rows) return;
    const RowPlaces<R> places(a, row0, kvh, ROPE ? a.rope_len : 0x7fffffff);
    float x[R][8], c[R][4], s[R][4];                     // dims 4l .. 4l + 3, and 64 more
#pragma unroll
    for (int r = 0; r < R; ++r) {                        // (padding rows are there to be read too)
        if (row0 + r < a.rows) {
            const float* p = (is_v ? v : k) + (size_t)(row0 + r) * a.kv_stride + kvh * 128 + 4 * l;
            load4<VEC>(p, x[r]);
            load4<VEC>(p + 64, x[r] + 4);
        }
    }
    if (ROPE) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int pos = places.position(r);
            if (!is_v && pos >= 0 && pos < a.rope_len) {
                load4<VEC>(a.cs + (size_t)pos * 64 + 4 * l, c[r]);
                load4<VEC>(a.sn + (size_t)pos * 64 + 4 * l, s[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        uint8_t* at = places.finish(r);
        if (!at) continue;                               // the whole warp
        if (ROPE && !is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = x[r][j], q = x[r][4 + j];
                x[r][j] = __fmaf_rn(p, c[r][j], -(q * s[r][j]));
                x[r][4 + j] = __fmaf_rn(p, s[r][j], q * c[r][j]);
            }
        }
        // Group l / 8 of the first 64 dims and of the others: lanes with an even l gather the first's minimum and maximum, the others
        // the second's. (Clamped afterwards: what lies outside gets the first or the last code all the same.)
        const bool odd = l & 1;
        const float lo_a = fminf(fminf(x[r][0], x[r][1]), fminf(x[r][2], x[r][3])), hi_a = fmaxf(fmaxf(x[r][0], x[r][1]), fmaxf(x[r][2], x[r][3]));
        const float lo_b = fminf(fminf(x[r][4], x[r][5]), fminf(x[r][6], x[r][7])), hi_b = fmaxf(fmaxf(x[r][4], x[r][5]), fmaxf(x[r][6], x[r][7]));
        float lo = fminf(odd ? lo_b : lo_a, __shfl_xor_sync(0xffffffffu, odd ? lo_a : lo_b, 1));
        float hi = fmaxf(odd ? hi_b : hi_a, __shfl_xor_sync(0xffffffffu, odd ? hi_a : hi_b, 1));
#pragma unroll
        for (int o = 2; o < 8; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        lo = fminf(fmaxf(lo, -kFp16Most), kFp16Most);
        hi = fminf(fmaxf(hi, -kFp16Most), kFp16Most);
        const __half low = __float2half_rn(lo), scale = __float2half_rn((hi - __half2float(low)) * (1.0f / 15.0f));
        const float m = __half2float(low), step = __half2float(scale), inv = step > 0.0f ? 1.0f / step : 0.0f;
        const float m2 = __shfl_xor_sync(0xffffffffu, m, 1), inv2 = __shfl_xor_sync(0xffffffffu, inv, 1);     // the other group's
        at += is_v * kK4Half;
        reinterpret_cast<unsigned short*>(at)[l] = (unsigned short)row_codes(x[r], odd ? m2 : m, odd ? inv2 : inv);
        reinterpret_cast<unsigned short*>(at + 32)[l] = (unsigned short)row_codes(x[r] + 4, odd ? m : m2, odd ? inv : inv2);
        if ((l & 6) == 0) reinterpret_cast<__half2*>(at + kK4Codes)[2 * odd + (l >> 3)] = __halves2half2(scale, low);
    }
}

template <bool VEC, int R>
__global__ void __launch_bounds__(kRowWarps * 32) kv4_read_kernel(const RowsArgs a, float* k, float* v) {
    const int lane = threadIdx.x & 31, unit = blockIdx.x * kRowWarps + (threadIdx.x >> 5), kvh = unit % a.c.n_kv, row0 = unit / a.c.n_kv * R;
    const int is_v = lane >> 4, l = lane & 15;
    if (a.use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    if (row0 >= a.rows) return;
    const RowPlaces<R> places(a, row0, kvh, 0x7fffffff);
    uint32_t word[R][2], pair[R][2];                     // of dims 4l .. 4l + 3, and 64 more
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint8_t* at = places.finish(r);
        word[r][0] = word[r][1] = pair[r][0] = pair[r][1] = 0;
        if (at) {
            at += is_v * kK4Half;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                word[r][h] = ld_l2(reinterpret_cast<const unsigned short*>(at + 32 * h) + l);
                pair[r][h] = ld_l2(reinterpret_cast<const uint32_t*>(at + kK4Codes) + 2 * h + (l >> 3));
            }
        }
    }
    float* to = is_v ? v : k;
    if (!to) return;
    to += (size_t)row0 * a.kv_stride + kvh * 128 + 4 * l;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (row0 + r >= a.rows) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&pair[r][h]));
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = p.y + p.x * (float)((word[r][h] >> (4 * j)) & 15u);
            float* out = to + (size_t)r * a.kv_stride + 64 * h;
            if (VEC) {
                *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] = x[j];
            }
        }
    }
}

// ---- the tables of the beams after a selection ---------------------------------------------------------------------------
// A group's beams all hold `length` tokens. Full blocks are shared, so a table row is its parent's; the block being filled is every
// beam's own: the first child keeps its parent's, a further one gets that of a beam without children and the filled rows are copied
// into it. Nothing is read that this launch writes: sources have children, targets have none, and the tables are two.
// CTA (x, y): part y of all that group x copies, and every gridDim.y-th of its table rows: each CTA has its share of the work, and the chain of length, parents
// and table entries in front of it is waited for once (64 x 8 beams: 20.5 us with CTAs a beam, two thirds of which found nothing to copy, 16.7 now).
// Bound by memory: length % 16 rows of 80 bytes, layers x heads x 2 times, in and out.
constexpr int kReorderThreads = 256, kReorderBatch = 8;  // 16-byte loads in flight a thread

__global__ void __launch_bounds__(kReorderThreads) kv4_reorder_kernel(const tenzo_kv4_cache c, int* table_out, const int* parent, const int* length, int beams,
                                                                      int use_pdl) {
    const int g = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (use_pdl) {
        pdl_launch_dependents();
        pdl_wait();
    }
    const int* rows = c.block_table + (size_t)g * beams * c.table_stride;      // the group's
    const bool mine = lane < beams;
    const int len = ld_l2(length + g);
    int p = mine ? ld_l2(parent + (size_t)g * beams + lane) : lane;
    const int col = len / kK4Slots, filled = len < 0 ? 0 : len % kK4Slots;
    const bool bad = (mine && (p < 0 || p >= beams)) || len < 0 || col + (filled > 0) > c.table_stride;
    const bool refused = __any_sync(0xffffffffu, bad);
    if (refused) {                                       // the group stays as it is
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(&g_kv4_rows_error, kK4ErrIndex);
        p = lane;
    }
    const unsigned all = beams == 32 ? 0xffffffffu : (1u << beams) - 1u;
    const unsigned alike = __match_any_sync(0xffffffffu, p) & all, below = (1u << lane) - 1u;
    unsigned further = __ballot_sync(0xffffffffu, mine && (alike & below));
    const unsigned childless = all & ~__reduce_or_sync(0xffffffffu, mine ? 1u << p : 0u);
    if (filled == 0) further = 0;                        // there is no block being filled
    int giver = filled > 0 ? p : lane;                   // whose block lane's beam goes on filling
    if ((further >> lane) & 1u) {                        // the n-th further child gets the n-th beam's without children; there are as many
        unsigned left = childless;
        for (int n = __popc(further & below); n > 0; --n) left &= left - 1u;
        giver = __ffs((int)left) - 1;
    }
    // Every warp has all of this. The tables, a warp a row:
    for (int i = blockIdx.y * (kReorderThreads / 32) + warp; i < beams; i += gridDim.y * (kReorderThreads / 32)) {
        const int from = __shfl_sync(0xffffffffu, p, i), tail = __shfl_sync(0xffffffffu, giver, i);
        int* out = table_out + ((size_t)g * beams + i) * c.table_stride;
        for (int x = lane; x < c.table_stride; x += 32) out[x] = ld_l2(rows + (size_t)(refused ? i : x < col ? from : x == col ? tail : i) * c.table_stride + x);
    }
    if (!further) return;
    // The blocks: lane's copy, if its beam is a further child (-1: none, or an entry out of range).
    int source = -1, target = -1;
    if ((further >> lane) & 1u) {
        source = ld_l2(rows + (size_t)p * c.table_stride + col);
        target = ld_l2(rows + (size_t)giver * c.table_stride + col);
        if (source < 0 || source >= c.n_blocks || target < 0 || target >= c.n_blocks) {
            if (warp == 0 && blockIdx.y == 0) atomicOr(&g_kv4_rows_error, kK4ErrIndex);
            source = -1;
        }
    }
    const unsigned halves = c.n_layers * c.n_kv * 2, units = filled * (kK4Row / 16), total = halves * units;       // 16-byte units of a half page, and of a block
    const unsigned by_units = 0xffffffffu / units + 1u;  // i / units for i below 2^32 / units
    constexpr unsigned kUnits = kK4Half / 16;
    const unsigned step = gridDim.y * kReorderThreads;
    for (; further; further &= further - 1u) {
        const int i = __ffs((int)further) - 1, s = __shfl_sync(0xffffffffu, source, i), t = __shfl_sync(0xffffffffu, target, i);
        if (s < 0) continue;
        const uint4* src = reinterpret_cast<const uint4*>(c.pool + (size_t)s * halves * kK4Half);
        uint4* dst = reinterpret_cast<uint4*>(c.pool + (size_t)t * halves * kK4Half);
        for (unsigned u0 = blockIdx.y * kReorderThreads + threadIdx.x; u0 < total; u0 += kReorderBatch * step) {
            uint4 w[kReorderBatch];
            size_t at[kReorderBatch];
#pragma unroll
            for (int n = 0; n < kReorderBatch; ++n) {
                const unsigned u = u0 + n * step, h = __umulhi(u, by_units);
                at[n] = (size_t)h * kUnits + (u - h * units);
                if (u < total) w[n] = ld_l2(src + at[n]);
            }
#pragma unroll
            for (int n = 0; n < kReorderBatch; ++n)
                if (u0 + n * step < total) dst[at[n]] = w[n];
        }
    }
}

static bool aligned16(const void* p) { return !(reinterpret_cast<uintptr_t>(p) & 15); }

static bool rows_args(const tenzo_kv4_cache* cache, int layer, int kv_stride, const int* pos, const int* seq, int rows, RowsArgs* a) {
    if (!cache || !kv4_cache_ok(*cache) || layer < 0 || layer >= cache->n_layers || !pos || rows < 1 || (long long)rows * cache->n_kv > 0x7fffffffLL) return false;
    if (kv_stride < cache->n_kv * 128LL) return false;
    if (!seq && rows > cache->table_rows) return false;
    a->c = *cache;
    a->layer = layer; a->rows = rows; a->kv_stride = kv_stride; a->pos = pos; a->seq = seq;
    return true;
}

// Rows a warp takes: two (their loads are in flight together) where that leaves every SM 32 warps, else one. Rows x heads by ones and by twos, over more than L2 holds, us:
//            1537 x 5    1184 x 8    1600 x 8     3200 x 8     8000 x 8     20000 x 8
//   append   5.5, 5.6    6.5, 6.0    7.2, 7.8    11.1, 11.3   23.0, 22.2   53.8, 50.6
//   read     5.4, 4.9    6.3, 5.5    6.7, 5.9    10.1, 8.7    22.0, 17.3   53.4, 38.9
// Reads gain on either side of the border, 9472; appends lose a little in places up to some 40000 and gain above.
static int rows_a_warp(int rows, int n_kv) { return (long long)rows * n_kv >= 4LL * 148 * 16 ? 2 : 1; }
static dim3 rows_grid(int rows, int n_kv, int r) { return dim3((unsigned)((((long long)rows + r - 1) / r * n_kv + kRowWarps - 1) / kRowWarps)); }

int* kv4_rows_flags() {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, g_kv4_rows_error) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

}  // namespace tz

extern "C" int tenzo_cuda_kv4_append(const tenzo_kv4_cache* cache, int layer, const float* k, const float* v, int kv_stride, const int* pos, const int* seq,
                                     int rows, const float* rope_cos, const float* rope_sin, int rope_len, int use_pdl, void* stream) {
    using namespace tz;
    RowsArgs a = {};
    if (rows == 0) return 0;
    if (!rows_args(cache, layer, kv_stride, pos, seq, rows, &a) || !k || !v) return -1;
    if ((rope_cos == nullptr) != (rope_sin == nullptr) || (rope_cos && rope_len <= 0)) return -1;
    a.cs = rope_cos; a.sn = rope_sin; a.rope_len = rope_len; a.use_pdl = use_pdl != 0;
    const bool vec = aligned16(k) && aligned16(v) && kv_stride % 4 == 0 && aligned16(rope_cos) && aligned16(rope_sin);
    const int r = rows_a_warp(rows, cache->n_kv);
    auto* kernel = r == 1 ? (rope_cos ? (vec ? kv4_append_kernel<true, true, 1> : kv4_append_kernel<false, true, 1>) : (vec ? kv4_append_kernel<true, false, 1> : kv4_append_kernel<false, false, 1>))
                          : (rope_cos ? (vec ? kv4_append_kernel<true, true, 2> : kv4_append_kernel<false, true, 2>) : (vec ? kv4_append_kernel<true, false, 2> : kv4_append_kernel<false, false, 2>));
    return kv4_launch(kernel, rows_grid(rows, cache->n_kv, r), kRowWarps * 32, 0, static_cast<cudaStream_t>(stream), a.use_pdl, a, k, v);
}

extern "C" int tenzo_cuda_kv4_read(const tenzo_kv4_cache* cache, int layer, float* k, float* v, int kv_stride, const int* pos, const int* seq, int rows,
                                   int use_pdl, void* stream) {
    using namespace tz;
    RowsArgs a = {};
    if (rows == 0) return 0;
    if (!rows_args(cache, layer, kv_stride, pos, seq, rows, &a) || (!k && !v)) return -1;
    a.use_pdl = use_pdl != 0;
    const bool vec = aligned16(k) && aligned16(v) && kv_stride % 4 == 0;
    const int r = rows_a_warp(rows, cache->n_kv);
    auto* kernel = r == 1 ? (vec ? kv4_read_kernel<true, 1> : kv4_read_kernel<false, 1>) : (vec ? kv4_read_kernel<true, 2> : kv4_read_kernel<false, 2>);
    return kv4_launch(kernel, rows_grid(rows, cache->n_kv, r), kRowWarps * 32, 0, static_cast<cudaStream_t>(stream), a.use_pdl, a, k, v);
}

extern "C" int tenzo_cuda_kv4_reorder(const tenzo_kv4_cache* cache, int* table_out, const int* parent, const int* length, int groups, int beams, int use_pdl,
                                      void* stream) {
    using namespace tz;
    if (!cache || !kv4_cache_ok(*cache) || !table_out || !parent || !length || groups < 1) return -1;
    if (beams < 1 || beams > TENZO_BEAMS_MOST) return -5;
    if ((long long)groups * beams != cache->table_rows) return -1;
    const uintptr_t from = reinterpret_cast<uintptr_t>(cache->block_table), to = reinterpret_cast<uintptr_t>(table_out), apart = from < to ? to - from : from - to;
    if (apart < (size_t)cache->table_rows * cache->table_stride * sizeof(int)) return -1;           // a row would be read after another had been written over it
    if ((long long)cache->n_layers * cache->n_kv > 16384) return -5;          // (a block's 16-byte units are numbered in 32 bits, and divided by multiplication)
    // Parts of a group: six CTAs an SM in all (64 x 8 beams: 2 an SM 20.1 us, 3 18.2, 6 16.7, 16 16.6), and a batch of loads each at the most.
    const long long units = (long long)cache->n_layers * cache->n_kv * 2 * (kK4Half / 16), most = (units + kReorderThreads * kReorderBatch - 1) / (kReorderThreads * kReorderBatch);
    long long parts = 6 * 148 / groups;
    parts = parts < 1 ? 1 : parts > most ? most : parts;
    return kv4_launch(kv4_reorder_kernel, dim3((unsigned)groups, (unsigned)parts), kReorderThreads, 0, static_cast<cudaStream_t>(stream), use_pdl != 0, *cache, table_out, parent,
                      length, beams, use_pdl != 0);
}
