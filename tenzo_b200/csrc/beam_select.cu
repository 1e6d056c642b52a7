// The k best continuations of a group of beams over beams x vocabulary.
//
// score(beam, token) = cum[beam] + (x - log sum exp x), in 64 bits: sums of log-probabilities lie close together between beams, and in 32
// bits each score would be rounded by itself, to steps of 2e-6 at -20 and of 2e-3 at -30000. Only exponentials have fewer bits (below): their error is one number a row, which moves its
// tokens together, by some 1e-8. Within a row the order is that of the logits. Two kernels:
//
//   1. A CTA takes a chunk of a row, each thread up to 32 logits in registers, read once. The k-th largest of the 256 threads' maxima is a
//      lower bound of the chunk's k-th largest logit, and hardly more logits reach it: those are listed, and their exponentials are taken and summed
//      in 64 bits. All others' (16 larger ones at least are on the list) are taken in 32, by the hardware's 2^x, and summed in 32 within a thread:
//      nothing is lost where a few tokens have the weight, and where thousands share it the errors hardly add up: the logarithm of the whole was off by some 1e-8
//      in random rows, by up to 1e-7 with logits that repeat, and cannot be by more than 2e-6. (An own 2^x good to 1e-8 costs thirteen instructions a logit
//      where there are two now.)
//   2. A CTA a group, a warp a row: the k best of the lists, with their scores; then the rows' scores that reach a common border are ranked
//      among one another.
// Sums are taken in an order that the data alone decides, or as integers, so that equal rows get equal sums and tie.
//
// 32 x 8 rows of 128256, k 16: 36 us. Loads alone take the first kernel 21 (131 MB at 6.2 TB/s), with everything else in it 29: some eight instructions and an ex2 a
// logit, and the barriers around the bisection, are hidden by the other CTAs' loads for two thirds only. The second kernel is 7, a chain of some 10 000 cycles.
#include "common.cuh"
#include "kv4.cuh"

#include <cfloat>

namespace tz {

constexpr int kBsThreads = 256, kBsWarps = kBsThreads / 32;
constexpr int kBsLeast = 16;                              // at least so many candidates are asked for in a chunk
constexpr int kBsWindow = 8;                              // and up to so many threads more are let in
constexpr int kBsMostK = 2 * TENZO_BEAMS_MOST;
constexpr int kBsMostPer = 32;                            // logits a thread holds at most
constexpr int kBsList = (kBsMostK + kBsWindow) * kBsMostPer;      // candidates lie in that many threads' logits
constexpr int kBsAhead = 148;                            // CTAs ahead whose logits are asked for into L2: one an SM
constexpr int kBsMergeWarps = 16;                         // rows that the second kernel merges at a time
constexpr int kBsHold = 1280;                             // entries of a row's lists that a warp keeps: 16 chunks of the most slots
constexpr int kBsPicks = 96;                              // entries that are ranked; more than k + kBsWindow

constexpr double kBsUnit = 281474976710656.0;             // 2^48
constexpr double kBsUnitOthers = 35184372088832.0;        // 2^45
constexpr float kLog2E = 1.4426950408889634f;

typedef unsigned long long u64;

// Order of the floats as integers above 0 (0: nothing there), and -0 as +0.
__device__ __forceinline__ uint32_t beam_key(float f) {
    const uint32_t b = f == 0.0f ? 0u : __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float beam_unkey(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ u64 beam_entry(uint32_t key, int token) { return ((u64)key << 32) | (uint32_t)~token; }      // larger key, then lower token
__device__ __forceinline__ int entry_token(u64 e) { return (int)~(uint32_t)e; }
__device__ __forceinline__ float entry_logit(u64 e) { return beam_unkey((uint32_t)(e >> 32)); }

struct __align__(16) BeamPart {                           // of a chunk
    double sum;                                           // of exp(x - most)
    float most;
};
struct BeamLaunch {
    tenzo_beam_select_args a;
    int per, chunks, slots;                               // logits a thread takes, chunks a row, entries a chunk's list has room for
    BeamPart* parts;                                      // [row][chunk]
    u64* lists;                                           // [row][chunk][slots], in any order; 0 where there is none
};

// Rows that the first kernel leaves out: finished beams, and those whose score is -infinity (or NaN).
__device__ __forceinline__ bool beam_dead(float cum) { return !(cum > -INFINITY); }
__device__ __forceinline__ bool beam_finished(const tenzo_beam_select_args& a, int row) { return a.finished && ld_l2(a.finished + row) != 0; }

// EAGER: few CTAs, so that time counts and not the bytes of rows that are left out.
template <bool VEC, int PER, bool EAGER>
__global__ void __launch_bounds__(kBsThreads, 4) beam_rows_kernel(const BeamLaunch L) {
    __shared__ uint32_t s_keys[kBsThreads];
    __shared__ u64 s_list[kBsList], s_sum[kBsWarps], s_listed[kBsWarps];
    __shared__ double s_unit;
    __shared__ float s_red[kBsWarps];
    __shared__ uint32_t s_bound;
    __shared__ int s_short, s_last, s_n;
    const tenzo_beam_select_args& a = L.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / L.chunks, chunk = blockIdx.x % L.chunks;
    pdl_launch_dependents();                              // the second kernel waits for this one, whatever its neighbours do
    if (a.use_pdl) pdl_wait();
    const float cum = ld_l2(a.scores + row);
    const bool out = beam_finished(a, row) || beam_dead(cum);
    if (!EAGER && out) return;                            // (eager: the logits are asked for meanwhile)
    const float* x = a.logits + (size_t)row * a.row_stride;
    const int base = chunk * kBsThreads * PER;
    // place of the j-th logit of a thread: consecutive fours (or ones) go to consecutive threads
    auto place = [&](int j) { return base + (VEC ? 4 * (tid + kBsThreads * (j >> 2)) + (j & 3) : tid + kBsThreads * j); };
    static_assert(PER <= 32, "one bit each");
    float v[PER];                                         // -infinity where there is nothing
    if (VEC && base + kBsThreads * PER <= a.vocab) {
        const float4* from = reinterpret_cast<const float4*>(x + base) + tid;
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            const float4 f = ld_l2(from + kBsThreads * (j >> 2));
            v[j] = f.x; v[j + 1] = f.y; v[j + 2] = f.z; v[j + 3] = f.w;
        }
    } else if (VEC) {
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            const int i = place(j);
            if (i + 3 < a.vocab) {
                f = ld_l2(reinterpret_cast<const float4*>(x + i));
            } else {
                if (i < a.vocab) f.x = ld_l2(x + i);
                if (i + 1 < a.vocab) f.y = ld_l2(x + i + 1);
                if (i + 2 < a.vocab) f.z = ld_l2(x + i + 2);
            }
            v[j] = f.x; v[j + 1] = f.y; v[j + 2] = f.z; v[j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = place(j) < a.vocab ? ld_l2(x + place(j)) : -INFINITY;
    }
    if (out) return;
    if (tid == 0) {
        s_n = 0;
        // Where CTAs come in waves, the logits of a later one on their way to L2 meanwhile (32 x 8 rows of 128256: 43.8 us without, 42.2 one CTA an SM ahead, 42.9 four)
        if (VEC && !EAGER && blockIdx.x + kBsAhead < gridDim.x) {
            const int r = (blockIdx.x + kBsAhead) / L.chunks, at = (blockIdx.x + kBsAhead) % L.chunks * kBsThreads * PER, n = min(a.vocab - at, kBsThreads * PER) & ~3;
            if (n > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.logits + (size_t)r * a.row_stride + at), "r"(4 * n) : "memory");
        }
    }
    // ---- what counts: NaN as -infinity (below), infinity as the largest number; the largest of all ------------------------------
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = fmaxf(top, v[j]); // (drops NaN)
    if (top == INFINITY) {
        top = FLT_MAX;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = fminf(fmaxf(v[j], -INFINITY), FLT_MAX);
    }
    s_keys[tid] = place(0) < a.vocab ? beam_key(top) : 0u;
    float most = warp_max(top);
    if (lane == 0) s_red[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBsWarps; ++w) most = fmaxf(most, s_red[w]);
    // ---- a bound that `want` threads' maxima reach, and hardly more -------------------------------------------------------------
    const int want = max(a.k, kBsLeast);
    auto at_least = [&](const uint32_t (&key)[kBsWarps], uint32_t b) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < kBsWarps; ++w) n += key[w] >= b;
        return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
    };
    if (warp == 0) {
        uint32_t key[kBsWarps], least = 0xffffffffu;
#pragma unroll
        for (int w = 0; w < kBsWarps; ++w) {
            key[w] = s_keys[32 * w + lane];
            least = min(least, key[w]);
        }
        uint32_t lo = __reduce_min_sync(0xffffffffu, least), hi = beam_key(most) + 1;       // all reach lo, none hi
        int reach = kBsThreads;
        while (reach > want + kBsWindow && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int n = at_least(key, mid);
            if (n >= want) { lo = mid; reach = n; } else hi = mid;
        }
        const int above = reach > want + kBsWindow ? at_least(key, hi) : 0;
        if (lane == 0) {
            s_bound = lo;
            s_short = lo > 0 && reach > want + kBsWindow ? want - above : 0;      // too many alike: so many of them, by index
            s_last = 0x7fffffff;
        }
    }
    __syncthreads();
    const float bound = s_bound <= beam_key(-INFINITY) ? -INFINITY : beam_unkey(s_bound);      // (no float below that one: all that is there is listed)
    if (s_short) {                                        // the first place of each thread's largest, then a place that enough of them reach
        int first = 0x7fffffff;
        if (s_keys[tid] == s_bound) {
#pragma unroll
            for (int j = PER - 1; j >= 0; --j)
                if (v[j] == bound && place(j) < a.vocab) first = place(j);
            if (bound == -INFINITY) first = place(0);     // (nothing but masks in these threads, and NaN is one: found by == or not)
        }
        __syncthreads();
        s_keys[tid] = (uint32_t)first;
        __syncthreads();
        if (warp == 0) {
            uint32_t key[kBsWarps];
#pragma unroll
            for (int w = 0; w < kBsWarps; ++w) key[w] = ~s_keys[32 * w + lane];
            uint32_t lo = ~(uint32_t)(base + kBsThreads * PER), hi = ~(uint32_t)base + 1u;     // (complements: a lower place is a larger key)
            int reach = at_least(key, lo);
            while (reach > s_short + kBsWindow && hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                const int n = at_least(key, mid);
                if (n >= s_short) { lo = mid; reach = n; } else hi = mid;
            }
            if (lane == 0) s_last = (int)~lo;
        }
        __syncthreads();
    }
    const int last = s_last;
    // ---- the others' exponentials, and the list of candidates -------------------------------------------------------------------
    // 2^(v log2(e) - shift) with one rounding: `shift` is most * log2(e), rounded, and what that rounding does to all of them alike is put right in the end. (log2(e) in
    // 24 bits is 1.3e-8 off.) That rounding is 2^-9 at most up to 32768; beyond, and where masked rows have the lowest number of all, the difference comes first.
    const float from = most == -INFINITY ? 0.0f : most, shift = -from * kLog2E;
    const bool far = !(fabsf(from) < 32768.0f);
    auto power = [&](float c, bool difference_first) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(difference_first ? (c - from) * kLog2E : __fmaf_rn(c, kLog2E, shift)));
        return e;
    };
    float rest = 0.0f;
    uint32_t reach_it = 0;                                // one bit a logit
    if (!far) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float e = power(v[j], false);
            if (v[j] >= bound) reach_it |= 1u << j; else rest += e;
        }
    }
    if (far || rest != rest) {                            // a NaN among them
        rest = 0.0f;
        reach_it = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            v[j] = fmaxf(v[j], -INFINITY);
            const float e = power(v[j], far);
            if (v[j] >= bound) reach_it |= 1u << j; else rest += e;
        }
    }
    for (const bool one = (reach_it & (reach_it - 1u)) == 0u; reach_it; reach_it &= reach_it - 1u) {
        const int i = place(__ffs((int)reach_it) - 1);
        if (i >= a.vocab) continue;
        float c = top;
        if (!one) {                                       // (a register's number is no variable)
            const int at = __ffs((int)reach_it) - 1;
#pragma unroll
            for (int j = 0; j < PER; ++j) c = j == at ? v[j] : c;
        }
        if (c == bound && i > last) {
            rest += power(c, far);
        } else {
            const int at = atomicAdd(&s_n, 1);
            if (at < kBsList) s_list[at] = beam_entry(beam_key(c), i);
        }
    }
    // Sums as whole numbers: up to 32 a thread, in units of 2^-21 and 2^-45, add up in two instructions a warp.
    const float units = rest * 2097152.0f, whole = floorf(units);
    const unsigned high = __reduce_add_sync(0xffffffffu, (unsigned)whole), low = __reduce_add_sync(0xffffffffu, (unsigned)((units - whole) * 16777216.0f));
    if (lane == 0) s_sum[warp] = ((u64)high << 24) + low;
    __syncthreads();
    const int n = min(s_n, kBsList);
    u64* to = L.lists + ((size_t)row * L.chunks + chunk) * L.slots;
    const bool few = n <= L.slots;
    if (few) {
        if (tid < L.slots) to[tid] = tid < n ? s_list[tid] : 0ull;
    } else {                                              // (many large ones in few threads) the best k go on
        for (int i = tid; i < n; i += kBsThreads) {
            const u64 e = s_list[i];
            int before = 0;
            for (int j = 0; j < n; ++j) before += s_list[j] > e;
            if (before < a.k) to[before] = e;
        }
        if (tid >= a.k && tid < L.slots) to[tid] = 0ull;
    }
    if (few && warp > 0) return;
    // The listed ones' exponentials, in units of 2^-48 (whole numbers add up the same in any order), by one warp or by all; and, as one more, the unit of the others.
    u64 mine = 0;
    double unit = 1.0;
    const double off = far ? 0.0 : (double)from * (double)kLog2E + (double)shift;      // (the product is exact)
#pragma unroll 1
    for (int i = tid; i <= n; i += few ? 32 : kBsThreads) {
        const double e = exp(i < n ? (double)entry_logit(s_list[i]) - (double)from : off * -0.69314718055994531);
        if (i == n) unit = e;
        else if (most > -INFINITY) mine += (u64)__double2ll_rn(e * kBsUnit);
    }
    const u64 listed = ((u64)__reduce_add_sync(0xffffffffu, (unsigned)(mine >> 26)) << 26) + __reduce_add_sync(0xffffffffu, (unsigned)mine & 0x3ffffffu);
    if (few) {
        unit = __shfl_sync(0xffffffffu, unit, n & 31);
    } else {
        if (tid == n % kBsThreads) s_unit = unit;
        if (lane == 0) s_listed[warp] = listed;
        __syncthreads();
        unit = s_unit;
    }
    if (tid == 0) {
        BeamPart p;
        u64 all = listed, others = 0;
#pragma unroll
        for (int w = 0; w < kBsWarps; ++w) others += s_sum[w];
        if (!few)
            for (int w = 1; w < kBsWarps; ++w) all += s_listed[w];
        p.sum = (double)all * (1.0 / kBsUnit) + (double)others * (unit / kBsUnitOthers);
        p.most = most;
        L.parts[(size_t)row * L.chunks + chunk] = p;
    }
}

// Order of the scores as integers, and back. (No score is NaN.)
__device__ __forceinline__ u64 score_key(double f) {
    const u64 b = f == 0.0 ? 0ull : (u64)__double_as_longlong(f);
    return (b >> 63) ? ~b : (b | 1ull << 63);
}
__device__ __forceinline__ double score_of(u64 k) { return __longlong_as_double((long long)((k >> 63) ? (k & ~(1ull << 63)) : ~k)); }

struct BeamGroup {
    u64 score[TENZO_BEAMS_MOST][kBsMostK];                // keys of a row's best, in order
    int token[TENZO_BEAMS_MOST][kBsMostK];
    int count[TENZO_BEAMS_MOST];
    u64 pick[kBsMergeWarps][kBsPicks];                    // what a warp found, unsorted
    u64 live[TENZO_BEAMS_MOST * kBsMostK];                // scores that may be among the group's best, and whose they are: 64 beam + place
    unsigned short whose[TENZO_BEAMS_MOST * kBsMostK];
    int n_live;
};

// Its loops are not unrolled further than their loads ask for: every instruction runs a few times only, and what runs once waits for its code (11 700 cycles at first, 10 200 when
// all of it is in the caches). Dynamic shared memory: the group, then `hold` entries a warp (0: the lists are longer and read from L2).
__global__ void __launch_bounds__(kBsMergeWarps * 32) beam_groups_kernel(const BeamLaunch L, const int hold) {
    extern __shared__ __align__(16) unsigned char bs_smem[];
    BeamGroup& G = *reinterpret_cast<BeamGroup*>(bs_smem);
    const tenzo_beam_select_args& a = L.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.x, k = a.k;
    u64* room = reinterpret_cast<u64*>(bs_smem + (sizeof(BeamGroup) + 15) / 16 * 16) + (size_t)warp * hold;
    pdl_launch_dependents();
    pdl_wait();
    if (tid == 0) G.n_live = 0;
#pragma unroll 1
    for (int b = warp; b < a.beams; b += kBsMergeWarps) {
        const int row = g * a.beams + b, most_tokens = min(k, a.vocab), n = L.chunks * L.slots;      // (an even number)
        const BeamPart* parts = L.parts + (size_t)row * L.chunks;
        const u64* list = L.lists + (size_t)row * n;
        const float cum = ld_l2(a.scores + row);
        const bool finished = beam_finished(a, row), done = finished && !beam_dead(cum);
        float first_most = -INFINITY;                     // of the lane's first chunk
        double first_sum = 0.0;
        if (lane < L.chunks) {
            first_most = ld_l2(&parts[lane].most);
            first_sum = ld_l2(&parts[lane].sum);
        }
        // the row's entries, and each lane's two largest logits (of a row that was left out they mean nothing)
        uint32_t one = 0, two = 0;
#pragma unroll 1
        for (int i0 = lane; i0 < n / 2; i0 += 8 * 32) {
            uint4 e[8];                                   // two entries each: token, logit, token, logit
#pragma unroll
            for (int u = 0; u < 8; ++u) e[u] = i0 + 32 * u < n / 2 ? ld_l2(reinterpret_cast<const uint4*>(list) + i0 + 32 * u) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (hold && i0 + 32 * u < n / 2) reinterpret_cast<uint4*>(room)[i0 + 32 * u] = e[u];
                two = max(two, min(one, e[u].y));
                one = max(one, e[u].y);
                two = max(two, min(one, e[u].w));
                one = max(one, e[u].w);
            }
        }
        const u64* entry = hold ? room : list;
        float most = -INFINITY;
        if (!finished && !beam_dead(cum)) {
            most = first_most;
#pragma unroll 1
            for (int c = lane + 32; c < L.chunks; c += 32) most = fmaxf(most, ld_l2(&parts[c].most));
            most = warp_max(most);
        }
        if (most == -INFINITY) {                          // finished, or nothing left: the lowest tokens at -infinity; in front of them a finished beam's end
            for (int i = lane; i < most_tokens; i += 32) {
                G.token[b][i] = !done ? i : i == 0 ? a.eos : i - 1 < a.eos ? i - 1 : i;
                G.score[b][i] = score_key(done && i == 0 ? (double)cum : -(double)INFINITY);
            }
            if (lane == 0) G.count[b] = most_tokens;
            continue;
        }
        double sum = 0.0;
#pragma unroll 1
        for (int c = lane; c < L.chunks; c += 32) {
            if (c >= 32) {
                first_most = ld_l2(&parts[c].most);
                first_sum = ld_l2(&parts[c].sum);
            }
            if (first_most > -INFINITY) sum += first_sum * exp((double)first_most - (double)most);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double lse = (double)most + log(sum);
        // ---- a bound that k of the lanes' two largest logits reach, and hardly more -------------------------------------------------
        u64 lo = 1, hi = ((u64)beam_key(most) + 1) << 32; // (0: nothing there)
        {
            auto at_least = [&](uint32_t x) { return __popc(__ballot_sync(0xffffffffu, one >= x)) + __popc(__ballot_sync(0xffffffffu, two >= x)); };
            uint32_t low = 1, high = beam_key(most) + 1;
            int reach = at_least(low);
            if (reach >= k) {                             // (else all there is)
                const uint32_t least = max(1u, __reduce_min_sync(0xffffffffu, k <= 32 ? one : two));
                if (at_least(least) >= k) low = least;
                reach = at_least(low);
#pragma unroll 1
                while (reach > k + kBsWindow && high - low > 1) {       // (in quarters: three counts take little longer than one)
                    const uint32_t half = low + (high - low) / 2, first = low + (half - low) / 2, third = half + (high - half) / 2;
                    const int m1 = at_least(first), m2 = at_least(half), m3 = at_least(third);
                    if (m3 >= k) { low = third; reach = m3; }
                    else if (m2 >= k) { low = half; reach = m2; high = third; }
                    else if (m1 >= k) { low = first; reach = m1; high = half; }
                    else high = first;
                }
                lo = (u64)low << 32;
            }
        }
        // ---- the entries that reach it; more than can be ranked (many alike, or in few lanes): the k-th of all, which differ -------
        __syncwarp();                                     // (the room)
        int m;
#pragma unroll 1
        for (;;) {
            int mine = 0;                                 // counted, and placed behind those of the lanes below
#pragma unroll 4
            for (int i = 2 * lane; i < n; i += 64) {      // two entries a load
                const ulonglong2 e = *reinterpret_cast<const ulonglong2*>(entry + i);
                mine += (e.x >= lo) + (e.y >= lo);
            }
            int at = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, at, o);
                if (lane >= o) at += other;
            }
            m = __shfl_sync(0xffffffffu, at, 31);
            at -= mine;
            if (m <= kBsPicks) {
#pragma unroll 4
                for (int i = 2 * lane; i < n; i += 64) {
                    const ulonglong2 e = *reinterpret_cast<const ulonglong2*>(entry + i);
                    if (e.x >= lo) G.pick[warp][at++] = e.x;
                    if (e.y >= lo) G.pick[warp][at++] = e.y;
                }
                break;
            }
#pragma unroll 1
            for (int reach = m; reach > kBsPicks && hi - lo > 1;) {
                const u64 mid = lo + (hi - lo) / 2;
                int c = 0;
#pragma unroll 4
                for (int i = lane; i < n; i += 32) c += entry[i] >= mid;
                c = (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
                if (c >= k) { lo = mid; reach = c; } else hi = mid;
            }
        }
        __syncwarp();
#pragma unroll 1
        for (int i = lane; i < m; i += 32) {
            const u64 e = G.pick[warp][i];
            int before = 0;
#pragma unroll 8
            for (int j = 0; j < m; ++j) before += G.pick[warp][j] > e;
            if (before < k) {
                const float x = entry_logit(e);
                G.token[b][before] = entry_token(e);
                G.score[b][before] = score_key(x == -INFINITY ? -(double)INFINITY : (double)cum + ((double)x - lse));
            }
        }
        if (lane == 0) G.count[b] = min(m, k);
        __syncwarp();
    }
    __syncthreads();
    // ---- a score that k entries reach: the worst of the rows' ceil(k / beams)-th, or the best of their k-th. What lies below is out. ----
    uint32_t worst = 0xffffffffu, best = 0, first = 0;    // (upper halves of the keys are enough)
    if (lane < a.beams) {
        const int each = (k + a.beams - 1) / a.beams, n = G.count[lane];
        worst = n >= each ? (uint32_t)(G.score[lane][each - 1] >> 32) : 0;
        first = n ? (uint32_t)(G.score[lane][0] >> 32) : 0;
        if (n >= k) best = (uint32_t)(G.score[lane][k - 1] >> 32);
    }
    worst = __reduce_min_sync(0xffffffffu, worst);
    best = __reduce_max_sync(0xffffffffu, best);
    first = __reduce_max_sync(0xffffffffu, first);
    u64 border = (u64)max(worst, best) << 32, high = ((u64)first + 1) << 32;
    // ... and closer to the k-th, by bisection over all (a place of the rows' lists a thread).
    auto place = [&](int i) { return i < a.beams * kBsMostK && i % kBsMostK < G.count[i / kBsMostK] ? G.score[i / kBsMostK][i % kBsMostK] : 0ull; };
    auto reaching = [&](u64 x) {
        int c = 0;
#pragma unroll 1
        for (int i0 = 0; i0 < a.beams * kBsMostK; i0 += kBsMergeWarps * 32) c += __syncthreads_count(place(i0 + tid) >= x);
        return c;
    };
    if (border == 0) border = 1;                          // (no score has the key 0)
    int reach = reaching(border);
#pragma unroll 1
    while (reach > k + 64 && high - border > 1) {       // (so many are ranked in less time than another step takes)
        const u64 mid = border + (high - border) / 2;
        const int c = reaching(mid);
        if (c >= k) { border = mid; reach = c; } else high = mid;
    }
#pragma unroll 1
    for (int i = tid; i < a.beams * kBsMostK; i += kBsMergeWarps * 32) {
        const u64 score = place(i);
        if (score >= border) {
            const int at = atomicAdd(&G.n_live, 1);
            G.live[at] = score;
            G.whose[at] = (unsigned short)i;
        }
    }
    __syncthreads();
    const int n = G.n_live;
#pragma unroll 1
    for (int i = tid; i < n; i += kBsMergeWarps * 32) {
        const u64 score = G.live[i];
        const int whose = G.whose[i];
        int before = 0;                                   // larger scores, and equal ones of lower beams, or in front in its own
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const u64 other = G.live[j];
            before += other > score;
            if (other == score) before += G.whose[j] < whose;
        }
        if (before < k) {
            const size_t to = (size_t)g * k + before;
            a.parent_out[to] = whose / kBsMostK;
            a.token_out[to] = G.token[whose / kBsMostK][whose % kBsMostK];
            a.score_out[to] = (float)score_of(score);
        }
    }
}

// Logits a thread takes: 32, or fewer where that would leave SMs without a CTA, as long as the second kernel's warps can keep a row's lists (1 x 4 beams: 10.7 us, where they do
// not 11.3; 8 x 32 beams with 64 candidates: 72.5 and 79.5).
static int beam_chunks(int per, int vocab) { return (int)(((long long)vocab + kBsThreads * per - 1) / (kBsThreads * per)); }
static int beam_slots(int k) { return ((k > kBsLeast ? k : kBsLeast) + 2 * kBsWindow + 1) / 2 * 2; }      // (even: they are read two at a time)
static int beam_per(int rows, int vocab, int k) {
    int per = kBsMostPer;
    while (per > 4 && (long long)rows * beam_chunks(per, vocab) < 128 && (long long)beam_chunks(per / 2, vocab) * beam_slots(k) <= kBsHold) per /= 2;
    return per;
}

static size_t beam_groups_smem(int hold) { return (sizeof(BeamGroup) + 15) / 16 * 16 + (size_t)kBsMergeWarps * hold * sizeof(u64); }
static_assert((sizeof(BeamGroup) + 15) / 16 * 16 + (size_t)kBsMergeWarps * kBsHold * sizeof(u64) <= kMaxSmem, "what an SM has");

// One wave of CTAs (logits of rows that are left out: 32 x 8 beams, one in ten finished: 37.9 us with them, 36.1 without).
static bool beam_eager(long long ctas) { return ctas <= 592; }

template <bool VEC, int PER, bool EAGER>
static int beam_rows_launch(const BeamLaunch& L, cudaStream_t st) {
    auto* kernel = beam_rows_kernel<VEC, PER, EAGER>;
    // Few CTAs: shared memory set up as the second kernel needs it, which otherwise waits until it is changed (5 x 12 rows of 50001: 15.7 us, 16.9 without). Many: as much of it for
    // loads on their way as there is (32 x 8 of 128256: 36.1 us, 39.4 otherwise). As with allow_smem every host thread sets the same for a kernel: one of its own for either.
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, EAGER ? cudaSharedmemCarveoutMaxShared : cudaSharedmemCarveoutDefault)) return (int)e;
    return kv4_launch(kernel, dim3((unsigned)(L.a.groups * L.a.beams) * (unsigned)L.chunks), kBsThreads, 0, st, L.a.use_pdl != 0, L);
}
template <bool VEC>
static int beam_rows_run(const BeamLaunch& L, cudaStream_t st) {
    if (!beam_eager((long long)L.a.groups * L.a.beams * L.chunks)) return beam_rows_launch<VEC, 32, false>(L, st);        // (fewer than 32 logits a thread: fewer than 256 CTAs)
    return L.per == 32 ? beam_rows_launch<VEC, 32, true>(L, st) : L.per == 16 ? beam_rows_launch<VEC, 16, true>(L, st) : L.per == 8 ? beam_rows_launch<VEC, 8, true>(L, st)
                                                                                                                                  : beam_rows_launch<VEC, 4, true>(L, st);
}

}  // namespace tz

extern "C" size_t tenzo_cuda_beam_select_workspace_bytes(int groups, int beams, int vocab, int k) {
    if (groups <= 0 || beams <= 0 || vocab <= 0 || k <= 0 || (long long)groups * beams > 0x7fffffffLL) return 0;
    const size_t chunks = (size_t)tz::beam_chunks(tz::beam_per(groups * beams, vocab, k), vocab);
    return (size_t)groups * beams * chunks * (sizeof(tz::BeamPart) + (size_t)tz::beam_slots(k) * sizeof(tz::u64));
}

extern "C" int tenzo_cuda_beam_select(const tenzo_beam_select_args* args, void* stream) {
    using namespace tz;
    if (!args) return -1;
    BeamLaunch L = {};
    L.a = *args;
    tenzo_beam_select_args& a = L.a;
    if (a.groups == 0) return 0;
    if (!a.logits || !a.scores || !a.parent_out || !a.token_out || !a.score_out || !a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 15)) return -1;
    if (a.groups < 0 || a.vocab <= 0 || a.beams < 1 || a.k < 1 || a.k > (long long)a.beams * a.vocab) return -1;
    if (a.finished && (a.eos < 0 || a.eos >= a.vocab)) return -1;
    if (a.beams > TENZO_BEAMS_MOST || a.k > kBsMostK) return -5;
    if (a.row_stride == 0) a.row_stride = a.vocab;
    if (a.row_stride < a.vocab) return -1;
    const long long rows = (long long)a.groups * a.beams;
    if (rows > 0x7fffffffLL) return -1;
    L.per = beam_per((int)rows, a.vocab, a.k);
    L.chunks = beam_chunks(L.per, a.vocab);
    L.slots = beam_slots(a.k);
    if (rows * L.chunks > 0x7fffffffLL || (long long)L.chunks * L.slots > 0x7fffffffLL || (long long)L.chunks * kBsThreads * L.per > 0x7fffffffLL) return -1;
    if (a.workspace_bytes < tenzo_cuda_beam_select_workspace_bytes(a.groups, a.beams, a.vocab, a.k)) return -1;
    L.parts = static_cast<BeamPart*>(a.workspace);
    L.lists = reinterpret_cast<u64*>(L.parts + (size_t)rows * L.chunks);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = !(reinterpret_cast<uintptr_t>(a.logits) & 15) && a.row_stride % 4 == 0;
    if (cudaError_t e = allow_smem(beam_groups_kernel, beam_groups_smem(kBsHold))) return (int)e;
    if (int rc = vec ? beam_rows_run<true>(L, st) : beam_rows_run<false>(L, st)) return rc;
    const int entries = L.chunks * L.slots, hold = entries <= kBsHold ? (entries + 1) / 2 * 2 : 0;
    return kv4_launch(beam_groups_kernel, dim3((unsigned)a.groups), kBsMergeWarps * 32, beam_groups_smem(hold), st, true, L, hold);
}
