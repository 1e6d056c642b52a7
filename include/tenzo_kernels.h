/* tenzo_kernels.h — flat C entry points, one per CUDA kernel of the quantized decode path.
 *
 * These are the device-pointer calls that sit underneath the engine ABI (tenzo.h) and the
 * tenzo::CUDARuntime backend class. Every pointer is a CUDA device pointer unless the name ends
 * in _host; `stream` is a cudaStream_t passed as void* (NULL = default stream). Calls enqueue
 * work and return without synchronising. Return value: 0 on success, a negative tenzo_status_t
 * value (tenzo.h) on bad arguments, or a positive cudaError_t if the launch failed.
 *
 * All kernels are sm_100a only; there is no CPU or other-backend fallback.
 *
 * Each entry names the reference code it replaces (paths inside catdlia/tenzo).
 */
#ifndef TENZO_KERNELS_H
#define TENZO_KERNELS_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#ifndef TENZO_API
#define TENZO_API __attribute__((visibility("default")))
#endif

/* ---- TL1 ternary GEMV with fused RMSNorm + absmax(31) quantiser ------------------------------
 * Replaces rms_norm_raw + build_lut + compute_single_block / compute_from_lut
 * (src/runtime/TenzoEngine.cpp:22-166) and the three call shapes that use them: the fused QKV
 * loop (:1547-1572), the fused gate/up loop + squared-ReLU GLU (:1593-1620), and the single
 * projections with residual add (:1585-1590, :1624-1628).
 *
 * Weights are the reference's own TL1 layout: [n_blocks][K/2][32 bytes]; byte c of a 32-byte
 * group carries row 64b+c (low nibble) and row 64b+32+c (high nibble) for columns (2k, 2k+1),
 * nibble = (w0+1)|((w1+1)<<2). K must be even, the weight pointer 16-byte aligned.
 *
 * Per sequence s in [0,batch):
 *   y   = do_norm ? x*(1/sqrt(mean(x^2)+eps))*norm_w : x                       (fp32)
 *   m   = max(1e-6, max|y|);  a_k = round(y_k*(31/m));  inv = m/31              (exact)
 *   acc_r = sum_k w[r][k]*a_k                                                    (int32, exact)
 *   v_r = (float)acc_r * (inv * scale_of_row_block)
 *   epilogue 0: out[r] = v_r
 *   epilogue 1: out[r] = resid[r] + v_r
 *   epilogue 2: rows [0,N/2) are gate, [N/2,N) up: out[r] = max(0,v_r)^2 * v_{r+N/2}, r < N/2
 */
enum { TENZO_EPI_STORE = 0, TENZO_EPI_RESIDUAL = 1, TENZO_EPI_RELU2_GLU = 2 };

typedef struct {
    const float* x;        /* [batch][x_stride] input activations */
    const float* norm_w;   /* [K] RMSNorm weight or NULL */
    int do_norm;
    float eps;             /* reference uses 1e-5 */
    const uint8_t* w;      /* TL1-packed weights, n_blocks*K/2*32 bytes */
    int n_blocks;          /* N/64 */
    int K;
    int seg_end[3];        /* row blocks [0,seg_end[0]) use seg_scale[0], [seg_end[0],seg_end[1]) ... */
    float seg_scale[3];    /* per-tensor weight scales (q/k/v or gate/up packed back to back) */
    int epilogue;
    const float* resid;    /* [batch][out_stride], epilogue 1 only */
    float* out;            /* [batch][out_stride] */
    int32_t* acc_out;      /* optional [batch][n_blocks*64] raw accumulators (parity checks) */
    int8_t* a_out;         /* optional [batch][K] quantised activations */
    float* inv_out;        /* optional [batch] m/31 */
    int batch;
    int x_stride, out_stride;
    const void* prefetch;  /* optional: memory the NEXT kernel in the stream will read (e.g. the next
                              layer's weights); requested into L2 while this kernel runs */
    size_t prefetch_bytes;
    void* workspace;       /* batch > 1 only: tenzo_cuda_tl1_gemv_workspace_bytes(batch, K) bytes, 16-byte
                              aligned; receives the packed int8 activations (contents need not be kept) */
    int use_pdl;           /* launch with programmatic stream serialisation (weights prefetch
                              overlaps the previous kernel's tail); 0 = ordinary launch */
} tenzo_tl1_gemv_args;

TENZO_API int tenzo_cuda_tl1_gemv(const tenzo_tl1_gemv_args* args, void* stream);
/* Cluster size along K (1, 2, 4 or 8 CTAs share one row block) the launcher picks for this shape; informational. */
TENZO_API int tenzo_cuda_tl1_gemv_ksplit(int n_blocks, int K, int epilogue);
/* Nine or more sequences (tensor-core path): CTAs of a thread-block cluster that share one 128-row tile's K range
 * (1, 2, 4 or 8; more than 1 when the row tiles alone would leave most SMs idle); 0 if that path does not take the
 * shape. Informational. */
TENZO_API int tenzo_cuda_tl1_gemm_ksplit(int n_blocks, int K, int batch, int epilogue);
/* Sequences a CTA of the tensor-core path holds for this shape (a multiple of 16, at most 256; several CTAs share the batch where it is fewer
 * than `batch`); 0 if that path does not take the shape. Informational; no counterpart in the reference. */
TENZO_API int tenzo_cuda_tl1_gemm_sequences(int n_blocks, int K, int batch, int epilogue);
/* The tensor-core path's layout of a CTA that holds min(batch, 256) sequences padded to 16 (tenzo_cuda_tl1_gemm_sequences says how many a shape's CTA holds):
 * ring slots (a multiple of four), groups of eight weight chunks in flight, dynamic shared memory in bytes, and the
 * bytes the epilogue may need in the two rings. Host arithmetic only (no device call); returns 0, or -1 for
 * fewer than nine sequences. Informational; no counterpart in the reference. */
TENZO_API int tenzo_cuda_tl1_gemm_layout(int batch, int* slots, int* weight_groups, size_t* smem_bytes, size_t* epilogue_bytes);
TENZO_API size_t tenzo_cuda_tl1_gemv_workspace_bytes(int batch, int K);
/* The kernel's waits on asynchronous copies are bounded. Returns 1 (and clears the flag) if any launch
 * since the last call gave up waiting — its output is then invalid; 0 otherwise; -1 if the query failed.
 * Synchronises with the device. */
TENZO_API int tenzo_cuda_tl1_gemv_take_timeouts(void);
/* One sequence: how many products since the last call were multiplied twice, because the integers presumed before the exact
 * root mean square was known did not stand (same results either way; one product in 200 to 600, and vectors whose
 * largest normalised magnitude is under the quantiser's floor of 1e-6 without being zero). -1 if the query failed. Synchronises with the device. */
TENZO_API int tenzo_cuda_tl1_gemv_take_repeats(void);
/* Test aid: launches a tiny kernel whose wait on a copy that is never issued runs out (after 2^8 polls), so that the flag
 * above is raised exactly as a real give-up raises it, without any fault or hang (the kernel finishes normally). Lets a
 * host exercise its own handling of the failure: the next tenzo_cuda_tl1_gemv_take_timeouts() returns 1, and an engine
 * call that checks the flags fails with its documented status. */
TENZO_API int tenzo_cuda_selftest_wait_expiry(void* stream);

/* ---- standalone fused RMSNorm + per-token absmax quantiser ------------------------------------
 * Replaces rms_norm_raw (:148-166) followed by the quantiser half of build_lut (:27-42,
 * qmax = 31) or of compute_logits (:1666-1678, qmax = 127: floor 1e-8, scale = amax/127,
 * q = clamp(round(y*(1/scale)))). y_out / q_out / scale_out are each optional.
 * scale_out receives m/31 (qmax 31) or amax/127 (qmax 127). */
TENZO_API int tenzo_cuda_rmsnorm_quant(const float* x, const float* norm_w, int do_norm, float eps, int dim,
                                       int qmax, int batch, int x_stride, float* y_out, int8_t* q_out,
                                       float* scale_out, void* stream);

/* ---- fused RoPE + INT8 KV append + GQA decode attention ---------------------------------------
 * Replaces FusedKVCache::forward_attention_raw in int8_fused mode (:447-533, :657-694, :823-851,
 * :911-913). Cache layout per sequence is the reference's: K,V int8 [layer][kv_head][max_seq][128],
 * scales fp32 [layer][kv_head][max_seq]; sequences are seq_stride_* apart. pos[s] is the slot the
 * new token is written to (= tokens already cached); attention then covers pos[s]+1 keys.
 * rope_cos/sin: [max_seq][head_dim/2] tables (built on the host with the reference's float
 * expressions so rotations are bit-identical); NULL skips RoPE. head_dim must be 128.
 * The kernel reproduces the reference's fp32 operation order (sequential sums over t, glibc expf
 * bits), so its output is bit-identical, not merely close. max_len is bounded at 36864 keys (without a workspace the score
 * vectors live in shared memory). */
typedef struct {
    const float* q;        /* [batch][q_stride]  n_q*128 used, pre-RoPE */
    const float* k;        /* [batch][kv_stride] n_kv*128 used, pre-RoPE new key */
    const float* v;        /* [batch][kv_stride] n_kv*128 used, new value */
    float* out;            /* [batch][n_q*128] */
    int q_stride, kv_stride; /* floats between sequences; 0 = dense (n_q*128 / n_kv*128) */
    int8_t* cache_k; int8_t* cache_v; float* scale_k; float* scale_v;
    size_t seq_stride_kv;  /* elements between sequences in cache_k/v */
    size_t seq_stride_sc;  /* elements between sequences in scale_k/v */
    const int* pos;        /* [batch] device */
    const float* rope_cos; const float* rope_sin;
    int layer, n_q, n_kv, head_dim, max_seq, batch;
    int max_len;           /* upper bound on pos[s]+1 for this launch (sizes the grid) */
    int append;            /* 1: quantise and store the new k,v at pos (normal decode); 0: the
                              cache already holds pos[s]+1 keys, k/v are ignored */
    int heads_per_cta;     /* 0 = choose automatically; 1, 2, 4 or 8 forces the query heads one CTA processes */
    int use_pdl;           /* launch with programmatic stream serialisation. The kernel launched immediately before must
                              then write none of pos, rope_cos / rope_sin or the cache rows below pos[s]: with the contiguous
                              cache and few items those are read before the wait for that kernel (q, k, v are read after).
                              With append == 0 nothing is read before it */
    int tiles;             /* 0 = choose automatically; 1 = force the variant whose scoring warps read K through TMA tiles
                              (two keys per lane; for many (sequence, kv head) items; returns -5 if it does not fit:
                              needs four 16 KB tile rings beside the weights, n_q/n_kv <= 4 heads per CTA, cache_k and
                              seq_stride_kv 16-byte aligned); 2 = force per-lane global loads; 3 = force the three kernels that
                              spread one launch's keys over all SMs (needs `workspace`; returns -5 if they do not fit) */
    /* kv_mode "paged_int8" (PagedKVCache of the reference, TenzoEngine.cpp:220-445, TenzoEngine.h:154-193). A non-NULL
     * block_table selects it: cache_k/cache_v are then the block pools int8 [block][n_layers][kv_head][16][128] and
     * scale_k/scale_v fp32 [block][n_layers][kv_head][16]; token t of sequence s lives in block
     * block_table[s*table_stride + t/16], slot t%16 (the entry for pos[s]/16 must exist before the call); seq_stride_*
     * are ignored. The arithmetic is that of PagedKVCache::forward_attention_raw, which is not the contiguous cache's
     * (two sets of eight FMA lanes, (dot*s_k)*scale, 1/(sum+1e-8), weights under 1e-7 dropped); outputs are
     * bit-identical to it. */
    const int* block_table; /* device */
    int table_stride;       /* ints between the tables of consecutive sequences; 0 = all query rows share one table */
    int n_layers;
    int n_pool_blocks;      /* blocks in the pools; 0 = not given, which rules out the TMA-tile variant (tiles == 1 then
                               returns -5): its tensor map needs the pool's extent */
    /* mode 0 (default): the reference's fp32 operation order, bit-identical outputs (above).
     * mode 1: tolerance mode. Same function, free evaluation order: the keys of a sequence are split over CTAs and
     * warps (online softmax, partials merged by log-sum-exp), both products run as fp16 tensor-core MMAs with fp32
     * accumulation (INT8 K/V are exact in fp16; the rotated query and the weights are rounded to fp16), exp is the
     * hardware ex2. Outputs agree with mode 0 to about 1e-4 of the output's largest magnitude (the specification asks
     * 1e-3 for floating-point outputs); the cache bytes written for the new token are identical in both modes.
     * Contiguous cache only (block_table must be NULL), 16-byte aligned caches, scales and out, max_seq a multiple of 4;
     * returns -5 otherwise. */
    int mode;
    int split_keys;         /* mode 1: keys per CTA (rounded up to 128); 0 = choose automatically */
    void* workspace;        /* 16-byte aligned, contents need not be kept. Mode 1: tenzo_cuda_attention_workspace_bytes(...)
                               bytes for the partial results of the splits; with less, or NULL, fewer splits are chosen,
                               down to one that needs none (slower for few sequences of many keys), and split_keys that
                               need more are refused (-1). Mode 0: optional,
                               tenzo_cuda_attention_exact_workspace_bytes(...) bytes for the score vectors (room for one
                               sequence at least); not used up to max_len 256. NULL keeps them in shared memory, which
                               is slower for all but few sequences of some hundred keys. Same results either way */
    size_t workspace_bytes;
} tenzo_attention_args;

TENZO_API int tenzo_cuda_attention_int8(const tenzo_attention_args* args, void* stream);
/* As tenzo_cuda_tl1_gemv_take_timeouts, for the attention kernel's bounded waits on its V-chunk copies (1). Also
 * returns 2 when a launch found a pos[s] outside [0, max_len): that CTA wrote nothing. */
TENZO_API int tenzo_cuda_attention_take_timeouts(void);
/* Scratch bytes mode 1 may need for these sizes (an upper bound over every split it can choose). */
TENZO_API size_t tenzo_cuda_attention_workspace_bytes(int batch, int n_q, int n_kv, int max_len);
/* Scratch bytes with which mode 0 takes whole batches at its best; bounded (about 64 MB, or one sequence's scores). */
TENZO_API size_t tenzo_cuda_attention_exact_workspace_bytes(int batch, int n_q, int n_kv, int max_len);
/* The same for mode 0 with many query rows over one contiguous cache (seq_stride_kv 0, append 0: a prompt's rows), whose scores
 * are worked out tile by tile; for calls of `batch` rows and of up to max_len keys. Never less than the above, and no more where no such call
 * has rows enough for the form. Bounded as well (about 256 MB and 1 KB a key and kv head). With less scratch such calls take smaller passes,
 * or the form that other batches take: same results. */
TENZO_API size_t tenzo_cuda_attention_rows_workspace_bytes(int batch, int n_q, int n_kv, int max_len);
/* Query heads one CTA will process for this shape (1..n_q/n_kv); informational. */
TENZO_API int tenzo_cuda_attention_heads_per_cta(int batch, int n_q, int n_kv, int max_len);

/* ---- INT8 LM head GEMV with fused final RMSNorm + absmax(127) quantiser + argmax --------------
 * Replaces compute_logits' int8 branch (:1634-1638, :1661-1719) and the greedy branch of
 * sample_top_k_top_p (:1745-1755: first maximum wins). logits/argmax_out/acc_out optional.
 * scratch: tenzo_cuda_lm_head_scratch_bytes(batch) bytes, 16-byte aligned. With two or more sequences, hidden a
 * multiple of 128 and vocab <= 262144 the product runs on the tensor cores (tcgen05 kind::i8): the activations are
 * normalised and quantised once, the vocabulary matrix is read once for all sequences; results are identical. */
TENZO_API int tenzo_cuda_lm_head_i8(const float* x, const float* norm_w, int do_norm, float eps,
                                    const int8_t* w, const float* row_scales, int vocab, int hidden,
                                    int batch, int x_stride, float* logits, int32_t* acc_out,
                                    int* argmax_out, void* scratch, int use_pdl, void* stream);
TENZO_API size_t tenzo_cuda_lm_head_scratch_bytes(int batch);
/* As tenzo_cuda_tl1_gemv_take_timeouts, for the bounded waits of the tensor-core LM head (two or more sequences). */
TENZO_API int tenzo_cuda_lm_head_take_timeouts(void);

/* ---- LM head without any allocation -------------------------------------------------------------
 * No counterpart in the reference. Same computation and results as tenzo_cuda_lm_head_i8, for
 * callers that are not allowed to allocate device memory while running (a server whose memory is
 * fully committed to its KV pool, a host application that bans cudaMalloc after start-up): the
 * argmax scratch is a fixed array inside the library (151,552 bytes held on each GPU that loads the
 * library, for the life of the process) instead of a caller-provided buffer, and the call performs
 * no cudaMalloc/cudaFree or other allocating routine.
 *   - batch <= tenzo_cuda_lm_head_static_max_batch() (32); larger batches return
 *     TENZO_ERROR_UNSUPPORTED (-5) and should use tenzo_cuda_lm_head_i8 with their own scratch.
 *   - The first call on each device looks up the array's device address (the device must be
 *     current); make that first call before starting any stream capture.
 *   - All calls on a device share the one array. It is fully rewritten by every call, so nothing
 *     needs clearing, but two calls that overlap on the GPU (different streams) would race on it:
 *     keep calls on one stream or otherwise ordered. */
TENZO_API int tenzo_cuda_lm_head_i8_static(const float* x, const float* norm_w, int do_norm, float eps,
                                           const int8_t* w, const float* row_scales, int vocab, int hidden,
                                           int batch, int x_stride, float* logits, int32_t* acc_out,
                                           int* argmax_out, int use_pdl, void* stream);
TENZO_API int tenzo_cuda_lm_head_static_max_batch(void);

/* ---- Sampling support: repetition penalty and top-k candidate selection on the device ----------------
 * Replaces the first half of sample_top_k_top_p (:1735-1768). tenzo_cuda_repetition_penalty applies
 * l > 0 ? l / penalty : l * penalty to logits[tokens[i]], counts[i] times (tokens distinct).
 * tenzo_cuda_topk_candidates finds the k-th largest logit v* (three-pass radix select, one CTA) and writes every
 * (value, index) with value >= v* in ascending index order: *count gets their number; values/indices (each
 * tenzo_cuda_topk_max_candidates() entries) are written only if it does not exceed that capacity. Running the
 * reference's streaming top-k over these candidates gives the same heap as over the whole vector. */
TENZO_API int tenzo_cuda_repetition_penalty(float* logits, int vocab, const int* tokens, const int* counts, int n, float penalty, void* stream);
TENZO_API int tenzo_cuda_topk_candidates(const float* logits, int vocab, int k, int* count, float* values, int* indices, void* stream);
TENZO_API int tenzo_cuda_topk_max_candidates(void);

/* ---- 4-bit paged KV cache: append, read, attention, and the tables of beams -----------------------------
 * No counterpart in the reference (its caches hold 8 bits). Pool: uint8 [block][layer][kv_head][K, V][16 slots][80], 16-byte
 * aligned. A row is 64 bytes of codes - dim d in nibble d % 2 of byte d / 2, the low nibble first - and four pairs (scale, minimum)
 * of fp16, one for each 32 dims; a value is minimum + scale * code. 160 bytes a token and kv head (the INT8 caches: 264).
 * A pool that tenzo_cuda_kv4_append did not fill has finite parameters too, and |minimum + 8 scale| <= 65504: the attention holds that sum in fp16 parts.
 * Token t of table row s lives in block block_table[s * table_stride + t / 16], slot t % 16. head_dim is 128.
 *
 * A position outside its range, a table row outside [0, table_rows) or a table entry outside [0, n_blocks) touches no memory: that row is
 * left out and a flag is raised, which tenzo_cuda_kv4_take_errors() returns and clears. Calls on one device share the flags only. */
typedef struct {
    uint8_t* pool;
    int n_blocks, n_layers, n_kv;
    const int* block_table;  /* device int32 [table_rows][table_stride] */
    int table_rows, table_stride;
} tenzo_kv4_cache;

/* Stores `rows` rows of keys and values: k, v [rows][kv_stride] fp32 (n_kv*128 used; rows may be strided, kv_stride >= n_kv*128), row i
 * at position pos[i] of table row seq[i] (seq NULL: table row i). pos[i] < 0 marks padding: nothing is stored. No two rows of a call may name
 * the same token. Keys are rotated first (rope tables [rope_len][64], position < rope_len; both NULL: no rotation) as pairs (i, i + 64):
 *   r_i = fma(x_i, c, -(x_{i+64} * s)),  r_{i+64} = fma(x_i, s, x_{i+64} * c).
 * Then per 32 dims, each step rounded to fp32: x = clamp(x, +-65504), minimum = fp16(min x), scale = fp16((max x - minimum) * (1/15)),
 * code = clamp(rint((x - minimum) * (1/scale)), 0, 15), ties to even; scale 0 gives codes 0. Values have to be finite (others spoil their own
 * 32 dims only). */
TENZO_API int tenzo_cuda_kv4_append(const tenzo_kv4_cache* cache, int layer, const float* k, const float* v, int kv_stride, const int* pos,
                                    const int* seq, int rows, const float* rope_cos, const float* rope_sin, int rope_len, int use_pdl, void* stream);
/* The stored rows as fp32: k, v [rows][kv_stride] (either may be NULL) receive minimum + scale * code, zeros for padding and for rows that are
 * refused. Keys come back rotated, as they are stored. */
TENZO_API int tenzo_cuda_kv4_read(const tenzo_kv4_cache* cache, int layer, float* k, float* v, int kv_stride, const int* pos, const int* seq, int rows,
                                  int use_pdl, void* stream);

/* out[row] = softmax(q K^T / sqrt(128)) V per query head over the keys 0 .. pos[row] of table row seq[row] (seq NULL: row), the query rotated at
 * pos[row] as above; query head h reads kv head h / (n_q / n_kv), any n_q that n_kv divides. Several rows may name one sequence
 * (a prompt's or a draft's rows, each with its own position). pos[row] < 0: zeros. A row whose position is max_len or more, or whose table row is
 * out of range, is not written and raises the flag; a table entry out of range leaves its 16 keys out and raises it. Sums and softmax in
 * fp32; the query is rounded to 23 bits of its head's largest number, products with the weights keep 22 bits (two fp16 parts), outputs agree with
 * 64 bits to about 1e-6 of the output's norm where scores are not above a few tens. A NaN or an infinity in a head's query makes that head's output NaN. */
typedef struct {
    const float* q;          /* [rows][q_stride], n_q*128 used, before rotation */
    float* out;              /* [rows][n_q*128] */
    tenzo_kv4_cache cache;
    const int* pos;          /* [rows] device */
    const int* seq;          /* [rows] device, or NULL */
    const float* rope_cos; const float* rope_sin;   /* [rope_len][64], rope_len >= max_len; both NULL: no rotation */
    int rope_len;
    int q_stride;            /* floats between rows; 0 = n_q*128 */
    int layer, n_q, rows;
    int max_len;             /* upper bound on pos + 1 (sizes the grid); at most 16 * table_stride */
    int split_keys;          /* keys a CTA takes (rounded up to 128); 0 = choose */
    int use_pdl;             /* launch with programmatic stream serialisation; nothing is read before the wait for the kernel in front */
    void* workspace;         /* 16-byte aligned, contents need not be kept: partial results of splits; NULL: none */
    size_t workspace_bytes;  /* rows * n_q * 520 a split; with less fewer splits are taken, and split_keys that need more are refused (-1). Enough for any split_keys:
                                tenzo_cuda_attention_kv4_workspace_bytes(...); for split_keys 0: 520 * rows * n_q * tenzo_cuda_attention_kv4_splits(...), nothing at 1 */
} tenzo_attention_kv4_args;
TENZO_API int tenzo_cuda_attention_kv4(const tenzo_attention_kv4_args* args, void* stream);
TENZO_API size_t tenzo_cuda_attention_kv4_workspace_bytes(int rows, int n_q, int n_kv, int max_len);
/* Splits that the call's own choice (split_keys 0) wants room for; 1: none, 0: arguments that the call refuses. */
TENZO_API int tenzo_cuda_attention_kv4_splits(int rows, int n_q, int n_kv, int max_len);
/* Error flags of the calls above and below this one since the last call (bit 0: a bounded wait was given up, bit 1: an index out of range);
 * -1 if the query failed, which leaves the flags as they are. Synchronises with the device: waits for all of its streams, so it cannot be called while one is
 * captured. */
TENZO_API int tenzo_cuda_kv4_take_errors(void);

/* The cache's half of a beam-search step. Table rows g*beams .. g*beams + beams - 1 are the beams of group g and hold length[g] tokens each; beam i goes
 * on from beam parent[g*beams + i] (0 .. beams - 1). With j = length / 16 and r = length % 16, row i of table_out gets its parent's entries below j (full
 * blocks are shared) and its own above j. The block being filled, entry j if r > 0, belongs to one beam alone (they must differ): the first child of a
 * parent takes its parent's; the n-th of the further children, by index, takes that of the n-th beam without children, and the r filled slots of all layers and heads are copied
 * into it. If r = 0, entry j stays the beam's own. No block is allocated or freed, and a prompt is forked the same way: parent 0 for
 * all. table_out [groups*beams][table_stride] must not overlap the table (-1); groups*beams = table_rows, beams <= TENZO_BEAMS_MOST and
 * n_layers*n_kv <= 16384 (-5 otherwise). A group with a parent or a length out of range is copied as it is and raises the flag. */
enum { TENZO_BEAMS_MOST = 32 };
TENZO_API int tenzo_cuda_kv4_reorder(const tenzo_kv4_cache* cache, int* table_out, const int* parent, const int* length, int groups, int beams, int use_pdl,
                                     void* stream);

/* ---- beam search: the k best continuations over beams x vocabulary -----------------------------------------
 * Beside the greedy argmax and the sampler (:1722-1807); the reference has no beam search. logits [groups*beams][row_stride] fp32,
 * scores [groups*beams] the beams' sums of log-probabilities. Per group, over all beams b and tokens t,
 *   score(b, t) = scores[b] + (x_t - log sum_u exp x_u)   in 64 bits
 * (exponentials other than the largest ones' enter the sum with 32: its logarithm is good to some 1e-7, to 2e-6 at the worst),
 * the k best go to parent_out / token_out / score_out [groups][k], best first; of equal scores the lower beam, in a beam the larger logit, then the
 * lower token. score_out is rounded to fp32.
 * A finished beam (finished[row] != 0) has its end token `eos` alone, at scores[b]. -inf masks a token; NaN counts as -inf, +inf as the largest finite
 * number. A beam with score -inf or NaN, or with no token left, has score -inf for every token (chosen only when nothing else is left, lowest index
 * first). beams <= TENZO_BEAMS_MOST and k <= 2 * TENZO_BEAMS_MOST (-5 otherwise); k <= beams * vocab. */
typedef struct {
    const float* logits;
    const float* scores;
    const int* finished;     /* [groups*beams] device, or NULL */
    int eos;                 /* used with `finished` only */
    int row_stride;          /* floats between rows of logits; 0 = vocab */
    int groups, beams, vocab, k;
    int use_pdl;
    int* parent_out; int* token_out; float* score_out;
    void* workspace;         /* tenzo_cuda_beam_select_workspace_bytes(...) bytes, 16-byte aligned, contents need not be kept */
    size_t workspace_bytes;
} tenzo_beam_select_args;
TENZO_API int tenzo_cuda_beam_select(const tenzo_beam_select_args* args, void* stream);
TENZO_API size_t tenzo_cuda_beam_select_workspace_bytes(int groups, int beams, int vocab, int k);

/* ---- INT8 caches: drafted trees, and caches of a bounded number of tokens ---------------------------------
 * No counterpart in the reference, which decodes one token at a time and keeps every token. The caches are those of tenzo_cuda_attention_int8: int8
 * [block][n_layers][n_kv][slots][128] for keys and for values and fp32 scales [block][n_layers][n_kv][slots] (a value is code * scale). The token at place t of table
 * row s lies in block block_table[s * table_stride + t / slots], slot t % slots; slots is a multiple of 16. The paged_int8 pools have 16 slots; the contiguous
 * cache [sequence][layer][kv_head][max_seq][128] is a pool of max_seq slots a block whose table has one entry a sequence. Caches and scales are 16-byte aligned and
 * hold fewer than 2^31 rows; scales are not negative. head_dim is 128.
 *
 * Here a token's place is not its rotary position: nodes of a tree that lie side by side have the same position, and behind an eviction positions and places
 * come apart for good. Calls that rotate take both.
 * An index out of range (a place, a position, a table row or entry, a length) touches no memory: that row is left out and a flag is raised, which
 * tenzo_cuda_kv8_take_errors() returns and clears. Calls on one device share the flags only. */
typedef struct {
    int8_t* k; int8_t* v;
    float* scale_k; float* scale_v;
    int n_blocks, n_layers, n_kv, slots;
    const int* block_table;  /* device int32 [table_rows][table_stride] */
    int table_rows, table_stride;
} tenzo_kv8_cache;
enum { TENZO_TREE_MOST = 256 };  /* nodes of a tree */

/* Stores `rows` rows of keys and values: k, v [rows][kv_stride] fp32 (n_kv*128 used, kv_stride >= n_kv*128), row i at place place[i] of table row seq[i]
 * (seq NULL: table row i). place[i] < 0 marks padding: nothing is stored. No two rows of a call may name the same token. Keys are rotated at rope_pos[i] (NULL: place[i];
 * tables [rope_len][64], position < rope_len; both NULL: no rotation) as tenzo_cuda_attention_int8 does, then both are quantised: scale = max(max|x|, 1e-8) * (1/127),
 * code = clamp(round(x * (1 / scale)), -128, 127), halves away from zero, each step rounded to fp32. (tenzo_cuda_attention_int8 divides by 127: its scales may differ in
 * the last bit, and a code next to a border by one.) Values have to be finite.
 * weight, position (either may be NULL), laid out as the scales: receive 0 and the row's rotary position, for the calls below. */
typedef struct {
    tenzo_kv8_cache cache;
    const float* k; const float* v;                 /* [rows][kv_stride] */
    const int* place;                               /* [rows] device */
    const int* seq; const int* rope_pos;            /* [rows] device, or NULL */
    const float* rope_cos; const float* rope_sin;   /* [rope_len][64], 16-byte aligned; both NULL: no rotation */
    float* weight; int* position;                   /* or NULL */
    int layer, kv_stride, rows, rope_len;
    int use_pdl;
} tenzo_kv8_append_args;
TENZO_API int tenzo_cuda_kv8_append(const tenzo_kv8_append_args* args, void* stream);

/* Attention of the nodes of a tree, for each of `sequences` trees of up to `nodes` nodes (1 .. TENZO_TREE_MOST): sequence s holds start[s] tokens, and node i's key and
 * value are stored at place start[s] + i already. Node i sees places 0 .. start[s] - 1, and node j if bit j % 32 of mask[(s*nodes + i)*mask_stride + j / 32] is
 * set (itself too: any bits will do). mask NULL: nodes 0 .. i, a chain (a prompt's next rows, one decoded token with nodes = 1). count[s] (NULL: nodes): nodes that
 * are there; the others are padding, are seen by none, and their rows of out are zeros. start[s] < 0: the whole sequence is padding.
 *   out[s*nodes + i] = softmax(q K^T / sqrt(128)) V per query head h, over kv head h / (n_q / n_kv), the query rotated at rope_pos[s*nodes + i] (NULL: start[s] + i);
 *   lse = log sum exp of the arguments (natural logarithm; -infinity and zeros in out where nothing is seen).
 * Sums and softmax in fp32 or whole numbers; the query is rounded to 2^-30 of its head's largest number, a weight times its value's scale to 2^-26 of the largest such product that the row
 * had met when it was last looked for: outputs agree with 64 bits as plain fp32 does, to about 1e-6 of their norm with arguments of ordinary size. (What an argument may be off by is some 2^-22 of itself, and 2^-30 of the
 * query's largest number times the key's sum of magnitudes / sqrt(128).) Scales of values are within 2^60 of each other where rows see them, and from 2^-60 on; smaller ones count as 0. A NaN or an infinity in a head's query makes that head's outputs NaN; what lies in places that are not seen has no part.
 * A sequence with start + count > max_len or a table row out of range, and a row whose position is, are not written and raise the flag; a table entry out
 * of range leaves its block's keys out and raises it. */
typedef struct {
    const float* q;          /* [sequences*nodes][q_stride], n_q*128 used, before rotation */
    float* out;              /* [sequences*nodes][n_q*128], 16-byte aligned, apart from q */
    float* lse;              /* [sequences*nodes][n_q], or NULL; apart from q and out where it is written */
    tenzo_kv8_cache cache;
    const int* start;        /* [sequences] device */
    const int* count;        /* [sequences] device, or NULL */
    const int* seq;          /* [sequences] device: table rows, or NULL: table row s */
    const int* mask;         /* [sequences*nodes][mask_stride] device, or NULL */
    const int* rope_pos;     /* [sequences*nodes] device, or NULL */
    const float* rope_cos; const float* rope_sin;   /* [rope_len][64]; both NULL: no rotation */
    int rope_len;
    int q_stride;            /* floats between rows; 0 = n_q*128 */
    int mask_stride;         /* words between rows; 0 = ceil(nodes / 32) */
    int layer, n_q, sequences, nodes;    /* n_q at most 2^17, n_kv at most 65535 (-5) */
    int max_len;             /* upper bound on start + count; at most slots * table_stride, and 2^30 (-5) */
    int shares;              /* equal shares that the keys of all sequences and kv heads are cut into, each of one CTA (or some, for many queries); 0 = choose, at most 65535 */
    int use_pdl;             /* launch with programmatic stream serialisation; nothing is read before the wait for the kernel in front */
    void* workspace;         /* 16-byte aligned, contents need not be kept, of one call at a time (two graphs that may run together have two): partial results where a
                                cut goes through a sequence's keys */
    size_t workspace_bytes;  /* tenzo_cuda_attention_tree_workspace_bytes(...), with shares = 0 10 MB and 8 bytes a sequence and kv head at most, whatever the lengths are. With less, or NULL, shares end with a sequence's kv head, which is
                                slower for few sequences and for unequal ones; shares > 0 is refused then (-1). With
                                shares = 0 it is not used where max_len <= 512 */
} tenzo_attention_tree_args;
TENZO_API int tenzo_cuda_attention_tree(const tenzo_attention_tree_args* args, void* stream);
/* (0 for arguments that the call refuses.) */
TENZO_API size_t tenzo_cuda_attention_tree_workspace_bytes(int sequences, int nodes, int n_q, int n_kv, int shares);

/* The attention weight that each cached token receives: weight[token] += sum over the nodes that see it and the query heads of its kv head of exp(s - lse), s the
 * argument of softmax above. args as for tenzo_cuda_attention_tree, whose lse this reads; out, workspace and shares are not used. weight is laid out as the scales.
 * All nodes count, also those of a draft that are refused later. To leave these out, call it behind tenzo_cuda_kv8_accept for the accepted ones, whose rows are a chain there: q, lse and rope_pos
 * gathered by path (anything where that is -1), count = accepted, mask NULL, start as it was; nodes and the arrays may be as long as before.
 * A row whose lse is not finite adds nothing; weights and sums below 2^-126 may count as 0. Every sum is taken in one order: equal calls give equal bits. No two sequences of a call may name
 * the same table row, or blocks in common (a token would lose what one of them adds); attention reads common blocks as well as others. */
TENZO_API int tenzo_cuda_kv8_weigh(const tenzo_attention_tree_args* args, float* weight, void* stream);

/* Cuts caches back to `keep` tokens, for each layer and kv head on its own: table rows seq[s] (NULL: s) hold length[s] tokens at places 0 .. length[s] - 1, with the
 * weight and position (16-byte aligned) that tenzo_cuda_kv8_append and _weigh left. Where length[s] > keep, the `keep` heaviest stay; a token whose position is protect_from[s] or more counts as
 * infinitely heavy (protect_from NULL: none does), NaN as -infinity, and of equal weights the lower place stays. Tokens that stay keep their places if those are below `keep`; the others
 * move, in the order of their places, to the places below `keep` that became free, in the order of those, with scales, weight and position. (Order means nothing to
 * attention over rotated keys: it takes one row's move a token evicted, not the whole cache's.) length_out[s] = min(length[s], keep), in
 * memory of its own (-1 where it has bytes in common with what the call reads). No two sequences of a call may name the same table row, or blocks in common.
 * A negative length, one above max_len, a table row out of range or a table entry out of range leaves the sequence as it is, with length_out[s] = length[s], and raises the
 * flag. max_len <= slots * table_stride; max_len <= 2^20 and sequences <= 65535 (-5 otherwise). */
typedef struct {
    tenzo_kv8_cache cache;
    float* weight; int* position;
    const int* length;                              /* [sequences] device */
    const int* seq; const int* protect_from;        /* [sequences] device, or NULL */
    int* length_out;                                /* [sequences] device */
    int sequences, keep, max_len;
    int use_pdl;
} tenzo_kv8_evict_args;
TENZO_API int tenzo_cuda_kv8_evict(const tenzo_kv8_evict_args* args, void* stream);

/* The nodes of drafted trees that the model agrees with, and their rows moved up behind the cached ones. token, parent, chosen [sequences][nodes]: node i's token, the node it
 * goes on from (below i; node 0 is the root, a token that counts already), and the token that the model chose after node i (its argmax, or a draw). From the root, the next node is the first whose
 * parent is the present one and whose token is the one chosen there, until there is none. path [sequences][nodes]: these nodes, root first, then -1; accepted[s]: how many; next[s]: the token
 * chosen after the last. Row d of a path is moved from place start[s] + path[d] to start[s] + d in all layers, with scales and weight and position (either may be NULL).
 * count, seq, start as for tenzo_cuda_attention_tree. A sequence of padding (start[s] < 0 or count[s] = 0) has accepted 0, next -1. So has one with start + count above slots * table_stride, with count
 * out of range or a table row out of range, which raises the flag; a table entry out of range leaves the rows that need it where they are, and raises it. No two sequences of a call may
 * name the same table row, or have blocks in common; sequences <= 65535, nodes <= TENZO_TREE_MOST (-5 otherwise). */
typedef struct {
    tenzo_kv8_cache cache;
    const int* token; const int* parent; const int* chosen;   /* [sequences][nodes] device */
    const int* start;                               /* [sequences] device */
    const int* count; const int* seq;               /* [sequences] device, or NULL */
    int* accepted; int* next; int* path;            /* device: [sequences], [sequences], [sequences][nodes], in memory of their own (-1 otherwise) */
    float* weight; int* position;                   /* or NULL */
    int sequences, nodes;
    int use_pdl;
} tenzo_kv8_accept_args;
TENZO_API int tenzo_cuda_kv8_accept(const tenzo_kv8_accept_args* args, void* stream);
/* Error flags of the calls of this section since the last call (bit 0: a bounded wait was given up, bit 1: an index out of range); -1 if the query failed, which leaves the
 * flags as they are. Synchronises with the device: waits for all of its streams, so it cannot be called while one is captured. */
TENZO_API int tenzo_cuda_kv8_take_errors(void);

/* ---- INT8 embedding row dequantisation ---------------------------------------------------------
 * Replaces embedding_lookup's int8 branch (:1299-1315): x = (float)W8[tok] * scale[tok].
 * vocab > 0: token ids outside [0, vocab) are read as row 0 rather than past the table; 0 = unchecked. */
TENZO_API int tenzo_cuda_embedding_i8(const int8_t* w, const float* row_scales, int hidden,
                                      const int* tokens, int batch, float* x, int x_stride, int vocab, void* stream);

/* ---- checkpoint rows -> TL1 layout --------------------------------------------------------------
 * Replaces pack_ternary_weights_raw (:1842-1884): raw [N/4][K] bytes (row r in bits 2*(r%4)) to
 * the [N/64][K/2][32] layout above. */
TENZO_API int tenzo_cuda_tl1_pack_rows2bit(const uint8_t* raw, int N, int K, uint8_t* packed, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TENZO_KERNELS_H */
