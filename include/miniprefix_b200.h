/*
 * miniprefix_b200.h -- C ABI of the B200 (sm_100a) MiniPrefix forward over paged KV.
 *
 * This is the drop-in boundary for the device half of TinyInfer MiniPrefix's
 * CudaRunner (TinyInfer v0.3.0, miniprefix/src/backend/cuda/llama_runner.cu). The
 * reference's host bookkeeping (KVManager, ExactPrefixCache, Engine) keeps owning
 * metadata; it calls these functions where CudaRunner called cudaMalloc, cuBLAS,
 * its seven kernels and cudaMemcpy*. Plain C types only; every pointer is
 * caller-owned unless stated. One context per GPU, single-threaded per context
 * (the reference's ModelRunner contract, miniprefix/include/miniprefix/kv_manager.h:18-19).
 *
 * Return codes: MP_OK or one of MP_ERR_*; mp_last_error() gives the message of
 * the last failure on the calling thread.
 */
#ifndef MINIPREFIX_B200_H
#define MINIPREFIX_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MP_OK 0
#define MP_ERR_INVALID 1     /* rejected argument; no state changed */
#define MP_ERR_CUDA 2        /* CUDA runtime failure */
#define MP_ERR_NONFINITE 3   /* a logit of the step was NaN/Inf */
#define MP_ERR_BOUNDS 4      /* device bounds check tripped (page id, token, region) */
#define MP_ERR_TIMEOUT 5     /* bounded wait expired (host sync or in-kernel copy wait) */
#define MP_ERR_NOMEM 6       /* device allocation failed */
#define MP_ERR_UNSUPPORTED 7 /* model geometry outside the specialised kernels */

typedef struct mp_context mp_context;

/* Mirrors miniprefix::ModelConfig (miniprefix/include/miniprefix/model.h:9-16). */
typedef struct {
    int32_t layers, hidden, intermediate, heads, kv_heads, vocabulary, context, eos;
    float rms_epsilon, rope_theta;
    int32_t tied;
} mp_model_config;

/* Paged KV pool and step capacities. block_tokens / max_blocks are
 * KvCacheConfig's (miniprefix/include/miniprefix/paged_kv.h:13-17); each of the K
 * and V pools holds max_blocks * layers * block_tokens * kv_width floats. On the
 * device a pool is layer-major, [layer][block][slot][kv_width], so that one layer's
 * pages share a compact address range; every pool offset this API takes (COW
 * regions, mp_kv_read / mp_kv_write) is an offset in the reference layout
 * [block][layer][slot][kv_width] (paged_kv.h:25-27) and is translated. */
typedef struct {
    int32_t block_tokens;
    int32_t max_blocks;
    int32_t max_sequences;      /* device block-table slots */
    int32_t table_stride;       /* entries per slot: >= ceil(context / block_tokens) */
    int32_t max_step_tokens;    /* most tokens one forward may carry (sum over sequences) */
    int32_t max_step_sequences; /* most sequences one forward may carry */
} mp_runtime_config;

/* One sequence of a forward: `count` new tokens appended at positions
 * start .. start+count-1 of the sequence whose block table lives in `slot`. The
 * table must already map every page that covers start+count tokens. */
typedef struct {
    int32_t slot, start, count;
} mp_sequence_desc;

/* One block-table entry: tables[slot][index] = block. */
typedef struct {
    int32_t slot, index, block;
} mp_table_entry;

/* KVManager::TailCopyRegion (miniprefix/include/miniprefix/kv_manager.h:38): float
 * element offsets into ONE pool; the copy is applied to both the K and V pools. */
typedef struct {
    uint64_t destination, source, pitch, width, rows;
} mp_tail_copy_region;

const char* mp_last_error(void);

/* Replaces CudaRunner's constructor (llama_runner.cu:78-87): selects `device`,
 * creates the stream, allocates weights, both pools (zeroed), tables and the
 * step workspace. */
int mp_create(int device, const mp_model_config* model, const mp_runtime_config* runtime, mp_context** out);
void mp_destroy(mp_context* ctx);

/* Replaces upload_parameter (llama_runner.cu:72-76): one MPFX0001 tensor by name,
 * [in, out] orientation as stored by the reference (miniprefix/src/model/model.cpp:28-38).
 * The tied head is read from the embedding; no transposed copy is made (:84). */
int mp_set_weight(mp_context* ctx, const char* name, const float* host, size_t elements);
/* Checks every tensor arrived and packs the device copies. Required before forward. */
int mp_finalize_weights(mp_context* ctx);

/* Replaces the incremental block-table upload (llama_runner.cu:139-143, :113):
 * entries [first, first+count) of `slot` := blocks. Queued on the context stream. */
int mp_table_write(mp_context* ctx, int32_t slot, int32_t first, const int32_t* blocks, int32_t count);

/* Replaces the COW cudaMemcpy2DAsync pair (llama_runner.cu:130-137), batched:
 * every region copies rows x width floats at pitch in both pools. */
int mp_cow_copy(mp_context* ctx, const mp_tail_copy_region* regions, int32_t count);

/* Replaces the append body (llama_runner.cu:128-170) for a BATCH of sequences:
 * uploads tokens, descriptors, block-table entries and COW regions in one copy,
 * applies the table entries, performs the COW copies (all layers, both pools,
 * before any layer runs), runs the 30-layer forward, and downloads per
 * sequence the greedy token (first index of the maximum, engine.cpp:99), a
 * finiteness flag (:94-95) and, when out_logits is not NULL, the full last-row
 * logits (sequences x vocabulary floats, the reference's append() result).
 * Blocks until the step completed or timeout_ms elapsed (MP_ERR_TIMEOUT).
 * Returns MP_ERR_NONFINITE when any sequence had a nonfinite logit (outputs are
 * still written) and MP_ERR_BOUNDS when a device bounds check tripped. */
int mp_forward(mp_context* ctx, const mp_sequence_desc* sequences, int32_t count, const int32_t* tokens,
               const mp_table_entry* entries, int32_t entry_count, const mp_tail_copy_region* regions,
               int32_t region_count, int32_t* out_tokens, int32_t* out_finite, float* out_logits,
               int32_t timeout_ms);

/* The same step split in three, for callers that keep inputs resident and time
 * the device work alone: prepare uploads, launch only enqueues kernels that read
 * device memory, collect downloads and waits. */
int mp_forward_prepare(mp_context* ctx, const mp_sequence_desc* sequences, int32_t count, const int32_t* tokens,
                       const mp_table_entry* entries, int32_t entry_count, const mp_tail_copy_region* regions,
                       int32_t region_count);
int mp_forward_launch(mp_context* ctx);
int mp_forward_collect(mp_context* ctx, int32_t* out_tokens, int32_t* out_finite, float* out_logits,
                       int32_t timeout_ms);

/* Failure-path tests (no counterpart in the reference, whose kernels have no
 * bounded waits): the next forward's first GEMM launch gets a producer that issues
 * no copies and waits bounded at `wait_us` microseconds (1 us .. 1 s). Its waits run
 * out, the kernel records the timeout bit, releases its tensor memory and returns,
 * and that forward reports MP_ERR_TIMEOUT (its outputs and the K/V rows it should
 * have written are garbage). The context stays usable: later forwards are normal. */
int mp_inject_wait_timeout(mp_context* ctx, int32_t wait_us);
/* Waits for all queued work with a bounded host wait (event polling). */
int mp_sync(mp_context* ctx, int32_t timeout_ms);

/* Device pointers of the K and V pools (layer-major, see mp_runtime_config) and
 * their element count (tests, tools). */
int mp_kv_pools(mp_context* ctx, float** keys, float** values, uint64_t* elements);
/* Synchronous host copies of pool payload (0 = K pool, 1 = V pool), element
 * offsets in the reference layout; for tests and tools that inspect or seed pages. */
int mp_kv_read(mp_context* ctx, int32_t pool, uint64_t offset, uint64_t count, float* host);
int mp_kv_write(mp_context* ctx, int32_t pool, uint64_t offset, uint64_t count, const float* host);
/* The context stream as a cudaStream_t (void* here to keep the ABI CUDA-free). */
void* mp_stream(mp_context* ctx);

/* Device event timing on the context stream: mp_timer_mark records a mark;
 * mp_timer_elapsed gives milliseconds between the last two marks. */
int mp_timer_mark(mp_context* ctx);
int mp_timer_elapsed(mp_context* ctx, float* milliseconds);
/* When enabled, forward launches bracket every attention launch with events;
 * mp_profile_read returns the summed attention milliseconds and launch count
 * since the last read (and resets them). */
int mp_profile_enable(mp_context* ctx, int32_t enabled);
/* No counterpart in the reference. Shared-prefix decode attention: decode rows
 * whose block tables start with the same physical pages (prefix reuse, forks)
 * form a group when at least min_rows rows share at least min_tokens tokens of
 * full pages, and a tensor-core kernel reads the group's shared pages once for
 * all its rows. min_rows 0 (the default) turns it off: every row then reads its
 * whole context, and the shared pages, read by many rows, stay in L2 -- measured
 * faster on B200 for every workload tried (1K-7K shared tokens x 256 rows, and
 * prefix-tree serving). */
int mp_set_shared_prefix(mp_context* ctx, int32_t min_rows, int32_t min_tokens);
int mp_profile_read(mp_context* ctx, float* attention_ms, int32_t* attention_launches, double* attention_bytes);
/* The same profiling (no counterpart in the reference) for the projection GEMMs:
 * the summed milliseconds and count of the intervals between one layer's attention
 * and the next layer's (each: O, gate/up and down of a layer plus the next layer's
 * QKV), and of the LM head GEMM; reset on read. */
int mp_profile_read_gemm(mp_context* ctx, float* layer_gemm_ms, int32_t* intervals, float* head_ms, int32_t* heads);
/* Cumulative counters of collected forwards: device time from the first to the
 * last kernel of each forward (CUDA events on the context stream), kernels
 * launched, and bytes moved host->device / device->host by the forwards;
 * shared_prefix_rows counts decode rows whose leading pages were served by the
 * shared-prefix kernel (once per forward), shared_prefix_tokens the tokens those
 * rows did not read themselves. host_prepare_ms, host_launch_ms and host_wait_ms
 * are host wall time spent in mp_forward_prepare (validation, attention plan,
 * metadata upload), mp_forward_launch (enqueueing the kernels) and waiting for
 * completion in mp_forward_collect. */
typedef struct {
    uint64_t forwards;
    double forward_ms;
    uint64_t kernel_launches;
    uint64_t h2d_bytes, d2h_bytes;
    uint64_t shared_prefix_rows, shared_prefix_tokens;
    double host_prepare_ms, host_launch_ms, host_wait_ms;
} mp_counters;
int mp_read_counters(mp_context* ctx, mp_counters* out, int32_t reset);

/* Device time of the COW copies of the last collected forward that had any
 * (milliseconds; 0 when it had none). Recorded only while cost timing is on. */
int mp_cow_timing(mp_context* ctx, int32_t enabled);
int mp_cow_elapsed(mp_context* ctx, float* milliseconds);

/* C = A . B^T (a [m][k], b [n][k], c [m][n] row-major, device buffers) through the
 * split-precision FP16 tcgen05 GEMM of the forward (each operand as FP16 halves,
 * three products per useful one; Store epilogue, with the forward's split-K
 * choice: shapes with few output tiles run as K slices summed in slice order);
 * n a multiple of 64, k of 32. Allocates its own scratch and synchronises
 * `stream`: a test/tool entry, not the hot path. */
int mp_gemm_f32(const float* a, const float* b, float* c, int32_t m, int32_t n, int32_t k, void* stream);

/* The paged-attention decode OPERATOR alone (one query row per sequence), on
 * caller device buffers: q [count][9*64] roped queries, pools in the reference
 * layout with `layers` layers, tables [count][table_stride] (device), out
 * [count][9*64]. `lengths` is a HOST array (tokens to attend per sequence);
 * pages_per_split 0 cuts the sequences' pages, concatenated, into one equal run
 * per CTA of a single wave (3 per SM); > 0 cuts each sequence into slices of
 * that many pages, pulled longest first by the wave. Runs on `stream`
 * (cudaStream_t, NULL = legacy default) and does not synchronise. Uses an
 * internal scratch buffer that grows on demand. */
int mp_paged_attention_decode(const float* q, const float* keys, const float* values, int32_t layers, int32_t layer,
                              int32_t block_tokens, int32_t max_blocks, const int32_t* tables, int32_t table_stride,
                              const int32_t* lengths, int32_t count, float* out, int32_t pages_per_split, void* stream);
/* No counterpart in the reference. The same decode operator for callers that
 * cannot allocate device memory -- e.g. a host embedding this library in another
 * runtime that owns all GPU memory or fixes its budget up front, or a path where
 * cudaMalloc/cudaFree must not run because they synchronise the device. It calls
 * no allocator: its scratch is one file-scope __device__ array of about 5 MB held
 * by every GPU that loads the library. At most 512 sequences and 2048 slices per
 * call (pages_per_split 0: equal runs per CTA, which always fit); larger requests return
 * MP_ERR_INVALID. All calls on a device share that array: calls whose device work
 * overlaps race. The first call on a device, with that device current, looks up
 * the array's address; make it before any stream capture. `device_error`
 * (optional, caller-owned device word, zeroed by the caller) receives the kernel's
 * error bits (1 = page id out of range, 2 = copy wait expired); when it is NULL the
 * bits go to a word inside the fixed array, which mp_paged_attention_status reads
 * and clears (before the next call on the device, which clears it again). */
int mp_paged_attention_decode_noalloc(const float* q, const float* keys, const float* values, int32_t layers,
                                      int32_t layer, int32_t block_tokens, int32_t max_blocks, const int32_t* tables,
                                      int32_t table_stride, const int32_t* lengths, int32_t count, float* out,
                                      int32_t pages_per_split, void* stream, uint32_t* device_error);
/* Synchronises `stream`, then reads and clears the decode operators' device error
 * words on the current device (mp_paged_attention_decode's, and the word that
 * mp_paged_attention_decode_noalloc fills when given no device_error): MP_OK,
 * MP_ERR_BOUNDS (a page id outside [0, max_blocks)) or MP_ERR_TIMEOUT (an in-kernel
 * copy wait expired; the allocating operator's arrival counters are reset). */
/* The paged-attention PREFILL operator alone: causal attention of chunks of
 * query rows (miniprefix/src/backend/cuda/llama_runner.cu:33-48 for rows past the
 * first; the CPU runner's loop miniprefix/src/backend/cpu/llama_runner.cpp:85-93).
 * Sequence i appends seq_counts[i] rows at positions seq_starts[i] ..
 * seq_starts[i] + seq_counts[i] - 1; its rows are consecutive in q and out
 * ([rows][9*64], sequences in order) and its K/V rows up to the last position are
 * already in the pools. Row r attends to the sequence's tokens 0 .. its position.
 * seq_starts / seq_counts are HOST arrays; tables [count][table_stride] (device).
 * Runs the tensor-core prefill kernel on `stream` without synchronising; shares
 * the decode operator's internal scratch (errors: mp_paged_attention_status). */
int mp_paged_attention_prefill(const float* q, const float* keys, const float* values, int32_t layers,
                               int32_t layer, int32_t block_tokens, int32_t max_blocks, const int32_t* tables,
                               int32_t table_stride, const int32_t* seq_starts, const int32_t* seq_counts,
                               int32_t count, float* out, void* stream);
int mp_paged_attention_status(void* stream);

/* ---------------------------------------------------------------- 8-bit paged KV cache
 * Operators on a paged K/V cache held in 8 bits, with one scale for each block of
 * block_tokens tokens, kv head and K or V (no counterpart in the reference; a quarter
 * of its FP32 cache's bytes). They stand beside the FP32 cache's operators above,
 * on caller device buffers:
 *   mp_kv8_append             rotates q and k, quantises k and v into the pages;
 *   mp_kv8_attention_decode   one query row per sequence over the pages;
 *   mp_kv8_attention_prefill  causal attention of packed chunks of rows.
 * A value is code * scale. Codes are INT8 (-127..127) or E4M3 (bytes of the 8-bit
 * float with 4 exponent and 3 mantissa bits, largest 448). The append chooses scales
 * that are powers of two; the attentions take any finite scale that is not negative (a K scale
 * times a row's largest |q| times |scale| has to stay in FP32's range).
 *
 * All arrays are device memory of the current device unless stated, and the metadata
 * (tables, lengths, row_offsets, starts) is read by the kernels only: no call copies
 * to the device, synchronises or allocates, so every call can be captured into a
 * graph and replayed with other metadata in the same buffers. A workspace may serve
 * both attentions and any number of captured calls as long as no two of them run at
 * the same time; after MP_ERR_TIMEOUT it must be zeroed again. Outputs must not overlap
 * a call's other buffers, unless stated. A null or misaligned pointer, a pointer that is not
 * memory of the current device, and sizes outside the stated ranges are refused with
 * MP_ERR_INVALID (a geometry without a kernel with MP_ERR_UNSUPPORTED) before
 * anything is queued. What only the device can see goes to `device_error`
 * (optional, caller-owned device word, zeroed by the caller; mp_kv8_status reads
 * and clears it): bit 1 = a block id outside [0, max_blocks) (an append leaves the
 * block's rows out, an attention reads block 0 instead); a length past the table (a row of
 * zeros); row_offsets that fall or leave `rows`, or positions outside the table or the
 * rotation tables (that sequence is left out whole: none of its rows is written; where offsets
 * fall, others may be left out too); more than 2^30 pieces of work for one SM (the call is left
 * out); bit 2 = a wait inside the
 * prefill kernel expired (its outputs are incomplete);
 * bit 4 = an appended value was NaN or infinite, or the scale of a block that already
 * held tokens was no power of two. */
#define MP_KV8_INT8 0
#define MP_KV8_E4M3 1
#define MP_TYPE_F32 0
#define MP_TYPE_BF16 1
#define MP_ROPE_HALF 0        /* pairs (i, i + rotary_dim / 2), the reference's */
#define MP_ROPE_INTERLEAVED 1 /* pairs (2i, 2i + 1) */

typedef struct {
    void* pages;          /* [max_blocks][kv_heads][2][block_tokens][head_dim] codes, 0 = K, 1 = V; 16-byte aligned */
    float* scales;        /* [max_blocks][kv_heads][2]; 8-byte aligned */
    int64_t page_stride;  /* bytes from a block to the next: a multiple of 16, >= kv_heads * 2 * block_tokens * head_dim */
    int64_t scale_stride; /* floats from a block's scales to the next block's: even, >= 2 * kv_heads */
    int32_t format;       /* MP_KV8_INT8 or MP_KV8_E4M3 */
    int32_t kv_heads;     /* 1 .. 256 */
    int32_t head_dim;     /* 64 or 128 */
    int32_t block_tokens; /* a multiple of 16, 16 .. 256 */
    int32_t max_blocks;
} mp_kv8_cache;

/* Rows of `count` sequences, packed: sequence i's rows are row_offsets[i] ..
 * row_offsets[i + 1] - 1 (row_offsets[0] = 0, nondecreasing; a sequence may have none),
 * at positions starts[i], starts[i] + 1, ...; `rows` is the number of rows that the
 * buffers hold: rows at or past row_offsets[count] are neither read nor written. A
 * row is heads (q) or kv_heads (k, v) x head_dim values of `type`; strides count
 * values between rows (a fused q | k | v projection: three pointers, one stride), with
 * 16-byte aligned rows.
 *
 * Every row's k is rotated by its position, and k and v go to slot position %
 * block_tokens of block tables[i][position / block_tokens]. With q, the rotated q goes
 * to q_out (which may be q itself, with its stride). Rotation of a pair (a, b): (a cos - b sin, b cos
 * + a sin) with row `position` of cos / sin ([max_positions][rotary_dim / 2]); dims at or
 * past rotary_dim pass unrotated (rotary_dim 0: no rotation, cos and sin unused). q is
 * rotated in FP32 (a rounded product and a fused multiply-add); k codes come from the exact
 * rotated value.
 *
 * The scale of a block written from its slot 0 on is the smallest power of two with
 * which the largest new magnitude fits the format (at least 2^-100); what the block
 * held is forgotten. A block that held tokens before (the first appended slot is past
 * 0) keeps its scale if that suffices, else takes the larger one and its codes are
 * rounded to it. A code is the nearest to value / scale, ties to even. An INT8 value
 * is then off by at most half its block's scale when appended, and by less than one
 * scale after any number of re-roundings (each scale is at least twice the one
 * before). NaN is stored as 0 and infinity as the largest code, with the error bit.
 * A block takes new rows from one place of one table per call; slots past a sequence's last
 * token keep their bytes. */
typedef struct {
    const void *q, *k, *v; /* q optional */
    void* q_out;           /* with q */
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const float *cos, *sin;     /* 16-byte aligned */
    const int32_t* tables;      /* [count][table_stride] block ids */
    const int32_t* row_offsets; /* [count + 1] */
    const int32_t* starts;      /* [count] */
    int32_t type;               /* MP_TYPE_* of q, k, v, q_out */
    int32_t heads;              /* query heads: 1 .. 64 per kv head, at most 1024 */
    int32_t rotary_dim;         /* a multiple of 8, 0 .. head_dim */
    int32_t rope_layout;        /* MP_ROPE_* */
    int32_t max_positions;
    int32_t table_stride;       /* table_stride * block_tokens <= 2^26 */
    int32_t count;              /* 1 .. 65536 */
    int32_t rows;
} mp_kv8_append_args;
int mp_kv8_append(const mp_kv8_cache* cache, const mp_kv8_append_args* args, uint32_t* device_error, void* stream);

/* out[i] = softmax(scale * q[i] K^T) V over tokens 0 .. lengths[i] - 1 of sequence i,
 * query head h reading kv head h / (heads / kv_heads). A length of 0 gives a row of
 * zeros. Sums, maxima and weights are FP32; products run on the tensor cores as FP16
 * halves (FP32-level: the codes are exact in FP16, an FP32 query and weight is two
 * halves; of a BF16 call's weights the high half alone). Counted as zero are weights below
 * 2^-126 of a row's largest, and weights times V scales below 2^-33 of the largest such
 * product. The rows' tokens are cut into equal runs over the device and joined. The limits on
 * heads, count and table_stride are the append's; rows are 16-byte aligned here, too. */
typedef struct {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const int32_t* tables;
    const int32_t* lengths; /* [count] */
    void* workspace;        /* 16-byte aligned, mp_kv8_decode_workspace bytes, zeroed before its first use; left as the next call needs it */
    size_t workspace_bytes;
    int32_t type, heads, table_stride, count;
    float scale;
} mp_kv8_decode_args;
size_t mp_kv8_decode_workspace(const mp_kv8_cache* cache, int32_t heads);
int mp_kv8_attention_decode(const mp_kv8_cache* cache, const mp_kv8_decode_args* args, uint32_t* device_error,
                            void* stream);

/* Causal attention of packed chunks of rows (row_offsets, starts, rows as for the
 * append): the row at position p attends to tokens 0 .. p of its sequence, which are in
 * the pages already (the chunk's own rows among them: append first). Calls with at most
 * 148 (row, kv head, 8 query heads) in their `rows` go row by row, others as tiles of
 * rows on the tensor cores, with the same error bounds. */
typedef struct {
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const int32_t* tables;
    const int32_t* row_offsets;
    const int32_t* starts;
    void* workspace; /* as for decode, of mp_kv8_prefill_workspace bytes */
    size_t workspace_bytes;
    int32_t type, heads, table_stride, count, rows;
    float scale;
} mp_kv8_prefill_args;
size_t mp_kv8_prefill_workspace(const mp_kv8_cache* cache, int32_t heads);
int mp_kv8_attention_prefill(const mp_kv8_cache* cache, const mp_kv8_prefill_args* args, uint32_t* device_error,
                             void* stream);
/* Synchronises `stream`, reads and clears *device_error: MP_OK, MP_ERR_BOUNDS,
 * MP_ERR_TIMEOUT or MP_ERR_NONFINITE (the first that applies in the order timeout,
 * bounds, nonfinite). */
int mp_kv8_status(uint32_t* device_error, void* stream);
/* Failure-path tests: the process's next mp_kv8_attention_prefill, if it goes as tiles, gets no V
 * tiles and bounds its waits at `wait_us` microseconds (1 us .. 1 s). They run out, the kernel
 * sets the timeout bit, waits for its products and copies, releases its tensor memory and returns. */
int mp_kv8_inject_wait_timeout(int32_t wait_us);

#ifdef __cplusplus
}
#endif
#endif
