/*
 * kvmem_hip.h -- C ABI of the MI355X (gfx950) KVMem reselect library.
 *
 * This is the device layer that replaces the reference's CUDA stage-in helper
 * (src/adapter/llama-kvmem-stagein.h:12-62, free functions over a global
 * singleton on cudaStreamPerThread) and the host scoring loop of the adapter
 * (src/adapter/llama-memory-kvmem.cpp:2869-2916).  Differences by design:
 *   - explicit context handle instead of the global `g_st` (stagein.cu:60-90);
 *   - explicit HIP stream (default: a stream owned by the context);
 *   - integer status codes (0 = ok) plus kvmem_hip_last_error() instead of
 *     `bool` + stderr (stagein.cu:92-98); no exception crosses this ABI.
 *
 * Pointer lifetimes: every `const void *` / `void *` that names device memory
 * is borrowed for the duration of the call and of the asynchronous work it
 * enqueues on the context stream; the caller keeps it alive until
 * kvmem_hip_sync() (or its own stream synchronisation) returns.  Host arrays
 * passed in (op lists, ids, slots, pointer tables) are copied before the call
 * returns and may be reused immediately.  Calls on one context are not
 * re-entrant: use one context per host thread.
 *
 * Numeric formats use ggml's type codes and block layouts:
 *   Q8_0 (8)  {f16 d; int8 qs[32]}             34 bytes / 32 elements
 *   Q5_0 (6)  {f16 d; u8 qh[4]; u8 qs[16]}     22 bytes / 32 elements
 *   Q4_0 (2)  {f16 d; u8 qs[16]}               18 bytes / 32 elements
 *   F16  (1)  raw half rows (copy)
 * Quantized bytes are bit-identical to ggml's quantize_row_*_ref applied to
 * the F16 rows converted to f32.
 */
#ifndef KVMEM_HIP_H
#define KVMEM_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define KVMEM_HIP_API __attribute__((visibility("default")))
#else
#define KVMEM_HIP_API
#endif

/* ---------------------------------------------------------------- status */
enum kvmem_hip_status {
    KVMEM_HIP_OK = 0,
    KVMEM_HIP_ERR_INVALID = 1,    /* bad argument (shape, alignment, range) */
    KVMEM_HIP_ERR_RUNTIME = 2,    /* a HIP runtime call failed */
    KVMEM_HIP_ERR_NOMEM = 3,      /* device or pinned allocation failed */
    KVMEM_HIP_ERR_STALE = 4,      /* selection epoch/rows mismatch */
    KVMEM_HIP_ERR_UNSUPPORTED = 5, /* type / head_dim not built */
    KVMEM_HIP_ERR_BUSY = 6         /* a shared resource is in use by overlapping work */
};

/* ggml_type codes (ggml.h) for the formats on this path. */
enum kvmem_hip_type {
    KVMEM_TYPE_F32 = 0,
    KVMEM_TYPE_F16 = 1,
    KVMEM_TYPE_Q4_0 = 2,
    KVMEM_TYPE_Q5_0 = 6,
    KVMEM_TYPE_Q8_0 = 8,
    KVMEM_TYPE_BF16 = 30
};

/* Layer combination of per-layer block scores. */
enum kvmem_hip_layer_reduce {
    KVMEM_LAYER_MEAN = 0, /* layer averaging, llama-memory-kvmem.cpp:2910-2913 */
    KVMEM_LAYER_MAX = 1,
    KVMEM_LAYER_SUM = 2
};

typedef struct kvmem_hip_ctx kvmem_hip_ctx;

/* ------------------------------------------------------------- lifetime */

/* Create a context on `device` (HIP ordinal).  Replaces the lazy singleton
 * set-up of kvmem_stagein_gpu_ready (llama-kvmem-stagein.h:12,
 * stagein.cu:319-393).  Scratch grows on demand inside later calls. */
KVMEM_HIP_API int kvmem_hip_create(int device, kvmem_hip_ctx **out);

/* Release every device/pinned buffer the context owns.  Replaces
 * kvmem_stagein_gpu_free (llama-kvmem-stagein.h:13, stagein.cu:395-438). */
KVMEM_HIP_API void kvmem_hip_destroy(kvmem_hip_ctx *ctx);

/* Message of the last failing call on this context ("" if none).  Replaces
 * the stderr line of cuda_ok (stagein.cu:92-98). */
KVMEM_HIP_API const char *kvmem_hip_last_error(const kvmem_hip_ctx *ctx);

/* Use `stream` (a hipStream_t; NULL = the context's own stream) for all
 * later work.  The reference hard-wires cudaStreamPerThread
 * (stagein.cu:100-102). */
KVMEM_HIP_API int kvmem_hip_set_stream(kvmem_hip_ctx *ctx, void *stream);
KVMEM_HIP_API void *kvmem_hip_get_stream(const kvmem_hip_ctx *ctx);

/* Block the host until all work enqueued by this context has finished.
 * Replaces kvmem_stagein_sync (llama-kvmem-stagein.h:27, stagein.cu:615-617). */
KVMEM_HIP_API int kvmem_hip_sync(kvmem_hip_ctx *ctx);

/* Shapes a caller will use, so that later calls of at most these sizes run
 * without allocating device or pinned memory.  Zero fields reserve nothing
 * for their part. */
typedef struct kvmem_hip_reserve_args {
    uint32_t n_layers;         /* scored history layers */
    uint32_t n_blocks;         /* history blocks scored / selected over */
    uint32_t n_head;           /* query heads */
    uint32_t n_head_kv;        /* KV heads */
    uint32_t head_dim;         /* 128 or 256 */
    uint32_t n_q_tokens;       /* query tokens per layer (per-token scorer) */
    uint32_t max_items;        /* largest id / op list passed in one call */
    uint32_t pad0;
    uint64_t h2d_block_bytes;  /* one block over every layer in a host source:
                                  F16 K+V rows (stagein_blocks_host) or packed
                                  rows (stagein_packed_host); 0 = none */
    uint64_t d2h_block_bytes;  /* one block's packed rows over every layer
                                  (stageout_blocks); 0 = none */
    uint64_t move_bytes;       /* bytes one kvmem_hip_move_slots call gathers */
} kvmem_hip_reserve_args;

/* Grow every scratch buffer, ring and upload slot to fit `args`.  Replaces
 * the up-front sizing of kvmem_stagein_gpu_ready(n_f32, n_packed)
 * (llama-kvmem-stagein.h:12, stagein.cu:319-393); buffers only grow, and
 * growing waits for work still reading the old ones. */
KVMEM_HIP_API int kvmem_hip_reserve(kvmem_hip_ctx *ctx, const kvmem_hip_reserve_args *args);

/* Memory the context holds and the number of device/pinned allocations it
 * has made since creation (a call that allocated nothing leaves the count
 * unchanged).  No counterpart in the reference; the singleton's sizes
 * n_f32 / n_q (stagein.cu:60-90) are the nearest. */
typedef struct kvmem_hip_scratch {
    uint64_t device_bytes;
    uint64_t pinned_bytes;
    uint64_t allocations;
} kvmem_hip_scratch;
KVMEM_HIP_API int kvmem_hip_scratch_info(const kvmem_hip_ctx *ctx, kvmem_hip_scratch *out);

/* Enqueue a copy of `n` host bytes to device memory `dst` on the context
 * stream.  Replaces kvmem_stagein_h2d_bytes (llama-kvmem-stagein.h:26,
 * stagein.cu:607-613): n == 0 is a no-op that succeeds, and no fence is
 * taken, so the host buffer stays unchanged until kvmem_hip_sync returns
 * (pinned buffers are read asynchronously; the runtime stages pageable ones
 * before it returns).  Counted in the profiling copy stage and h2d_bytes. */
KVMEM_HIP_API int kvmem_hip_h2d_async(kvmem_hip_ctx *ctx, void *dst, const void *src, size_t n);

/* 1 if `type` can be produced by the stage-in kernels.  Replaces
 * kvmem_stagein_quant_ok (llama-kvmem-stagein.h:16; the reference accepts
 * only Q8_0 and Q4_0, stagein.cu:444-446). */
KVMEM_HIP_API int kvmem_hip_quant_ok(int type);

/* Bytes of a row of n elements of `type` (ggml_row_size), 0 if unsupported
 * or n % 32 != 0.  Used as at llama-memory-kvmem.cpp:2738-2739. */
KVMEM_HIP_API size_t kvmem_hip_row_size(int type, int64_t n);

/* ------------------------------------------------------------- stage-in */

/* One quantize-scatter operation: n_rows rows of n_embd F16 values at `src`
 * (row stride src_stride bytes, 0 = n_embd*2) become n_rows contiguous rows
 * of kvmem_hip_row_size(type, n_embd) bytes at `dst`.  src and dst must be
 * 16-byte aligned, src_stride a multiple of 16, n_embd a multiple of 32. */
typedef struct kvmem_hip_quant_op {
    const void *src;
    void *dst;
    uint32_t n_rows;
    uint32_t n_embd;
    int32_t type;
    uint32_t src_stride;
} kvmem_hip_quant_op;

/* Enqueue a batch of quantize-scatter operations (one kernel launch per
 * output type present).  Replaces the enqueue_k/enqueue_v + flush slab
 * sequence and kvmem_stagein_quantize (llama-kvmem-stagein.h:25,31-40;
 * stagein.cu:579-605, 632-753, 776-840), fused: F16 rows are read once from
 * HBM and written once in the pool's format. */
KVMEM_HIP_API int kvmem_hip_stagein_quant(kvmem_hip_ctx *ctx,
                                          const kvmem_hip_quant_op *ops,
                                          int n_ops);

/* Device-resident F16 block history: for each of K and V, the layer-major
 * array [n_layers][capacity_blocks][block_tokens][n_embd] of halves (one
 * 128-token block of one layer is contiguous, as RawKvStore keeps it per
 * (block, layer), raw_kv_store.hpp:98-117), of which blocks
 * [0, n_blocks) hold history.  v may be NULL (K only). */
typedef struct kvmem_hip_history {
    const void *k;
    const void *v;
    uint32_t n_layers;
    uint32_t n_blocks;
    uint32_t block_tokens;
    uint32_t n_embd_k;
    uint32_t n_embd_v;
    uint32_t last_block_tokens; /* tokens in block n_blocks-1 (0 = full) */
    uint32_t capacity_blocks;   /* blocks per layer in memory (0 = n_blocks) */
} kvmem_hip_history;

/* How the cache expects its rows: the transform the stage-in applies to the
 * F16 history rows before it quantizes them, in the order of the reference's
 * raw-K stage-in (kvmem_stagein_flush for K items, llama-kvmem-stagein.cu:
 * 704-740: widen -> NeoX RoPE -> Walsh-Hadamard -> quantize):
 *   RoPE (K only; rope_neox_kernel stagein.cu:159-178, kvmem/src/host/
 *   rope.cpp:8-45): in every head, for i < n_rot/2, with a = (float)p *
 *   theta[i] at the token's position p,
 *       x'[i]          = x[i]*cos(a) - x[i+n_rot/2]*sin(a)
 *       x'[i+n_rot/2]  = x[i]*sin(a) + x[i+n_rot/2]*cos(a)
 *   (separate IEEE products and sums; cos/sin of the fp32 angle are the
 *   library's own, within one rounding of the exact values); elements at
 *   n_rot and beyond are unchanged.
 *   attn_rot (llama-kvmem-quant.h:22-94; fwht_kernel stagein.cu:104-130):
 *   every run of `width` elements of a head becomes H x, H the orthonormal
 *   Walsh-Hadamard matrix: the run is first scaled by 1/sqrtf(width), then
 *   butterflies (a+b, a-b) of span 1, 2, 4, ... width/2.  The reference
 *   uses width = the largest power of two dividing head_dim (>= 64) for K
 *   (kvmem_hadamard_nrot_k) and 64 for V, on quantized caches.
 * Limits: head_dim 64, 128, 256 or 512 dividing n_embd; n_rot a multiple of
 * 16 up to head_dim; widths 64..512 dividing head_dim; a workgroup chunk of
 * 512 groups may span at most 4096 (row, rotary pair) entries, i.e.
 * (16384 / n_embd + 1) * n_rot / 2 <= 4096. */
typedef struct kvmem_hip_transform {
    uint32_t head_dim;
    uint32_t n_rot;           /* K rotary dims (0 = no RoPE) */
    const float *theta;       /* host [n_rot/2] pair frequencies (rope.cpp:
                                 freq_base^(-2i/n_rot) * freq_scale) */
    uint32_t hadamard_k;      /* K rotation width (0 = none) */
    uint32_t hadamard_v;      /* V rotation width (0 = none) */
    const int32_t *pos0;      /* host, one per staged block of a call: the
                                 position of its token 0 (NULL = block_id *
                                 block_tokens, the block's original start) */
} kvmem_hip_transform;

/* Slot pool: per layer one K and one V tensor of n_slots*block_tokens rows
 * of kvmem_hip_row_size(type, n_embd) bytes (the cache tensors of
 * llama-memory-kvmem.cpp:2736-2742; cell = slot*block_tokens + t,
 * llama-kvmem-batch.cpp:48).  k_layers/v_layers are host arrays of device
 * pointers, 16-byte aligned.  v_layers may be NULL.  xf (may be NULL: rows
 * stored as given) is applied by the block stage-in calls. */
typedef struct kvmem_hip_pool {
    uint32_t n_layers;
    uint32_t n_slots;
    uint32_t block_tokens;
    uint32_t n_embd_k;
    uint32_t n_embd_v;
    int32_t type_k;
    int32_t type_v;
    void *const *k_layers;
    void *const *v_layers;
    const kvmem_hip_transform *xf;
} kvmem_hip_pool;

/* Quantize blocks block_ids[i] of a device-resident history into pool slot
 * slots[i], every layer, K and V.  The single-launch-per-kind replacement
 * of write_block_to_gpu's per-(block, layer) slab items
 * (llama-memory-kvmem.cpp:2726-2791). */
KVMEM_HIP_API int kvmem_hip_stagein_blocks(kvmem_hip_ctx *ctx,
                                           const kvmem_hip_history *hist,
                                           const kvmem_hip_pool *pool,
                                           const uint32_t *block_ids,
                                           const uint32_t *slots,
                                           uint32_t n);

/* Host-resident history, block-major: block b occupies one contiguous span
 * of n_layers*(block_tokens*(n_embd_k+n_embd_v)) halves laid out
 * [layer][K rows then V rows].  When all n_blocks spans lie inside one
 * pinned allocation (hipHostMalloc, torch pin_memory), the quantize kernel
 * reads them over the link itself: one launch, no device staging.  Other
 * host memory is copied with hipMemcpyAsync on a side stream into a device
 * ring and quantized on the context stream as each copy lands.  Replaces
 * the 32 MiB slab H2D of kvmem_stagein_flush (stagein.cu:632-753), which
 * event-synchronises every H2D. */
typedef struct kvmem_hip_host_history {
    const void *base;           /* pinned host memory */
    uint32_t n_layers;
    uint32_t n_blocks;
    uint32_t block_tokens;
    uint32_t n_embd_k;
    uint32_t n_embd_v;
    uint32_t last_block_tokens;
} kvmem_hip_host_history;

KVMEM_HIP_API int kvmem_hip_stagein_blocks_host(kvmem_hip_ctx *ctx,
                                                const kvmem_hip_host_history *hist,
                                                const kvmem_hip_pool *pool,
                                                const uint32_t *block_ids,
                                                const uint32_t *slots,
                                                uint32_t n);

/* Packed host rows: the pool's own row formats kept in pinned host memory
 * per block, as the reference's RawKvStore keeps packed GPU rows per (block,
 * layer) (k_gpu / v_gpu, kvmem/include/kvmem/raw_kv_store.hpp:98-117).
 * Block-major: block b occupies one span of
 *     n_layers * block_tokens * (row_k + row_v) bytes
 * laid out [layer][block_tokens rows of K][block_tokens rows of V], rows of
 * kvmem_hip_row_size(pool type, n_embd) bytes; a block of n_tokens rows
 * uses the first n_tokens rows of each run. */
typedef struct kvmem_hip_packed_host {
    void *base;                 /* pinned host memory */
    uint32_t n_layers;
    uint32_t n_blocks;          /* blocks the memory holds */
    uint32_t block_tokens;
} kvmem_hip_packed_host;

/* Stage-out: copy the packed rows of pool slot slots[i] (every layer, K and
 * V, n_tokens[i] rows) to block block_ids[i] of the packed host store.
 * A store inside one pinned allocation is written by one copy launch on the
 * context stream.  Otherwise the rows are gathered into a device ring in
 * the host layout by one copy launch per 128 MiB batch, then copied
 * device-to-host on the side stream, so a later call's gathers overlap
 * earlier copies.
 * Asynchronous: the host rows are complete after kvmem_hip_sync.  Replaces
 * kvmem_stageout_enqueue / submit / wait (llama-kvmem-stagein.h:40-47,
 * stagein.cu:842-963: gather kernel into a 32 MiB slab, D2H into two
 * pinned slabs) and the per-block harvest of packed rows
 * (llama-memory-kvmem.cpp:2317-2394). */
KVMEM_HIP_API int kvmem_hip_stageout_blocks(kvmem_hip_ctx *ctx, const kvmem_hip_pool *pool,
                                            const kvmem_hip_packed_host *dst,
                                            const uint32_t *block_ids, const uint32_t *slots,
                                            const uint32_t *n_tokens, uint32_t n);

/* Stage-in of packed rows, the reference's live path (write_block_to_gpu:
 * copy_k_gpu / copy_v_gpu into the slab, enqueue_v, flush,
 * llama-memory-kvmem.cpp:2726-2791): the rows go into slot slots[i] of
 * every layer (n_tokens[i] rows), no quantization.  A store inside one
 * pinned allocation is read by one copy launch; otherwise block spans go
 * host-to-device into the device ring on the side stream and one copy
 * launch per batch scatters them.  The pool transform (xf) does not apply: packed rows are
 * already in the cache's form. */
KVMEM_HIP_API int kvmem_hip_stagein_packed_host(kvmem_hip_ctx *ctx,
                                                const kvmem_hip_packed_host *src,
                                                const kvmem_hip_pool *pool,
                                                const uint32_t *block_ids, const uint32_t *slots,
                                                const uint32_t *n_tokens, uint32_t n);

/* Move slots inside the pool: the first n_tokens[i] rows of slot
 * src_slots[i] -> slot dst_slots[i] for every layer, K and V (quantized
 * bytes copied unchanged; the destination's rows past n_tokens[i] keep
 * their bytes).  n_tokens == NULL moves whole slots.  The result is as if
 * every source were read before any destination is written, whatever the
 * overlap.  When sources are distinct and destinations are distinct (a
 * canonical layout's moves) and the layer tensors and rows are 16-byte
 * aligned, chains and cycles of moves are walked in segments and the bytes
 * move once; other sets are gathered to device scratch and scattered,
 * destinations in list order.  Every layer tensor of the pool must be
 * non-null (KVMEM_HIP_ERR_INVALID otherwise, nothing issued).  Replaces the
 * gather/scatter D2D of layout_gpu_slots_by_orig_pos, which moves each
 * block's n_tokens rows (llama-memory-kvmem.cpp:1003-1093). */
KVMEM_HIP_API int kvmem_hip_move_slots(kvmem_hip_ctx *ctx,
                                       const kvmem_hip_pool *pool,
                                       const uint32_t *src_slots,
                                       const uint32_t *dst_slots,
                                       const uint32_t *n_tokens,
                                       uint32_t n);

/* Batched device-to-device byte copies in one launch.  Replaces
 * kvmem_d2d_batched (llama-kvmem-stagein.h:52-53, stagein.cu:965-998);
 * no 8192-op limit. */
KVMEM_HIP_API int kvmem_hip_d2d_batched(kvmem_hip_ctx *ctx,
                                        const void *const *src,
                                        void *const *dst,
                                        const size_t *nbytes,
                                        int n);

/* -------------------------------------------------------------- scoring */

/* Per-token max block scorer on the matrix cores:
 *   s[l][b] = max_{t<n_q_tokens, hq<n_head, j<n_tok(b)}
 *             (q[l][t][hq] . k[l][b][j][hq / (n_head/n_head_kv)]) / sqrt(head_dim)
 * with fp32 accumulation, and scores[b] = reduce_l s[l][b].
 *   q       : device [n_layers][n_q_tokens][n_head][head_dim], bf16 or f16
 *   hist->k : device history (see kvmem_hip_history), n_embd_k must equal
 *             n_head_kv*head_dim
 *   layer_scores (device [n_layers][n_blocks] f32, may be NULL), scores
 *   (device [n_blocks] f32).
 * The reference's scorer is mean-K cosine on the host
 * (llama-memory-kvmem.cpp:2869-2916, per-block std::vector per head); its
 * GQA head map (qh_i = h*g + gi, :2890-2892) is kept. */
typedef struct kvmem_hip_score_args {
    const void *q;
    int32_t q_type;             /* KVMEM_TYPE_BF16 or KVMEM_TYPE_F16 */
    uint32_t n_q_tokens;
    uint32_t n_head;
    uint32_t n_head_kv;
    uint32_t head_dim;          /* 128 or 256 */
    int32_t layer_reduce;       /* kvmem_hip_layer_reduce */
    float *layer_scores;
    float *scores;
} kvmem_hip_score_args;

KVMEM_HIP_API int kvmem_hip_score(kvmem_hip_ctx *ctx,
                                  const kvmem_hip_history *hist,
                                  const kvmem_hip_score_args *args);

/* kvmem_hip_score that allocates nothing: no counterpart in the reference.
 * For callers that cannot allocate (tight serving loops, harnesses that
 * forbid hipMalloc).  Same arguments and the same scores, bit for bit.
 * The scorer's partial maxima (and the per-layer scores when
 * args->layer_scores is NULL) live in a static device array of 8 MiB that
 * every GPU the library runs on holds until the process ends; a call
 * needing more returns KVMEM_HIP_ERR_INVALID before any work (the 256K
 * workload -- 16 layers x 2048 blocks, 4 KV heads, 64 query tokens x 24
 * heads -- needs 2.1 MiB).  Every call on one GPU shares that GPU's array
 * and overwrites it (nothing in it has to start at zero).  One context's
 * calls follow each other (kvmem_hip_set_stream waits for the old stream);
 * a call from another context while the last call on the array has not
 * finished returns KVMEM_HIP_ERR_BUSY with nothing issued (the caller
 * synchronises, or uses kvmem_hip_score).  The array's last
 * user is tracked on the host: two processes on one GPU each have their
 * own array.  A call on a stream under HIP graph capture issues only two
 * kernel launches (no allocation, copy, memset or synchronisation), so it
 * can be captured; the capturing context becomes the array's owner, but
 * the replays run outside the library's view: the caller orders them with
 * its own calls and keeps other contexts' calls on this GPU from
 * overlapping them (such calls are not refused).  Not timed by
 * kvmem_hip_perf_*. */
KVMEM_HIP_API int kvmem_hip_score_noalloc(kvmem_hip_ctx *ctx,
                                          const kvmem_hip_history *hist,
                                          const kvmem_hip_score_args *args);

/* Top-k block selection on device.  From scores[0..n) (device, finite),
 * keep every id in forced[] (host array, the sink / mandatory / recent
 * blocks already charged by the host), then the `need` best remaining ids
 * by score (equal scores: lower id first if tie_lower_index, else higher id
 * first as kvmem_store.cpp:602-609), and write the union in ascending id
 * order to sel_out (host array, capacity n_forced + need); *n_sel receives
 * its length.  Replaces the nth_element fill of pick_topk_ungrouped
 * (kvmem_store.cpp:594-622).  Returns once the selection is on the host:
 * the kernel writes it to the context's coherent pinned buffer and sets a
 * completion word there, on which the calling thread spins (work queued
 * earlier on the context stream, e.g. the scorer, completes first).
 * n <= 1048576 (more than 16384 blocks take a kernel that recomputes
 * the keys from the scores in every radix pass). */
KVMEM_HIP_API int kvmem_hip_topk(kvmem_hip_ctx *ctx,
                                 const float *scores, uint32_t n,
                                 const uint32_t *forced, uint32_t n_forced,
                                 uint32_t need, int tie_lower_index,
                                 uint32_t *sel_out, uint32_t *n_sel);

/* ---------------------------------------------- mean-K cosine (reference) */

/* Mean-K producer: for every listed block and every layer of a device
 * history, k_sum[l][b][e] = fp32 sum of the block's F16 keys in token order
 * and mean_tokens[l][b] = the tokens summed (RawKvStore::capture_mean_f16,
 * kvmem/src/host/raw_kv_store.cpp:184-202; bit-identical sums).  k_sum is
 * device [n_layers][capacity][n_embd_k] f32 (16-byte aligned), mean_tokens
 * device [n_layers][capacity] u32; n_embd_k a multiple of 8, <= 2048. */
KVMEM_HIP_API int kvmem_hip_meank_sums(kvmem_hip_ctx *ctx, const kvmem_hip_history *hist,
                                       const uint32_t *block_ids, uint32_t n,
                                       float *k_sum, uint32_t *mean_tokens);

/* The same producer over a pinned host history (kvmem_hip_host_history,
 * block-major), for a deployment that keeps the history on the host only,
 * as the reference's RawKvStore does (its key sums are made on the host,
 * raw_kv_store.cpp:674-694, 976-1043): the kernel reads the listed blocks'
 * K rows over the link itself.  The whole history must lie inside one
 * pinned allocation (KVMEM_HIP_ERR_UNSUPPORTED otherwise).  k_sum /
 * mean_tokens are [n_layers][capacity_blocks] (0 = hist->n_blocks) as
 * kvmem_hip_meank_sums writes them; the sums are bit-identical. */
KVMEM_HIP_API int kvmem_hip_meank_sums_host(kvmem_hip_ctx *ctx, const kvmem_hip_host_history *hist,
                                            const uint32_t *block_ids, uint32_t n,
                                            uint32_t capacity_blocks, float *k_sum,
                                            uint32_t *mean_tokens);

/* Query-sum producer (the reference's Q harvest into q_sum_,
 * src/adapter/llama-memory-kvmem.cpp:2164-2172 and :2206-2219): for every
 * layer and channel, q_sum[l][e] += q[l][t][e] over the listed tokens in
 * list order, fp32 additions as the reference (bit-identical).
 *   q       device [n_layers][n_tokens][n_embd_q], F32, F16 or BF16
 *   tokens  host list of token indices (the query span; NULL = every token
 *           in order), n_list entries
 *   reset   nonzero: start from 0 (q_sum_ cleared), else add onto q_sum
 *   q_sum   device [n_layers][n_embd_q] f32
 * The caller counts the rows (q_count_) itself. */
KVMEM_HIP_API int kvmem_hip_q_accumulate(kvmem_hip_ctx *ctx, const void *q, int32_t q_type,
                                         uint32_t n_layers, uint32_t n_tokens, uint32_t n_embd_q,
                                         const uint32_t *tokens, uint32_t n_list, int reset,
                                         float *q_sum);

/* Decode-time mean-K producer (the reference's running sum on the GPU,
 * kvmem_meank_zero / kvmem_meank_add, llama-kvmem-stagein.cu:1020-1063):
 * for e < n_embd, acc[e] (+)= K[t][e / head_dim][e % head_dim] over the
 * tokens t = tok0 .. tok0 + n_keep - 1 in token order (fp32 additions,
 * bit-identical to the reference's loop).  K is device memory of k_type
 * F32, F16 or BF16 addressed with byte strides nb0 (element), nb1 (head),
 * nb2 (token), as the ggml K view the reference reads.  acc is device
 * [n_embd] f32, e.g. a row of the key sums kvmem_hip_meank_sums writes;
 * count (device, may be NULL) is that row's token count, increased by
 * n_keep.  reset != 0 starts both from zero (kvmem_meank_zero). */
KVMEM_HIP_API int kvmem_hip_meank_add(kvmem_hip_ctx *ctx, const void *k, int32_t k_type,
                                      uint32_t n_embd, uint32_t head_dim, size_t nb0, size_t nb1,
                                      size_t nb2, uint32_t tok0, uint32_t n_keep, int reset,
                                      float *acc, uint32_t *count);

/* Per-token query window (the rows the per-token scorer reads; the
 * reference keeps only their sum, q_sum_, from the pre-RoPE post-q_norm
 * query rows of its query span, llama-memory-kvmem.cpp:2157-2172,
 * 2206-2219).  Write: for i < n, row rows[i] of `window` (device
 * [capacity][n_head*head_dim] f32, one layer) receives token tokens[i] of
 * the strided device view q (element (d, h, t) at d*nb0 + h*nb1 + t*nb2
 * bytes, as ggml lays Qcur out and the reference reads it,
 * bytes_to_f32_token_major :2066-2090), widened exactly to f32 from F32,
 * F16 or BF16.  Rows must be distinct within a call and below capacity
 * (KVMEM_HIP_ERR_INVALID, nothing issued, otherwise). */
KVMEM_HIP_API int kvmem_hip_q_window_write(kvmem_hip_ctx *ctx, const void *q, int32_t q_type,
                                           uint32_t n_head, uint32_t head_dim, size_t nb0, size_t nb1,
                                           size_t nb2, const uint32_t *tokens, const uint32_t *rows,
                                           uint32_t n, float *window, uint32_t capacity);
/* Gather: out[l][i][:] = window[l][rows[i]][:] for every layer (window
 * device [n_layers][capacity][n_embd_q] f32), converted to out_type (BF16
 * and F16 round to nearest even; F32 copies) -- the [n_layers][n][n_head]
 * [head_dim] query kvmem_hip_score reads. */
KVMEM_HIP_API int kvmem_hip_q_window_gather(kvmem_hip_ctx *ctx, const float *window, uint32_t n_layers,
                                            uint32_t capacity, uint32_t n_embd_q, const uint32_t *rows,
                                            uint32_t n, int32_t out_type, void *out);

/* The reference's retrieval scorer (llama_memory_kvmem::score_retrieval,
 * src/adapter/llama-memory-kvmem.cpp:2869-2916): per block the mean over
 * layers with query rows of the mean over KV heads of
 *   cos(sum_{gi<g} q_sum[h*g+gi] / (q_count*g), k_sum_h / mean_tokens)
 * (denominator sqrt|q|^2 * sqrt|k|^2 + 1e-6), layer and block sums in
 * double; blocks without keys in any layer score 0.
 *   q_sum       device [n_layers][n_head*head_dim] f32 (sums of query rows)
 *   q_count     host   [n_layers] rows summed (0 = layer not scored)
 *   k_sum, mean_tokens as produced by kvmem_hip_meank_sums
 *   scores      device [n_blocks] f32
 * At most 256 layers (KVMEM_HIP_ERR_UNSUPPORTED beyond). */
typedef struct kvmem_hip_meank_args {
    const float *q_sum;
    const uint32_t *q_count;
    const float *k_sum;
    const uint32_t *mean_tokens;
    uint32_t n_layers;
    uint32_t n_blocks;
    uint32_t capacity_blocks;   /* 0 = n_blocks */
    uint32_t n_head;
    uint32_t n_head_kv;
    uint32_t head_dim;          /* 128 or 256 */
    float *scores;
} kvmem_hip_meank_args;

KVMEM_HIP_API int kvmem_hip_score_meank(kvmem_hip_ctx *ctx, const kvmem_hip_meank_args *args);

/* --------------------------------------------- new tokens and attention */

/* The calls of a decode or prefill batch over the pool: kvmem_hip_slot_map
 * (where the batch's tokens go), then per layer kvmem_hip_qkv_rows (their rows
 * into the pool) and kvmem_hip_attention (the batch's queries over the pool's
 * rows).  Lengths, tables and cells stay in device memory and no call waits
 * for the host, so a batch can be captured into a graph and replayed with
 * other contents.  In the reference these are llama.cpp's own graph (the
 * KV cache's cells and its flash attention over quantized rows); the window
 * they work on is the one the reselect path fills. */

/* A table entry without a slot: its keys do not exist. */
#define KVMEM_HIP_NO_SLOT 0xffffffffu

/* Block tables, cells and positions of the new tokens of `n_seq` requests
 * (at most 4096; KVMEM_HIP_ERR_UNSUPPORTED beyond) that share one pool, from
 * their lengths.  Request s has kv_len[s] tokens in its blocks and brings
 * n_new[s] more; block b of request s lives in slot table[s*table_stride + b].
 * Blocks a request starts take the next entries of free_slots, request by
 * request, block by block:
 *   table         new blocks' entries are written, all others stay.  A block
 *                 gets KVMEM_HIP_NO_SLOT when the free list is exhausted; a
 *                 block beyond table_stride has no entry.
 *   kv_len_out[s] = kv_len[s] + n_new[s]
 *   q_start       [n_seq + 1]: first token of each request, then their number
 *   positions[t]  pos0[s] + i for token i of request s (pos0 NULL: kv_len[s])
 *   cells[t]      slot * block_tokens + offset, -1 where the block has no slot
 *   free_used_out entries of free_slots taken so far (free_used + the new ones)
 *   n_missing     blocks that got no entry, of the free list or of the table
 * positions and cells have max_tokens entries; those behind the last token are
 * 0 and -1, and tokens beyond max_tokens get none.  An entry of free_slots or
 * table at or beyond n_slots counts as no slot (one of free_slots is used up all
 * the same, and its block is not counted in n_missing).  Every array is device
 * memory, 4-byte aligned; outputs do not overlap inputs (table is both).  The
 * call is idempotent: repeated with the same inputs it writes the same values. */
typedef struct kvmem_hip_slot_map_args kvmem_hip_slot_map_args;
struct kvmem_hip_slot_map_args {
    uint32_t n_seq;
    uint32_t block_tokens;
    uint32_t n_slots;          /* slots of the pool; n_slots*block_tokens < 2^31 */
    uint32_t table_stride;     /* entries per request; n_seq*table_stride < 2^32 */
    uint32_t max_tokens;
    uint32_t n_free;           /* entries of free_slots */
    const uint32_t *n_new;     /* [n_seq] */
    const uint32_t *kv_len;    /* [n_seq] */
    const int32_t *pos0;       /* [n_seq] or NULL */
    const uint32_t *free_slots;/* [n_free] */
    const uint32_t *free_used; /* [1] */
    uint32_t *table;           /* [n_seq][table_stride] */
    uint32_t *kv_len_out;      /* [n_seq] */
    uint32_t *q_start;         /* [n_seq + 1] */
    int32_t *positions;        /* [max_tokens] */
    int32_t *cells;            /* [max_tokens] */
    uint32_t *free_used_out;   /* [1] */
    uint32_t *n_missing;       /* [1] */
};

KVMEM_HIP_API int kvmem_hip_slot_map(kvmem_hip_ctx *ctx, const kvmem_hip_slot_map_args *args);

/* Rows of new tokens, from a layer's projections to attention's inputs, in
 * one pass.  Per head of q and k:
 *   y = x / sqrt(mean(x^2) + eps) * weight   (weight NULL: y = x)
 *   q_norm / k_norm (if set) receive y: the pre-RoPE rows that
 *     kvmem_hip_q_window_write and the raw history take
 *   RoPE and the Walsh-Hadamard rotation of the transform, as the stage-in
 *     applies them (kvmem_hip_transform; hadamard_k for q and k, hadamard_v
 *     for v), at positions[t]
 *   q_out / k_out (if set) receive the result, contiguous
 *     [n_tokens][heads][head_dim] of out_type
 * With a pool, k and v rows are quantized into row cells[t] of layer `layer`'s
 * tensors (n_embd_k = n_embd_v = n_head_kv*head_dim); cells outside the pool
 * (-1) keep nothing.  Two tokens with the same cell leave one of their rows'
 * bytes in each part of it.  The transform is `xf`, or the pool's where xf is
 * NULL (its pos0 is not read); a pool passed for k and v whose rows the
 * stage-in also writes wants the same transform for both.
 * q, k, v (any may be NULL) are strided device views: element (d, h, t) at
 * d*size + h*nb1 + t*nb2 bytes; 16-byte aligned views are read 16 bytes at a
 * time.  Sums of squares are fp32, whatever a row's magnitude (a row whose
 * squares leave fp32's range is scaled by a power of two first); rows are fp32
 * until they are stored, each output rounded once (nearest even).  Outputs are 16-byte aligned and do not
 * overlap inputs.  head_dim 64, 128, 256 or 512; at most 2^26 tokens. */
typedef struct kvmem_hip_qkv_args kvmem_hip_qkv_args;
struct kvmem_hip_qkv_args {
    const void *q;
    const void *k;
    const void *v;
    int32_t type;              /* of q, k, v: F32, F16 or BF16 */
    int32_t out_type;          /* of q_out, k_out, q_norm, k_norm */
    uint32_t n_tokens;
    uint32_t n_head;
    uint32_t n_head_kv;
    uint32_t head_dim;
    size_t q_nb1, q_nb2;       /* bytes between heads, between tokens */
    size_t k_nb1, k_nb2;
    size_t v_nb1, v_nb2;
    const float *q_weight;     /* device [head_dim], 16-byte aligned */
    const float *k_weight;
    float eps;
    const int32_t *positions;  /* device [n_tokens] (NULL without RoPE) */
    const int32_t *cells;      /* device [n_tokens] (NULL without a pool) */
    const kvmem_hip_transform *xf;
    void *q_out;
    void *k_out;
    void *q_norm;
    void *k_norm;
};

KVMEM_HIP_API int kvmem_hip_qkv_rows(kvmem_hip_ctx *ctx, const kvmem_hip_pool *pool, uint32_t layer,
                                     const kvmem_hip_qkv_args *args);

/* Attention of new tokens over the pool's rows.  Token i of request s (its
 * m = q_start[s+1] - q_start[s] tokens are the last m of its kv_len[s] keys)
 * attends, in query head h, the keys of KV head h / (n_head/n_head_kv):
 *   key j < kv_len[s], and j <= kv_len[s] - m + i if causal, that
 *   table[s*table_stride + j/block_tokens] gives a slot
 *   out = sum_j softmax_j(scale * q . K_j) V_j
 * K_j, V_j being the values row slot*block_tokens + j%block_tokens of layer
 * `layer` stands for (Q4_0, Q5_0, Q8_0 or F16, K and V each their own).  Keys
 * were rotated when they were written (and with hadamard_k, which
 * kvmem_hip_qkv_rows applies to q as well); where the pool's transform has
 * hadamard_v, the output is rotated back to the value's own coordinates.
 * A query without any key gets zeros and lse -inf.  Rows of out and lse behind
 * the last request's tokens are left as they are.  No row of the pool that holds
 * no key reaches a result, whatever it contains; of such rows only row 0 is read
 * (in the place of keys that do not exist).
 *   q       strided device view, element (d, h, t) at d*2 + h*nb1 + t*nb2
 *           bytes, 16-byte aligned (strides too)
 *   out     contiguous [n_tokens][n_head][head_dim], 16-byte aligned
 *   lse     [n_tokens][n_head] log of the softmax's sum, or NULL
 * out, lse and the workspace overlap no input and not one another.
 * q_start NULL: request s has token s.  A request's tokens beyond max_q or
 * n_tokens, and keys beyond max_kv or the table, are not attended (both bounds
 * size the launch; device lengths beyond them never reach out of range).
 * Scores, softmax statistics and sums are fp32.  Rounded on the way, to f16:
 * softmax weights, cached values once they are scaled (so values beyond f16's
 * range become infinite), and in calls with many queries the scaled keys (a
 * key that passes f16's range as a whole by a power of two: it stays finite).
 * The dim of a value that is not finite is not finite either (NaN, or the value)
 * in the rows that attend it, and only in those.
 * head_dim 64, 128 or 256, any n_head that is a multiple of n_head_kv; at most
 * 65535 requests, 2^23 (token, head) rows and 2^31 - 1 keys a request, and
 * requests x max_q within one launch (KVMEM_HIP_ERR_INVALID otherwise: fewer
 * than 2^24 workgroups, 2^23 in calls with many queries); the pool has at least
 * one slot.
 * Keys are split over workgroups when there are few queries; the parts are
 * joined from a workspace: the caller's (kvmem_hip_attention_workspace bytes,
 * 16-byte aligned, contents free) or, where it is NULL, one the context keeps
 * and grows.  A captured call must bring its own (KVMEM_HIP_ERR_INVALID
 * otherwise): graphs that can be replayed at the same time need one each.
 * Results do not depend on the order in which workgroups run. */
typedef struct kvmem_hip_attn_args kvmem_hip_attn_args;
struct kvmem_hip_attn_args {
    const void *q;
    int32_t q_type;            /* F16 or BF16 */
    int32_t out_type;          /* F32, F16 or BF16 */
    size_t q_nb1, q_nb2;       /* bytes between heads, between tokens */
    void *out;
    float *lse;
    uint32_t n_tokens;         /* tokens of q and out */
    uint32_t n_seq;
    uint32_t max_q;            /* most tokens of one request */
    uint32_t max_kv;           /* most keys of one request */
    uint32_t n_head;
    uint32_t n_head_kv;
    uint32_t head_dim;
    uint32_t table_stride;
    const uint32_t *q_start;   /* device [n_seq + 1] or NULL */
    const uint32_t *kv_len;    /* device [n_seq], the new tokens included */
    const uint32_t *table;     /* device [n_seq][table_stride] */
    int32_t causal;
    float scale;               /* 0 = 1/sqrt(head_dim) */
    void *workspace;
    size_t workspace_bytes;
};

/* Workspace bytes of a call with these arguments (0 = none needed). */
KVMEM_HIP_API size_t kvmem_hip_attention_workspace(const kvmem_hip_pool *pool, const kvmem_hip_attn_args *args);
KVMEM_HIP_API int kvmem_hip_attention(kvmem_hip_ctx *ctx, const kvmem_hip_pool *pool, uint32_t layer,
                                      const kvmem_hip_attn_args *args);

/* ------------------------------------ recurrent layers, drafted tokens */

/* What stands between the attention layers of a hybrid model, and what decides
 * how far a step of drafted tokens advances: per recurrent layer
 * kvmem_hip_conv_rows (its projections' short convolution) and
 * kvmem_hip_linear_attention (attention through a state), after the last layer
 * kvmem_hip_verify_draft.  Its n_keep says on the device how many of a request's
 * tokens stay, and both layer calls take it as n_use: a step of drafts is first
 * computed with state_out NULL, then its kept tokens are folded into the states
 * with out NULL.  As for attention, lengths and slots stay in device memory and
 * no call waits for the host.  (The reference leaves these layers to llama.cpp
 * and folds kept tokens into their state with kernels of its patch,
 * patches/llama-kvmem-current.patch:418-474.)
 *
 * Batches: token i of request s is row q_start[s] + i (q_start NULL: request s
 * has row s); requests lie in any order and share no row, and one whose next start
 * is below its own has no tokens.  The first n_use[s] tokens of a request take part
 * (NULL: all); rows of the others, and rows of no request, are left as they are.
 * Tokens beyond max_q or n_tokens take no part: both bounds size the launch and
 * device lengths beyond them never reach out of range.  State of request s is
 * entry slots[s] (NULL: s) of `state`; it goes to the same entry of state_out,
 * which may be `state` itself, also where no token takes part.  state NULL, or a
 * slot at or beyond n_slots: the state starts at zero (and such a slot stores
 * nothing).  Slots of one call are distinct; entries no request names stay as
 * they are.  Otherwise outputs overlap neither inputs nor one another. */

/* Causal depthwise convolution of rows of n_channels, per token t and channel c
 *   y = bias[c] + sum_{j<width} weight[c][j] * x[t - (width-1) + j][c]
 *   y = y / (1 + exp(-y))                            (silu != 0)
 *   y = y / sqrt(sum y^2 + eps)   over runs of norm_dim channels, for the first
 *                                 norm_channels channels (queries and keys)
 * where x before the request's first token are the width-1 rows of its state,
 * oldest first; the new state is the last width-1 rows of both together.
 * Sums are fp32 whatever the rows' type (a run whose squares leave fp32's range
 * is summed in fp64; a run of zeros stays zero), each output is
 * rounded once (nearest even), and states are the rows' own values.
 * width 2 to 8; norm_dim 32, 64, 128, 256 or 512; at most 2^24 channels, 65535
 * requests and 2^26 tokens, and no more workgroups than one launch holds.  x is a
 * strided view, element (c, t) at c*size + t*x_nb bytes; rows, states and outputs that
 * are 16-byte aligned with n_channels a multiple of 8 are moved 16 bytes at a time. */
typedef struct kvmem_hip_conv_args kvmem_hip_conv_args;
struct kvmem_hip_conv_args {
    const void *x;
    int32_t type;              /* of x, states and out: F32, F16 or BF16 */
    int32_t silu;
    size_t x_nb;               /* bytes between tokens */
    uint32_t n_tokens;         /* rows of x and out */
    uint32_t n_seq;            /* at most 65535 */
    uint32_t max_q;            /* most tokens of one request */
    uint32_t n_channels;
    uint32_t width;
    uint32_t n_slots;
    uint32_t norm_channels;    /* a multiple of norm_dim (0: no norm) */
    uint32_t norm_dim;
    const float *weight;       /* device [n_channels][width]; the last tap meets the token itself */
    const float *bias;         /* device [n_channels] or NULL */
    float eps;
    uint32_t pad0;
    const uint32_t *q_start;   /* device [n_seq + 1] or NULL */
    const uint32_t *n_use;     /* device [n_seq] or NULL */
    const uint32_t *slots;     /* device [n_seq] or NULL */
    const void *state;         /* device [n_slots][width-1][n_channels] or NULL */
    void *state_out;           /* the same, or NULL: not stored */
    void *out;                 /* [n_tokens][n_channels], or NULL: the state alone */
};

KVMEM_HIP_API int kvmem_hip_conv_rows(kvmem_hip_ctx *ctx, const kvmem_hip_conv_args *args);

/* Linear attention through a state S [head_dim_k][head_dim_v] per request and
 * head, for each token in order
 *   S = exp(log_decay) S + k (x) d        d = v
 *                                         or, with beta (the delta rule),
 *                                         d = beta (v - exp(log_decay) S^T k)
 *   out = scale * S^T q
 * Query and key head of head h: h / (n_head / n_head_k).
 *   q, k, v  strided device views, element (d, h, t) at d*size + h*nb1 + t*nb2
 *            bytes, 16-byte aligned (strides too); q may be NULL where out is
 *   log_decay, beta  f32, element (h, t) at h*4 + t*nb bytes: an nb of 0 is one
 *            value per head; log_decay NULL: no decay.  -inf clears the state.
 *   state    f32 [n_slots][n_head][head_dim_k][head_dim_v], 16-byte aligned
 *   out      contiguous [n_tokens][n_head][head_dim_v], 16-byte aligned
 * The state, sums and decays are fp32 or wider; out is rounded once.  Calls of
 * few tokens a request go token by token, longer ones by chunks of tokens on
 * the matrix cores: there every factor is scaled by a power of two (states,
 * values and their like column by column) and taken as two f16 parts of 22 bits
 * together, cut 2^-39 below the largest (2^-25 where that is near fp32's smallest),
 * whatever the type of out.
 * A value that is not finite reaches no earlier token, and where only a v is not
 * finite no other dim; what it reaches is not finite either (NaN, or the value).
 * By chunks a d that leaves fp32's range takes its dim's other tokens of the same 64
 * with it.
 * head_dim_k 64, 128 or 256, head_dim_v a multiple of 32 up to 512; at most 4096
 * heads, 65535 requests and 2^26 tokens, and no more workgroups than one launch holds
 * (KVMEM_HIP_ERR_INVALID otherwise).  Calls by chunks keep their chunks' factors
 * in a workspace: the caller's (kvmem_hip_linear_attention_workspace bytes,
 * 16-byte aligned, contents free) or, where it is NULL, one the context keeps
 * and grows.  A captured call that needs one must bring its own
 * (KVMEM_HIP_ERR_INVALID otherwise): graphs that can be replayed at the same time
 * need one each.  Results do not depend on the order in which workgroups run. */
typedef struct kvmem_hip_linear_args kvmem_hip_linear_args;
struct kvmem_hip_linear_args {
    const void *q;
    const void *k;
    const void *v;
    int32_t type;              /* of q, k, v: F32, F16 or BF16 */
    int32_t out_type;          /* F32, F16 or BF16 */
    size_t q_nb1, q_nb2;       /* bytes between heads, between tokens */
    size_t k_nb1, k_nb2;
    size_t v_nb1, v_nb2;
    uint32_t n_tokens;         /* rows of q, k, v and out */
    uint32_t n_seq;
    uint32_t max_q;            /* most tokens of one request */
    uint32_t n_head_k;         /* heads of q and k */
    uint32_t n_head;           /* heads of v, states and out: a multiple of n_head_k */
    uint32_t head_dim_k;
    uint32_t head_dim_v;
    uint32_t n_slots;
    const float *log_decay;
    const float *beta;
    size_t decay_nb, beta_nb;  /* bytes between tokens */
    float scale;               /* 0 = 1/sqrt(head_dim_k) */
    uint32_t pad0;
    const uint32_t *q_start;   /* device [n_seq + 1] or NULL */
    const uint32_t *n_use;     /* device [n_seq] or NULL */
    const uint32_t *slots;     /* device [n_seq] or NULL */
    const float *state;        /* NULL: zero */
    float *state_out;          /* NULL: not stored */
    void *out;                 /* NULL: the state alone */
    void *workspace;
    size_t workspace_bytes;
};

/* Workspace bytes of a call with these arguments (0 = none needed). */
KVMEM_HIP_API size_t kvmem_hip_linear_attention_workspace(const kvmem_hip_linear_args *args);
KVMEM_HIP_API int kvmem_hip_linear_attention(kvmem_hip_ctx *ctx, const kvmem_hip_linear_args *args);

/* Verification of drafted tokens.  Request s has rows q_start[s] to
 * q_start[s+1] - 1 (NULL: max_draft + 1 rows each): row r holds the step's token
 * tokens[r] and the logits of what follows it, so the request's first token is
 * given and the next, at most max_draft, are drafts (rows beyond max_draft + 1 or
 * n_rows are not looked at).  With p = softmax(logits / temperature) and q the
 * draft's distribution (probs; NULL: the draft had probability 1), in order of
 * the rows:
 *   draft x = tokens[r+1] stays where u_accept[r] * q_r(x) < p_r(x)
 * and at the first that does not the next token is drawn from max(p_r - q_r, 0)
 * (from p_r without x where probs is NULL; from p_r where that leaves nothing);
 * where all stay it is drawn from the last row's p.  Drawn from weights w:
 *   the lowest id whose sum_{i <= id} w_i > u_sample[s] * sum_i w_i and w_id > 0
 *   (rounded sums that leave none: the last id with w_id > 0)
 * Exponentials and sums are fp64, so a choice differs from the formula's only
 * where u falls within about 1e-13 of a border.  A temperature that is not above
 * 0 (NULL: 1), and a row with a logit of +inf: the largest logit (the lowest id of
 * equal ones) has probability 1, whatever the draft's distribution.  NaN logits count as -inf;
 * a row of nothing but -inf keeps no draft and gives -1.  A draft outside [0,
 * n_vocab) does not stay.
 *   tokens_out[s]  [max_draft + 1]: the drafts that stay, the next token, -1 behind
 *   n_accepted[s]  drafts that stay
 *   n_keep[s]      n_accepted + 1: the request's tokens that stay (0 without rows)
 *   kv_len_out[s]  kv_len[s] - rows + n_keep: the keys that stay of kv_len, which
 *                  counts all the step's tokens (both may be NULL)
 * Rows of logits and probs are contiguous, element (v, r) at v*size + r*nb bytes,
 * size-aligned.  probs are not
 * negative; only the rows whose draft is tested, and of these the one that refuses,
 * are read.
 * At most 65535 requests, 127 drafts, 2^24 ids.  Parts of rows meet in a workspace
 * (kvmem_hip_verify_draft_workspace bytes, 16-byte aligned): the rules are
 * linear attention's. */
typedef struct kvmem_hip_verify_args kvmem_hip_verify_args;
struct kvmem_hip_verify_args {
    const void *logits;
    const void *probs;
    int32_t type;              /* of logits: F32, F16 or BF16 */
    int32_t probs_type;        /* F32, F16 or BF16 */
    size_t logits_nb, probs_nb; /* bytes between rows */
    uint32_t n_vocab;
    uint32_t n_rows;
    uint32_t n_seq;
    uint32_t max_draft;
    const uint32_t *q_start;   /* device [n_seq + 1] or NULL */
    const int32_t *tokens;     /* device [n_rows] */
    const float *temperature;  /* device [n_seq] or NULL */
    const float *u_accept;     /* device [n_rows], in [0, 1) */
    const float *u_sample;     /* device [n_seq], in [0, 1) */
    const uint32_t *kv_len;    /* device [n_seq] or NULL */
    int32_t *tokens_out;       /* device [n_seq][max_draft + 1] */
    uint32_t *n_accepted;      /* device [n_seq] */
    uint32_t *n_keep;          /* device [n_seq] or NULL */
    uint32_t *kv_len_out;      /* device [n_seq] or NULL; may be kv_len */
    void *workspace;
    size_t workspace_bytes;
};

KVMEM_HIP_API size_t kvmem_hip_verify_draft_workspace(const kvmem_hip_verify_args *args);
KVMEM_HIP_API int kvmem_hip_verify_draft(kvmem_hip_ctx *ctx, const kvmem_hip_verify_args *args);

/* -------------------------------------------------------- self-check */

/* Check, on this device and over every float of their ranges, the two
 * shortcuts the quantizers use for ggml's scale divisions: a / 127 for
 * every non-negative float a (q8_0's d) and 1 / d for every normal |d| <=
 * 2^126 (the id of all three formats); each count is the number of inputs
 * where the shortcut differs from the IEEE quotient (0 expected).  Takes a
 * few hundred milliseconds; no counterpart in the reference. */
KVMEM_HIP_API int kvmem_hip_check_scale_arith(kvmem_hip_ctx *ctx, uint64_t *div127_mismatches,
                                              uint64_t *recip_mismatches);

/* ---------------------------------------------------- failure injection */

/* Kinds of operation kvmem_hip_debug_fail_after can fail. */
enum kvmem_hip_fail_kind {
    KVMEM_HIP_FAIL_ALLOC = 1,  /* a device or pinned allocation */
    KVMEM_HIP_FAIL_COPY = 2,   /* a host<->device copy (table uploads included) */
    KVMEM_HIP_FAIL_LAUNCH = 4  /* a kernel launch */
};

/* Make the nth_op-th later operation of a kind in `kinds` (a mask of
 * kvmem_hip_fail_kind) on this context fail before it is issued: the entry
 * point that reaches it returns an error and kvmem_hip_last_error names
 * it ("...: injected failure"); nothing is enqueued for that operation and
 * injection then switches off.  nth_op = 0 or kinds = 0 switches it off.
 * Host-side only, it never makes a kernel fault.  The reference's callers
 * recover from a failed device call by falling back to host writes
 * (llama-memory-kvmem.cpp:2752-2758, 993-998, 1094-1099); this is how such
 * recovery is tested here.  No counterpart in the reference. */
KVMEM_HIP_API int kvmem_hip_debug_fail_after(kvmem_hip_ctx *ctx, uint32_t kinds, uint64_t nth_op);
/* Operations still to pass before the injected failure (0 = not armed:
 * it fired, or was never set). */
KVMEM_HIP_API uint64_t kvmem_hip_debug_fail_left(const kvmem_hip_ctx *ctx);

/* ------------------------------------------------------------ profiling */

/* Per-stage GPU time (hipEvent pairs on the context stream), the device
 * analogue of the KVMEM_RETR_SUM buckets (llama-memory-kvmem.cpp:2918-2936):
 * score = scoring kernels, topk = selection kernel, set = stage-in kernels
 * (quantizing or packed), copy = kvmem_hip_h2d_async, layout = slot moves
 * and their slot saves, stage_out = packed rows gathered and copied to the
 * host (kvmem_hip_stageout_blocks), plan = the slot plan (the device plan
 * kernel of the engine's apply_retrieval, or the host time of the engine's
 * own diff and slot plan when it plans on the host).  Milliseconds summed
 * over calls since the last reset; counts are numbers of timed calls; a
 * call that fails is not timed.
 * after_score_ms: from the end of a call's scoring to the end of the last
 * stage-in before the next scoring (top-k, the slot plan, moves, stage-in
 * and the idle stream between them); n_after_score such spans.
 * h2d_bytes / d2h_bytes / d2d_bytes: the bytes of kvmem_hip_transfer_get.
 * meank_cos_ms: the mean-K scorer's cosine kernel alone (events attached to
 * its launch), the one kernel of that scorer that streams the key sums;
 * score_ms covers both of its kernels (query, cosine) and the gap between
 * them.  The per-token scorer is one kernel, timed in score_ms the
 * same way. */
typedef struct kvmem_hip_perf {
    double score_ms;
    double topk_ms;
    double set_ms;
    double copy_ms;
    double layout_ms;
    uint64_t n_score;
    uint64_t n_topk;
    uint64_t n_set;
    uint64_t n_copy;
    uint64_t n_layout;
    uint64_t h2d_bytes;
    uint64_t d2d_bytes;
    double after_score_ms;
    uint64_t n_after_score;
    double stage_out_ms;
    double plan_ms;
    uint64_t n_stage_out;
    uint64_t n_plan;
    uint64_t d2h_bytes;
    double meank_cos_ms;
    uint64_t n_meank_cos;
} kvmem_hip_perf;

/* Data this context moved, per direction: [0] host to device, [1] device
 * to host, [2] device to device -- llama_kvmem_transfer_stats
 * (src/adapter/llama-kvmem-hooks.h:127-132), whose copy call sites
 * kvmem_copy_async / kvmem_tensor_set / _get count the same way
 * (src/adapter/llama-kvmem-transfer.h:9-31).  A call is one copy launch or
 * one runtime copy: a stage-in kernel reading pinned host blocks over the
 * link is one host-to-device call of the F16 (or packed) bytes it reads; a
 * slot-move chain walk and its slot saves are one device-to-device call
 * each; a stage-out through the device ring is its gather launches (device
 * to device) and its runtime copies (device to host).  Quantizing kernels
 * reading a device-resident history are compute, not transfers, and launch
 * tables are not counted.  Always counted (perf_enable not needed); cleared
 * by kvmem_hip_perf_reset. */
typedef struct kvmem_hip_transfer_stats {
    uint64_t bytes[3];
    uint64_t calls[3];
} kvmem_hip_transfer_stats;

KVMEM_HIP_API int kvmem_hip_transfer_get(const kvmem_hip_ctx *ctx, kvmem_hip_transfer_stats *out);

KVMEM_HIP_API int kvmem_hip_perf_enable(kvmem_hip_ctx *ctx, int on);
/* Which stages perf_enable times (default all): a mask of
 * KVMEM_PERF_STAGE_* bits.  Each timed stage records two events on the
 * stream, and each event holds the stream idle for a few microseconds, so
 * timing fewer stages perturbs a call less.  after_score_ms needs SCORE and
 * SET. */
#define KVMEM_PERF_STAGE_SCORE 1u
#define KVMEM_PERF_STAGE_TOPK 2u
#define KVMEM_PERF_STAGE_SET 4u
#define KVMEM_PERF_STAGE_COPY 8u
#define KVMEM_PERF_STAGE_LAYOUT 16u
#define KVMEM_PERF_STAGE_STAGE_OUT 32u
#define KVMEM_PERF_STAGE_PLAN 64u
#define KVMEM_PERF_STAGE_MEANK_COS 128u
KVMEM_HIP_API int kvmem_hip_perf_stages(kvmem_hip_ctx *ctx, uint32_t mask);
KVMEM_HIP_API int kvmem_hip_perf_get(kvmem_hip_ctx *ctx, kvmem_hip_perf *out);
/* Zero every bucket, count and transfer counter; a stage a failed call
 * left open is dropped. */
KVMEM_HIP_API void kvmem_hip_perf_reset(kvmem_hip_ctx *ctx);

#ifdef __cplusplus
}
#endif
#endif
