/*
 * gfd_b200.h -- C ABI of the B200-native scattered host->device gather library.
 *
 * Plain C types only (pointers, sizes, integer status codes), so any FFI can bind
 * it: ctypes, cgo, JNI, N-API.  The C++ drop-in API in include/gfd/ (CpuPollingThread,
 * WarpSpecSession, SGWarpSpecSession, device primitives) is implemented on top of
 * these entry points.
 *
 * Data path: sm_100a kernels read the scattered tokens directly out of pinned,
 * device-mapped host memory over PCIe (16-byte vector loads, one warp per >= 512 B
 * span) and store them to HBM; evenly strided layouts may go to the copy engines as 2D
 * copies instead (see GFD_GATHER_DEFAULT).  No host core copies payload bytes (the one
 * exception is opt-in: under GFD_GATHER_PAGEABLE the CUDA driver stages pageable sources).
 *
 * Error behaviour: every entry point returns GFD_OK (0) or a GFD_ERR_* code and
 * never throws; gfd_last_error() gives a one-line reason for the last failure on
 * that context.  Entries are validated before any kernel reads them: a source
 * outside pinned host memory (outside mapped host memory under GFD_GATHER_PAGEABLE),
 * a destination outside device memory of the context's
 * GPU, or a range running past its allocation is rejected with GFD_ERR_INVALID and
 * nothing is copied.
 */
#ifndef GFD_B200_H
#define GFD_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GFD_B200_ABI_VERSION 1

enum {
    GFD_OK = 0,
    GFD_ERR_INVALID = 1,      /* bad argument or entry rejected by validation      */
    GFD_ERR_TIMEOUT = 2,      /* a bounded wait (host or device) expired           */
    GFD_ERR_CUDA = 3,         /* CUDA runtime / driver call failed                 */
    GFD_ERR_NOMEM = 4,        /* host or device allocation failed                  */
    GFD_ERR_UNSUPPORTED = 5,  /* feature unavailable on this device / build        */
    GFD_ERR_STATE = 6         /* call not valid in the object's current state      */
};

/* One scatter-gather entry.  Same layout as gfd::SGEntry
 * (reference include/gfd/copy_engine.h:29-33): dst device pointer, src host
 * pointer, size in bytes; 24 bytes. */
typedef struct gfd_sg_entry {
    uint64_t dst;
    const void* src;
    size_t size;
} gfd_sg_entry;

/* gfd_gather* flags */
#define GFD_GATHER_DEFAULT 0u      /* SM pull, except host->device calls that reduce to at most
                                      three evenly strided groups of rows >= 16 KiB (or of any
                                      length when the call is <= 256 KiB): those go to the copy
                                      engines as 2D copies, which measured faster             */
#define GFD_GATHER_FORCE_CE 1u     /* copy engine (one copy per merged run or strided group)  */
#define GFD_GATHER_AUTO_CE 2u      /* copy engine only for runs >= the context's CE threshold */
#define GFD_GATHER_TRUSTED 4u      /* skip host-side range validation (caller guarantees)   */
#define GFD_GATHER_FORCE_PULL 8u   /* SM pull for every entry, never the copy engine        */
#define GFD_GATHER_PEER_DST 32u    /* gfd_gather_device only: the destination window may lie
                                      in another GPU's memory that this context reaches (peer
                                      access enabled, or a CUDA IPC mapping): the pull reads
                                      over this GPU's host link and stores over NVLink, so a
                                      GPU with a faster host link can fetch rows for a peer   */
#define GFD_GATHER_BULK_STAGE 16u  /* SM pull whose warps move 4 KiB pieces with cp.async.bulk
                                      (host memory -> shared memory -> HBM) instead of 16-byte
                                      loads and stores; implies FORCE_PULL unless FORCE_CE or
                                      AUTO_CE is set; host -> device only (scatter ignores it).
                                      Measured at the same rate as the default pull: the
                                      link's 128-byte read requests bound both             */
#define GFD_GATHER_PAGEABLE 64u    /* gfd_gather / gfd_gather_sync only: a source outside
                                      pinned memory is accepted when every page it covers is
                                      mapped host memory (malloc, mmap, stack) that the driver
                                      does not know as device or managed memory.  A kernel
                                      cannot read such pages, so their runs go to the copy
                                      engine (cudaMemcpyAsync from pageable memory, which the
                                      CUDA driver stages through its own pinned buffers);
                                      pinned entries of the same call still take the SM pull.
                                      Unmapped pages are rejected with GFD_ERR_INVALID before
                                      anything is copied.  Not with GFD_GATHER_TRUSTED
                                      (refused: the source check is what finds pageable
                                      runs).  CpuPollingThread::submit_direct
                                      sets it: the reference's CPU gather reads any host
                                      memory (src/direct_submit.cpp:68-142)                 */

typedef struct gfd_ctx gfd_ctx;
typedef struct gfd_ring gfd_ring;

typedef struct gfd_stats {
    uint64_t calls;           /* gather calls accepted                 */
    uint64_t entries;         /* entries moved                         */
    uint64_t bytes;           /* payload bytes moved                   */
    uint64_t pull_launches;   /* SM-pull kernel launches               */
    uint64_t ce_copies;       /* copy-engine copies issued             */
    uint64_t rejected;        /* calls rejected by validation          */
    uint64_t prep_ns;         /* host time validating entries / building row tables */
    uint64_t launch_ns;       /* host time issuing kernels and copies               */
    uint64_t wait_ns;         /* host time waiting for completion (sync calls)      */
} gfd_stats;

/* ---- context (one per GPU; thread-safe) ------------------------------------
 * Replaces the per-GPU CUDA context + copy-engine setup of the reference
 * (CpuPollingThread::init_copy_engine, src/cpu_polling.cpp:141;
 *  CopyEngineManager::init, src/copy_engine.cpp:13-46).                      */
int gfd_ctx_create(int device, gfd_ctx** out);
int gfd_ctx_destroy(gfd_ctx* ctx);
int gfd_ctx_device(const gfd_ctx* ctx);
const char* gfd_last_error(const gfd_ctx* ctx);
/* Bound for host-side waits of this context (default 10 s). */
int gfd_set_timeout_ns(gfd_ctx* ctx, uint64_t ns);
/* Runs at least this long go to the copy engine under GFD_GATHER_AUTO_CE. */
int gfd_set_ce_threshold(gfd_ctx* ctx, uint64_t bytes);
int gfd_get_stats(const gfd_ctx* ctx, gfd_stats* out);

/* ---- host pools --------------------------------------------------------------
 * Pinned, device-mapped host memory bound to a NUMA node (numa_node < 0: the GPU's
 * own node).  Replaces the reference's pinned pools and hugepage staging
 * (include/gfd/staging_pool.h:29-189; examples/05_multi_gpu_benchmark.cu:217-231).
 * Memory obtained from cudaMallocHost / cudaHostAlloc elsewhere is accepted without
 * registration; gfd_pool_register pins caller-owned (malloc/mmap) memory.        */
int gfd_pool_alloc(gfd_ctx* ctx, size_t bytes, int numa_node, void** out_host);
int gfd_pool_free(gfd_ctx* ctx, void* host);
int gfd_pool_register(gfd_ctx* ctx, void* host, size_t bytes);
int gfd_pool_unregister(gfd_ctx* ctx, void* host);
/* NUMA node that a pool from gfd_pool_alloc is bound to (-1: not bound; any address
 * inside the pool).  An explicit numa_node that the host cannot bind makes
 * gfd_pool_alloc fail with GFD_ERR_INVALID; the GPU's own node (numa_node < 0) is used
 * when the host reports one and binds, else the pool stays unbound.  The reference
 * places pools with set_mempolicy(MPOL_BIND) around cudaMallocHost
 * (examples/05_multi_gpu_benchmark.cu:217-231) and does not report the node.       */
int gfd_pool_numa_node(gfd_ctx* ctx, const void* host, int* node);

/* ---- direct submit -------------------------------------------------------------
 * Gather n entries (host array; copied before return) into device memory.
 * gfd_gather is asynchronous on `stream` (NULL: the context's stream); the entry
 * array may be reused as soon as the call returns.  gfd_gather_sync waits for the
 * bytes to land and reports the host wall-clock latency in microseconds.
 * Replaces CpuPollingThread::submit_direct (reference src/direct_submit.cpp:28-164)
 * and its CPU gather + CE DMA data path (src/parallel_gather.cpp:10-116,
 * src/copy_engine.cpp:89-177).                                                   */
int gfd_gather(gfd_ctx* ctx, const gfd_sg_entry* entries, int64_t n, void* stream, uint32_t flags);
int gfd_gather_sync(gfd_ctx* ctx, const gfd_sg_entry* entries, int64_t n, uint32_t flags,
                    double* elapsed_us);
/* ---- device -> host scatter (reverse path) ------------------------------------
 * The reverse of gfd_gather: entries {dst, src, size} with dst in pinned,
 * device-mapped host memory and src in device memory of the context's GPU (KV-cache
 * offload, spilling activations).  Same kernel, validation, run merging, flags and
 * staging as gfd_gather; each CTA fences at system scope before the completion word,
 * so the bytes are visible to the CPU when gfd_scatter_sync returns (gfd_scatter:
 * when `stream` is synchronised).  No counterpart exists in the reference; it is the
 * future work its architecture notes name (docs/Architecture.md:993).            */
int gfd_scatter(gfd_ctx* ctx, const gfd_sg_entry* entries, int64_t n, void* stream, uint32_t flags);
int gfd_scatter_sync(gfd_ctx* ctx, const gfd_sg_entry* entries, int64_t n, uint32_t flags,
                     double* elapsed_us);

/* Same as gfd_gather, for an entry array already resident in device memory (e.g. written by a
 * routing kernel).  The GPU validates every entry against the context's pools and
 * the window [dst_base, dst_base + dst_bytes), merges contiguous runs (warp ballot +
 * prefix scan) and pulls them.  `status` (may be NULL) receives GFD_OK or
 * GFD_ERR_INVALID after the stream reaches the call; rejected entries are skipped.
 * flags: 0, or GFD_GATHER_PEER_DST (the window is one allocation of a peer GPU that this
 * context can access; the entry array stays in this GPU's memory). */
int gfd_gather_device(gfd_ctx* ctx, const gfd_sg_entry* d_entries, int64_t n, void* dst_base,
                      size_t dst_bytes, void* stream, uint32_t flags);
/* Status of the most recent gfd_gather_device on this context (synchronises). */
int gfd_gather_device_status(gfd_ctx* ctx, int64_t* first_bad_entry);

/* ---- allocation-free device gather --------------------------------------------
 * No counterpart in the reference.  For callers that may not allocate device memory
 * themselves: operator plugins inside an engine that owns all device memory through
 * its own pooling allocator, and latency-critical serving paths where cudaMalloc /
 * cudaFree (which can synchronise the device or fail under a memory budget) must not
 * run.  Same work as gfd_gather_device, without a gfd_ctx and without allocating:
 * its scratch is a fixed device array of about 258 KiB per GPU, held until exit.
 *   - at most GFD_NOALLOC_MAX_ENTRIES entries per call (more: GFD_ERR_INVALID and a
 *     message on stderr); n == 0 is a no-op;
 *   - src_base/src_bytes: a pinned, device-mapped host window holding every source;
 *     dst_base/dst_bytes: a device window holding every destination; entries outside
 *     them are skipped and reported through status_out; each window (and the entry
 *     list) must lie inside one allocation -- one mapping, for cuMemMap'd memory --
 *     or the call returns GFD_ERR_INVALID;
 *   - status_out (NULL or 2 x int64 in device or pinned host memory) receives
 *     {GFD_OK or GFD_ERR_INVALID, first rejected entry or -1} when `stream` reaches
 *     the call;
 *   - runs in the calling thread's current CUDA context; the first call in each
 *     context resolves the scratch array's address (cudaGetSymbolAddress) and keeps it
 *     under the context's driver ID, so a context destroyed and replaced by another
 *     (even one given the same handle) resolves afresh -- make the first call in each
 *     context before any stream capture;
 *   - every call on a GPU shares the one scratch array: calls that overlap on the GPU
 *     race and must be ordered by the caller (same stream, or events).            */
#define GFD_NOALLOC_MAX_ENTRIES 4096
int gfd_gather_device_noalloc(const gfd_sg_entry* d_entries, int64_t n, const void* src_base,
                              size_t src_bytes, void* dst_base, size_t dst_bytes, void* stream,
                              int64_t* status_out);

/* ---- MoE routing front end -----------------------------------------------------
 * Routes `tokens` tokens over `experts` experts from fp32 router logits (device,
 * row-major [tokens x experts]) and gathers the selected rows into per-expert
 * contiguous segments of dst_base, all stream-ordered on the GPU with no host round
 * trip.  Each token picks its k highest logits (ties: lower expert id first; NaN
 * ranks below every number).  The destination holds tokens*k rows of row_bytes:
 * expert 0's rows first, then expert 1's, ..., each expert's rows in ascending token
 * order -- the order of the reference's per-expert SG lists
 * (examples/09_sg_warp_spec.cu:246-276).  Row of token t comes from the pinned host
 * address d_token_src[t] (device array).  Outputs (device): d_counts[e] rows routed to
 * e, d_offsets[e] first row of e's segment, d_entries (tokens*k) the gather list.
 * experts <= 1024, k <= 32.  GFD_MOE_ROUTE_ONLY: route and write the list, skip the
 * gather.  The gather itself is gfd_gather_device (status via
 * gfd_gather_device_status).                                                      */
#define GFD_MOE_ROUTE_ONLY 1u
int gfd_moe_route_gather(gfd_ctx* ctx, const float* d_logits, int64_t tokens, int experts, int k,
                         const uint64_t* d_token_src, size_t row_bytes, void* dst_base,
                         size_t dst_bytes, uint32_t* d_counts, uint32_t* d_offsets,
                         gfd_sg_entry* d_entries, void* stream, uint32_t flags);

/* ---- paged KV cache ------------------------------------------------------------
 * No counterpart in the reference: what a serving program does with the KV blocks that
 * the gathers fetch.  A cache is a set of equal blocks in device memory, each holding
 * block_tokens tokens of K and V for every KV head; a block table gives each sequence its
 * blocks in order, so token j of sequence s lies in block table[s][j / block_tokens] at
 * place j % block_tokens.  Every call is asynchronous on `stream` (NULL: the context's
 * stream), allocates nothing and can be captured into a CUDA graph; lengths, tables and
 * row starts are read on the device when the call runs.
 *
 * What is checked before anything is launched (GFD_ERR_INVALID): shapes, types, strides,
 * alignment, and that every array lies in device memory of the context's GPU.  What only
 * the device knows is checked there: offending parts are skipped and reported by OR-ing
 * GFD_KV_* bits into *status (a device word, or NULL).                              */
enum { GFD_BF16 = 0, GFD_FP16 = 1, GFD_FP32 = 2 };

#define GFD_KV_BAD_PAGE 1u   /* a block id outside [0, blocks): its keys count as masked, a row
                                that would be stored there is not stored                  */
#define GFD_KV_BAD_LENGTH 2u /* kv_len[s] below 0, below the sequence's rows or beyond its
                                table, or more rows than max_q_len: sequence s is skipped, its
                                output rows stay as they were.  row_start not rising from
                                >= 0 to <= rows: the whole call is skipped                 */
#define GFD_KV_GAVE_UP 4u    /* a kernel got nowhere for 10 s and gave up: outputs undefined */

#define GFD_KV_MAX_SEQS 4096

/* Strides count elements, are multiples of 8, and (as the first element's address) keep
 * every head's head_dim elements contiguous and 16-byte aligned. */
typedef struct gfd_kv_cache {
    void* k;               /* block 0, token 0, head 0 of K */
    void* v;               /* the same of V; strides as K's */
    int64_t blocks;
    int64_t block_stride;
    int64_t token_stride;
    int64_t head_stride;
    int32_t block_tokens;  /* a multiple of 16, at most 1024 */
    int32_t heads;         /* KV heads, at most 1024         */
    int32_t head_dim;      /* 64 or 128                      */
    int32_t dtype;         /* GFD_BF16 or GFD_FP16           */
} gfd_kv_cache;

/* The sequences of one call.  Sequence s owns rows row_start[s] .. row_start[s + 1] - 1 of
 * the call's row arrays (possibly none), and they are the last rows of its kv_len[s]
 * tokens: row i of it stands at position kv_len[s] - (its rows) + i.  Rows before
 * row_start[0] and from row_start[seqs] on belong to no sequence and are left alone. */
typedef struct gfd_kv_batch {
    const int32_t* row_start;  /* device, seqs + 1                          */
    const int32_t* kv_len;     /* device, seqs                              */
    const int32_t* table;      /* device, seqs rows of table_width block ids */
    int64_t table_stride;      /* elements from one table row to the next    */
    int64_t rows;              /* rows of the call's row arrays              */
    int32_t seqs;              /* at most GFD_KV_MAX_SEQS                    */
    int32_t table_width;
} gfd_kv_batch;

/* A row array [rows][heads][head_dim]. */
typedef struct gfd_kv_rows {
    void* data;
    int64_t row_stride;
    int64_t head_stride;
} gfd_kv_rows;

/* Appends the batch's rows of K and V to the cache, rotating K (and Q, when given) by
 * position on the way.  The first rot_dim elements of a head are rotated in pairs by the
 * angle position * inv_freq[i], i < rot_dim / 2: elements (i, i + rot_dim / 2), or
 * (2 i, 2 i + 1) with interleaved; angles are formed in 64 bits, the rotation in 32, and
 * each value rounds once.  rot_dim 0: copies.  q_out may be q (same strides).  Two rows of
 * a call must not fall on the same place of the cache (sequences may share blocks that the
 * call does not write). */
typedef struct gfd_kv_append_args {
    gfd_kv_rows k;             /* cache.heads heads, the cache's type                       */
    gfd_kv_rows v;
    gfd_kv_rows q;             /* q_heads heads, the cache's type; q_heads 0: no Q          */
    gfd_kv_rows q_out;
    const float* inv_freq;     /* device, rot_dim / 2                                      */
    const int32_t* positions;  /* device, rows: angles' positions; NULL: the cache position */
    uint32_t* status;
    int32_t q_heads;
    int32_t rot_dim;           /* a multiple of 16, at most head_dim                       */
    int32_t interleaved;
    int32_t _pad;
} gfd_kv_append_args;
int gfd_kv_append(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch,
                  const gfd_kv_append_args* args, void* stream);

/* Attention of the batch's rows over the cache (each KV head serves q_heads / heads query
 * heads in a row).  The row at position p sees key j < kv_len[s] when
 *     j < prefix_len[s]  or  ((!causal or j <= p) and (window == 0 or j > p - window))
 * with score  z = softcap * tanh(scale * q.k / softcap) + alibi[head] * (j - p)  (cap and
 * bias only where given); out = sum exp(z) v / sum exp(z), lse = log sum exp(z) in 32 bits.
 * A row that sees no key, or only scores of -inf, gets zeros and lse = -inf.  What lies in
 * masked places of the cache (unwritten tokens, NaN, infinities) never reaches a result.
 * out is of the cache's type or GFD_FP32 and must not be q.                          */
typedef struct gfd_kv_attend_args {
    gfd_kv_rows q;              /* q_heads heads, the cache's type                          */
    gfd_kv_rows out;            /* q_heads heads, out_dtype                                 */
    float* lse;                 /* device, rows x q_heads contiguous, or NULL               */
    const float* alibi;         /* device, q_heads slopes, or NULL                          */
    const int32_t* prefix_len;  /* device, seqs, or NULL                                    */
    void* workspace;            /* device, 256-byte aligned; calls that may overlap (other
                                   streams, graphs replayed side by side) need one each     */
    size_t workspace_bytes;     /* at least gfd_kv_attend_workspace                         */
    uint32_t* status;
    int32_t q_heads;            /* a multiple of cache.heads                                */
    int32_t out_dtype;
    int32_t max_q_len;           /* the most rows any sequence has; 0: not known             */
    int32_t causal;
    int32_t window;             /* 0: no window                                             */
    float scale;
    float softcap;              /* 0: no cap                                                */
    int32_t _pad;
} gfd_kv_attend_args;
int gfd_kv_attend(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch,
                  const gfd_kv_attend_args* args, void* stream);

/* The same behind a prefix that all sequences share: shared_len tokens whose blocks
 * shared_table (device) lists.  Position j < shared_len is the shared prefix's token j; the
 * batch's lengths and tables describe what follows it, so position shared_len + j is token
 * j of the sequence's own table, and rows stand at shared_len + kv_len[s] - (its rows) + i.
 * The prefix is read once for all rows of the batch, not once per sequence.           */
int gfd_kv_attend_shared(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch,
                         const int32_t* shared_table, int64_t shared_len,
                         const gfd_kv_attend_args* args, void* stream);

/* Bytes of workspace for a call of these shapes (only q_heads, max_q_len of args, rows and
 * seqs of batch, and the cache's shape are read; no array is touched).  Enough for every
 * call of the same cache and q_heads with no more rows, seqs, max_q_len (0 is the most) and
 * shared_len. */
int gfd_kv_attend_workspace(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch,
                            const gfd_kv_attend_args* args, int64_t shared_len, size_t* bytes);

/* Joins partial results over disjoint sets of keys (a resident and a fetched part of a
 * context, say): lse = log sum_i exp(lse_i), out = sum_i exp(lse_i - lse) out_i.  A part
 * with lse_i = -inf is not read into the sum; where every part has it, out is zero and lse
 * -inf.  part i is the row array parts.data + i * part_stride.  out may not be a part. */
typedef struct gfd_kv_merge_args {
    gfd_kv_rows parts;        /* part 0                                                   */
    int64_t part_stride;      /* elements                                                 */
    const float* part_lse;    /* device, parts x rows x heads contiguous                  */
    gfd_kv_rows out;
    float* lse;               /* device, rows x heads contiguous, or NULL                 */
    int64_t rows;
    int32_t part_count;       /* 1 .. 1024                                                */
    int32_t heads;
    int32_t head_dim;         /* 64 or 128                                                */
    int32_t part_dtype;       /* GFD_BF16, GFD_FP16 or GFD_FP32                           */
    int32_t out_dtype;
    int32_t _pad;
} gfd_kv_merge_args;
int gfd_kv_merge(gfd_ctx* ctx, const gfd_kv_merge_args* args, void* stream);

/* ---- GPU-queued submit: descriptor ring consumer ------------------------------
 * Attaches to a gfd::DescriptorQueue written by GPU producers (device.cuh /
 * device_primitives.cuh / sg protocol).  Between gfd_ring_start and gfd_ring_stop a
 * device-resident kernel (the ring agent: one front CTA + `movers` mover CTAs) polls
 * the commit markers, copies committed runs out, clears the markers, advances read_idx,
 * validates and run-merges the descriptors, pulls the bytes and publishes done_idx (and,
 * when attached, per-tile counters or per-list completion).  No host core reads a
 * descriptor or a payload byte.  Replaces the reference's CPU poller + batch processor
 * (src/cpu_polling.cpp:337-436, src/batch_processor.cpp:69-831).
 * `tiled` is a gfd::TiledQueue* whose .base is `queue` (or NULL); `sg` is a
 * gfd::SGTaskQueue* for per-list signalling (or NULL).                          */
int gfd_ring_create(gfd_ctx* ctx, void* queue, void* tiled, void* sg, gfd_ring** out);
int gfd_ring_destroy(gfd_ring* ring);
/* Launches the agent (in resident mode: returns once all its CTAs run, GFD_ERR_TIMEOUT
 * if they cannot become resident within 2 s, so kernels launched afterwards find it on
 * the GPU).  By default the agent leaves after `linger_ns` with nothing committed
 * (cudaDeviceSynchronize and cudaFree wait for every kernel of the context) and a
 * service thread relaunches it when the next commit marker appears; that thread reads
 * no descriptor or payload, only answers range queries (below) and watches one marker
 * while the agent is away.
 * Sources must be pinned, device-mapped host memory and destinations device memory of
 * the context's GPU: the agent checks every descriptor against ranges it has cached
 * and asks the host once about a range it has not seen (rejected descriptors are
 * skipped, counted and their run still completes). */
int gfd_ring_start(gfd_ring* ring);
/* Stops the agent after it has drained every slot committed so far.  Once stopped (and
 * in gfd_ring_destroy) the ring no longer reads the queue, so the caller may free it. */
int gfd_ring_stop(gfd_ring* ring);
/* Without gfd_ring_start: one drain pass from the calling thread (the descriptors are
 * read and validated on the host; one pull kernel per committed run); *launched = number
 * of drains launched.  While the ring runs it does nothing (the agent consumes). */
int gfd_ring_poll(gfd_ring* ring, int* launched);
/* Waits until done_idx >= target (bounded by the context timeout). */
int gfd_ring_wait(gfd_ring* ring, uint64_t target);
int gfd_ring_counters(const gfd_ring* ring, uint64_t* consumed, uint64_t* drains,
                      uint64_t* bytes);
/* Agent settings, before gfd_ring_start (the environment variables GFD_RING_MOVERS,
 * GFD_RING_LINGER_NS and GFD_RING_RESIDENT set the same at gfd_ring_create):
 * movers: mover CTAs (1..32, 0: 8); linger_ns: idle time before the agent leaves
 * (default 20 us); resident != 0: the agent stays until gfd_ring_stop (bounded by the
 * context timeout when idle) -- for producer kernels that occupy every SM and wait on
 * done_idx; the application then synchronises with streams or events, because
 * cudaDeviceSynchronize waits for the agent too, and loads its kernels before the ring
 * starts (cudaFuncGetAttributes, or CUDA_MODULE_LOADING=EAGER): with lazy loading, the
 * first launch of a kernel waits for the kernels already running, the agent included.
 * No counterpart in the reference, whose consumer is a host thread.                  */
int gfd_ring_configure(gfd_ring* ring, uint32_t movers, uint64_t linger_ns, int resident);
/* Declares a window the agent may trust without asking (pinned host memory as a source,
 * device memory as a destination); bytes == 0: the whole allocation holding ptr.
 * CpuPollingThread::start declares its constructor's gpu_base / cpu_base this way.    */
int gfd_ring_allow(gfd_ring* ring, const void* ptr, size_t bytes);
/* What the agent did so far. */
typedef struct gfd_ring_agent_stats_t {
    uint64_t launches;      /* agent launches (start + relaunches after idle exits)        */
    uint64_t queries;       /* range queries the agent asked the host                      */
    uint64_t rejected;      /* descriptors rejected by validation                          */
    uint64_t timeouts;      /* bounded waits of the agent that gave up                     */
    uint64_t idle_exits;    /* launches that ended after linger_ns / the idle bound         */
    uint64_t stop_exits;    /* launches that ended on gfd_ring_stop                        */
    uint64_t error_exits;   /* launches that ended on a wait that gave up                  */
    uint64_t resident;      /* 1 if the ring is configured resident                        */
    /* last launch, nanoseconds after its front CTA started (0: did not happen):           */
    uint64_t last_first_batch_ns;  /* first batch published                                 */
    uint64_t last_done_ns;         /* last batch completed (done_idx published)            */
    uint64_t last_exit_ns;         /* launch ended                                          */
} gfd_ring_agent_stats_t;
int gfd_ring_agent_stats(const gfd_ring* ring, gfd_ring_agent_stats_t* out);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* GFD_B200_H */
