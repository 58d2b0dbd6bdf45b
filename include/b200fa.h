/*
 * b200fa.h -- C ABI of libb200fa.so, the sm_100a flash-attention forward.
 *
 * One operator: non-causal grouped-query attention forward,
 *     O[b,h] = softmax(Q[b,h] K[b,kv(h)]^T * scale) V[b,kv(h)],
 *     kv(h) = h / (Hq / Hkv),
 * with FP16 Q [B,Hq,Nq,128], K and V [B,Hkv,Nk,128] and FP16 normalized
 * O [B,Hq,Nq,128], all contiguous (BHND, "BNSD" in torch_npu terms).
 *
 * This library replaces the native call pair of the reference's CCE
 * backends,
 *   aclnn<Op>GetWorkspaceSize(q, k, v, q_block, k_block, q_l1, groups,
 *                             capture, phase, [gray], sp, partial, trace,
 *                             stats, running, output, &ws_size, &executor)
 *   aclnn<Op>(workspace, ws_size, executor, stream)
 * bound in backends/cce_fa_nqkq_nz_resident_v13_q768_pool_i4_p128/binding.py:20-26
 * and called at binding.py:72-80 (the FP32 twin,
 * backends/cce_fa_nk_nz_vector_fp32_v5_sumpack/binding.py, has the same
 * shape).  The ACLNN executor and its tiling (op_host/*.cpp:53-89) collapse
 * into the plain-pointer call b200fa_fwd below; the host-side shape checks of
 * binding.py:87-98 and op_host/*.cpp:8-19 become the negative return codes.
 *
 * Conventions
 *   - All tensor pointers are CUDA device pointers owned by the caller; the
 *     library allocates no device memory and keeps no per-call state.
 *   - Calls are asynchronous on the caller's stream (cudaStream_t passed as
 *     void*, NULL = legacy default stream); nothing synchronizes implicitly
 *     except b200fa_read_status.
 *   - Return value 0 = success, negative = argument validation error (no
 *     CUDA call was made), positive = CUDA runtime error code from a launch
 *     or attribute call.  b200fa_last_error_string() describes the last
 *     failure on the calling thread.
 *   - Device-side failures (a bounded wait that ran out) do not abort the
 *     kernel's caller: the kernel records a status word in the workspace
 *     and returns; b200fa_read_status() reads it.
 */
#ifndef B200FA_H_
#define B200FA_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Variant selector: softmax arithmetic of the two shipped kernels.
 * B200FA_VARIANT_FP16 mirrors the reference CCE FP16 kernel
 *   (backends/cce_fa_nqkq_nz_resident_v13_q768_pool_i4_p128): row sums in
 *   FP16 partial sums of the FP16 P (FP32 exponentials).
 * B200FA_VARIANT_FP32 mirrors the CCE FP32 kernel
 *   (backends/cce_fa_nk_nz_vector_fp32_v5_sumpack): FP32 softmax throughout.
 * Both keep P in FP16 for the tensor-core PV product and accumulate O in
 * FP32 in tensor memory. */
#define B200FA_VARIANT_FP16 0
#define B200FA_VARIANT_FP32 1

/* Status / error codes. */
#define B200FA_OK                 0
#define B200FA_ERR_NULL          -1   /* a required pointer is NULL            */
#define B200FA_ERR_HEAD_DIM      -2   /* D != 128                              */
#define B200FA_ERR_SHAPE         -3   /* B, Hq, Hkv, Nq or Nk <= 0             */
#define B200FA_ERR_GROUPING      -4   /* Hq % Hkv != 0                         */
#define B200FA_ERR_TOO_LARGE     -5   /* Nq, Nk or unit count >= 2^31          */
#define B200FA_ERR_UNIT_RANGE    -6   /* unit range outside [0, num_units]     */
#define B200FA_ERR_ALIGNMENT     -7   /* a tensor pointer is not 16-B aligned  */
#define B200FA_ERR_WORKSPACE     -8   /* workspace NULL, misaligned or small   */
#define B200FA_ERR_VARIANT       -9   /* unknown variant                       */
#define B200FA_ERR_SCALE        -10   /* scale not finite or not positive      */
#define B200FA_ERR_OPTIONS      -11   /* malformed b200fa_options              */
#define B200FA_ERR_NO_DRIVER    -12   /* cuTensorMapEncodeTiled unavailable    */
#define B200FA_ERR_TENSOR_MAP   -13   /* cuTensorMapEncodeTiled rejected a map */
#define B200FA_ERR_DTYPE        -14   /* unknown element type                  */
#define B200FA_ERR_PAGE_SIZE    -15   /* page size not a power of two, 8..2^20 */
#define B200FA_ERR_STRIDE       -16   /* a stride that the kernels cannot read */
#define B200FA_ERR_ROTARY       -17   /* malformed rotary description          */

/* Device status word values (b200fa_read_status, status[0]). */
#define B200FA_DEV_OK             0
#define B200FA_DEV_TIMEOUT        1   /* a bounded mbarrier wait ran out       */
/* Checking build only (libb200fa_debug.so, compiled with B200FA_DEBUG): */
#define B200FA_DEV_BOUNDS         2   /* a coordinate, index or layout check failed;
                                         site low byte = 0x80 + check number    */
#define B200FA_DEV_PHASE          3   /* the roles' key-block counts disagreed at exit */

#define B200FA_DEV_PAGE           4   /* paged attention: a request's block table ended
                                         early or named a page outside the cache; the
                                         keys there were read as zeros          */

/* Element types of the serving operators. */
#define B200FA_DTYPE_FP16         0
#define B200FA_DTYPE_BF16         1
#define B200FA_DTYPE_FP32         2   /* b200fa_rotary only                     */

/* Option flags (b200fa_options.flags). */
#define B200FA_FLAG_TRACE          1u /* write one trace record per CTA        */
/* Test-only: softmax group 1 (the odd key blocks, in both CTAs of every
 * pair) withholds its first P-ready arrival, so the PV issuer's bounded
 * wait runs out and the kernel reports B200FA_DEV_TIMEOUT.  Used by the
 * failure-detection test only. */
#define B200FA_FLAG_TEST_WITHHOLD_P 2u
/* Debug, checking build only (libb200fa_debug.so; the product build ignores
 * the flag): both CTAs of the first pair record SM-clock timestamps of their
 * softmax, MMA-issuer / forwarder and TMA threads for the first
 * B200FA_TIMELINE_BLOCKS key blocks of their first work item into the
 * timeline area of the workspace (pipeline analysis). */
#define B200FA_FLAG_TIMELINE       4u
/* Debug capture (the counterpart of the reference's `capture` attribute,
 * binding.py:39-41, vector_output.h:94-106): per key block and query row the
 * kernel writes its online-softmax state into b200fa_options.capture, FP32,
 * laid out [plane][b*Hq + hq][key block][query row] with planes
 *   0  m      reference maximum after the block (log2 domain: scores times
 *             scale*log2(e)); it moves only when a block maximum exceeds it
 *             by more than 8 (lazy rescaling)
 *   1  l      running row sum after the block, relative to m
 *   2  alpha  factor applied to l and O at this block (2^(m_old - m_new);
 *             1 when m did not move, 0 at the first block)
 *   3  z      the block's own row sum, relative to m
 * followed by the O plane, [b*Hq + hq][key block][query row][128]:
 *   O after the block's P V product (unnormalised, relative to m); the
 *   block's own partial product is O_j - alpha_j * O_(j-1).
 * The reference's capture holds the same (m, l, alpha, z, O) per packet.
 * Key blocks are B200FA_BLOCK_KEYS keys wide.  Rows of the unit range only;
 * other entries are left untouched.  The buffer must be 16-byte aligned;
 * size: b200fa_capture_bytes() = 528 * B * Hq * ceil(Nk / 128) * Nq.  The
 * capture serialises each block's softmax with its P V product: a debug
 * mode, not a fast path. */
#define B200FA_FLAG_CAPTURE        8u
/* Test-only, checking build only: the producer offsets its first Q tile's
 * row coordinate past the end of the problem; the bounds check catches it
 * before the copy is issued and the kernel reports B200FA_DEV_BOUNDS.  The
 * product build ignores the flag (it has no checks and never offsets). */
#define B200FA_FLAG_TEST_BOUNDS   16u
/* Causal mask (top-left aligned, as torch's is_causal): query row i attends
 * keys 0..i only.  Key blocks past the diagonal of a work item's last query
 * block are skipped; the block that crosses a row's diagonal is masked.
 * Runs separate kernels (b200_fa_fp{16,32}_causal_kernel); not combined
 * with B200FA_FLAG_CAPTURE (B200FA_ERR_OPTIONS). */
#define B200FA_FLAG_CAUSAL        32u
/* Sliding window with sinks, on top of B200FA_FLAG_CAUSAL (required): query
 * row i attends keys i - window < j <= i and the first `sinks` keys j <= i
 * (b200fa_options.window >= 1, .sinks >= 0).  A row that sees no key (Nq > Nk)
 * gets zeros.  Key blocks that no row of a work item sees are not read, nor is
 * V of any key that none of them sees.
 * Runs a separate kernel (b200_fa_window_kernel), the same for both variants:
 * softmax sums in FP32. */
#define B200FA_FLAG_WINDOW        64u
#define B200FA_BLOCK_KEYS        128

typedef struct b200fa_options {
    uint32_t struct_size;   /* sizeof(b200fa_options); 16 (no capture fields)
                               and 32 (no window fields) are accepted too    */
    uint32_t flags;         /* B200FA_FLAG_*                                  */
    uint32_t timeout_us;    /* bound of every device-side wait; 0 = 2 s       */
    int32_t  max_ctas;      /* cap on the persistent grid (CTAs; rounded down
                               to whole pairs, at least one pair); <= 0 = one
                               pair per TPC                                  */
    float*   capture;       /* B200FA_FLAG_CAPTURE: device buffer             */
    uint64_t capture_bytes; /* its size, >= b200fa_capture_bytes(...)        */
    int32_t  window;        /* B200FA_FLAG_WINDOW: keys of the window, >= 1   */
    int32_t  sinks;         /* B200FA_FLAG_WINDOW: first keys always visible  */
} b200fa_options;

/* Workspace layout (bytes, 256-B aligned, zeroed once by the owner):
 *   [0, 256)       status header: u32 status, u32 site, u32 cta, u32 spare...
 *                  site = (pair rank << 16) | (warp << 8) | barrier slot of
 *                  the first wait that ran out
 *   [256, 256 + 32 * B200FA_MAX_CTAS)
 *                  trace records, one per CTA (B200FA_FLAG_TRACE):
 *                  {u32 smid, u32 items, u64 t_start_ns, u64 t_end_ns,
 *                   u32 pair rank, u32 0}; both CTAs of a pair count the
 *                  pair's items
 *   [B200FA_WS_TIMELINE_OFFSET, + B200FA_WS_TIMELINE_BYTES)
 *                  timeline (B200FA_FLAG_TIMELINE): u64 clock64 stamps,
 *                  [pair rank 0..1][role 0..B200FA_TIMELINE_ROLES-1]
 *                  [block 0..B200FA_TIMELINE_BLOCKS-1][event 0..7], roles =
 *                  softmax warps 0-7, MMA issuers (rank 0) / forwarder
 *                  (rank 1), TMA.
 * The status is sticky: it stays set until b200fa_reset_status. */
#define B200FA_WS_HEADER_BYTES 256u
#define B200FA_WS_TRACE_BYTES   32u
#define B200FA_MAX_CTAS       1024
#define B200FA_TIMELINE_BLOCKS  48u
#define B200FA_TIMELINE_ROLES   10u
#define B200FA_WS_TIMELINE_OFFSET (B200FA_WS_HEADER_BYTES + B200FA_WS_TRACE_BYTES * B200FA_MAX_CTAS)
#define B200FA_WS_TIMELINE_BYTES  (2u * B200FA_TIMELINE_ROLES * B200FA_TIMELINE_BLOCKS * 8u * 8u)

/* Number of work units: (b, hq, 128-row query block) triples, linearised as
 * ((b * Hq) + hq) * ceil(Nq / 128) + qb -- the order of the reference's
 * task split, cce_task.h:28-35 / panel_kernel.h:264-274.  Returns a negative
 * validation code for non-positive sizes. */
int64_t b200fa_num_units(int64_t B, int64_t Hq, int64_t Nq);

/* Contiguous near-equal split of [0, total) into `parts` ranges, remainder to
 * the first parts -- the semantics of cce::PartitionContiguous
 * (cce_task.h:28-35).  Writes part `index`'s [begin, end).  0 or
 * B200FA_ERR_UNIT_RANGE. */
int b200fa_partition(int64_t total, int32_t parts, int32_t index,
                     int64_t* begin, int64_t* end);

/* Bytes of workspace b200fa_fwd needs (header + trace area for the maximum
 * grid).  Replaces aclnn<Op>GetWorkspaceSize (binding.py:72-77); the value
 * does not depend on the shape beyond validation.  Negative on invalid
 * arguments. */
int64_t b200fa_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq,
                              int64_t Nk, int64_t D, int32_t variant);

/* Attention forward over work units [unit_begin, unit_end) (the whole
 * problem is [0, b200fa_num_units(B, Hq, Nq))).  Rows of O outside the range
 * are not written.  Replaces aclnn<Op> (binding.py:72-80) and the tiling
 * kernel launch (op_host/*.cpp:53-89, panel_kernel.h:216-343). */
int b200fa_fwd(const void* q, const void* k, const void* v, void* o,
               int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq, int64_t Nk,
               int64_t D, float scale, int32_t variant,
               int64_t unit_begin, int64_t unit_end,
               void* workspace, uint64_t ws_bytes, void* stream);

/* b200fa_fwd with options (trace records, wait bound, grid cap, test
 * flags).  opts may be NULL. */
int b200fa_fwd_ex(const void* q, const void* k, const void* v, void* o,
                  int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq, int64_t Nk,
                  int64_t D, float scale, int32_t variant,
                  int64_t unit_begin, int64_t unit_end,
                  void* workspace, uint64_t ws_bytes, void* stream,
                  const b200fa_options* opts);

/* Synchronizes `stream`, then copies the 4-word status header of `workspace`
 * into status[0..3] = {status, site, cta, spare}.  Returns 0 or a CUDA error. */
int b200fa_read_status(const void* workspace, void* stream, uint32_t* status);

/* Clears the status header (async on `stream`). */
int b200fa_reset_status(void* workspace, void* stream);

/* Kernel symbol of a variant ("b200_fa_fp16_kernel" / "b200_fa_fp32_kernel"),
 * the names the harness profiler matches backends by; NULL for a bad id. */
const char* b200fa_kernel_name(int32_t variant);

/* Host-side work-item plan (no GPU): item `index` of the range
 * [unit_begin, unit_end) as {bh, first q-block, count (1..2)}: up to two
 * consecutive query blocks of one head, one per CTA of a pair.  Returns
 * the number of items, or a negative code. */
int64_t b200fa_plan_item(int64_t B, int64_t Hq, int64_t Nq,
                         int64_t unit_begin, int64_t unit_end, int64_t index,
                         int64_t* bh, int64_t* qblock, int64_t* count);

/* Bytes of the B200FA_FLAG_CAPTURE buffer:
 * 528 * B * Hq * ceil(Nk / B200FA_BLOCK_KEYS) * Nq (four scalar FP32 planes
 * and the 128-float O plane).  Negative on invalid sizes. */
int64_t b200fa_capture_bytes(int64_t B, int64_t Hq, int64_t Nq, int64_t Nk);

/* Description of the last error on the calling thread ("" if none). */
const char* b200fa_last_error_string(void);

/* Library version string. */
const char* b200fa_version(void);

/* Test hook, no counterpart in the reference: evaluates the softmax's two
 * exponential forms elementwise on n device floats, asynchronously on
 * `stream` -- poly[i] = the FMA-pipe 2^x the kernels use for part of every
 * row (Cody-Waite split, degree-3 minimax polynomial, input clamped at -120),
 * mufu[i] = the MUFU ex2.approx.ftz form they use for the rest.  Lets a test
 * check the compiled device function against exp2 over the softmax's input
 * range.  0, B200FA_ERR_NULL, B200FA_ERR_SHAPE (n < 0 or >= 2^31) or a CUDA
 * error code. */
int b200fa_test_exp2(const float* x, float* poly, float* mufu, int64_t n, void* stream);

/* Allocation-free forward.  This entry point has no counterpart in the
 * reference; it exists for callers that cannot hand the library a
 * workspace: a C or FFI host with no device allocator of its own, a runtime
 * that has reserved the whole device pool for itself and forbids side
 * allocations, or a latency-critical path that must not call cudaMalloc
 * (which can synchronize the device).  Same computation and arguments as
 * b200fa_fwd_ex minus the workspace: the status header and trace records
 * live in a static device array of B200FA_NOALLOC_SCRATCH_BYTES bytes
 * (256-byte header + trace records for at most B200FA_NOALLOC_TRACE_CTAS
 * CTAs), one copy on every device that loads the library, held until the
 * process exits.  Nothing is allocated: no cudaMalloc, cudaFree or
 * allocating library routine is called.
 *   - The first call on a device resolves that device's copy of the array
 *     (cudaGetSymbolAddress) and sets the kernel attributes; make that first
 *     call before any stream capture.
 *   - Each call clears the status header on `stream` before its launch.
 *     All calls share the array: calls that overlap on the GPU (e.g. on
 *     different streams) race on the status header and trace records.
 *   - A call whose scratch need exceeds the array -- tracing
 *     (B200FA_FLAG_TRACE) with a persistent grid of more than
 *     B200FA_NOALLOC_TRACE_CTAS CTAs -- is rejected with
 *     B200FA_ERR_WORKSPACE before anything is launched; cap the grid with
 *     opts->max_ctas or trace less.  B200FA_FLAG_TIMELINE is not supported
 *     here (its area alone exceeds the array) and is rejected the same way.
 *   - A call with an empty unit range launches nothing but still clears the
 *     status header, so a status read afterwards describes this call.
 *   - scratch_out (may be NULL) receives the device address of this
 *     device's scratch, for b200fa_read_status / b200fa_reset_status. */
#define B200FA_NOALLOC_TRACE_CTAS 128u
#define B200FA_NOALLOC_SCRATCH_BYTES \
    (B200FA_WS_HEADER_BYTES + B200FA_WS_TRACE_BYTES * B200FA_NOALLOC_TRACE_CTAS)
int b200fa_fwd_noalloc(const void* q, const void* k, const void* v, void* o,
                       int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq, int64_t Nk,
                       int64_t D, float scale, int32_t variant,
                       int64_t unit_begin, int64_t unit_end,
                       void* stream, const b200fa_options* opts, void** scratch_out);

/* ------------------------------------------------------------------------
 * Serving: a paged K/V cache, the tables of a step, and the attention that
 * reads them (additions; the reference has no cache).
 *
 * A cache is two tensors of pages, K and V, [num_pages][page_size][Hkv][128]
 * in any order of the outer three dimensions (strides in elements, multiples
 * of 8; the head dim is contiguous).  Token i of request r lives at offset
 * i % page_size of page block_table[r][i / page_size]; its slot is
 * page * page_size + offset.  Page sizes are powers of two. */

/* The tables of one step, from request lengths, on the device.  Request r
 * holds ctx_lens[r] tokens in ceil(ctx/page_size) pages and adds new_lens[r];
 * the pages it needs beyond those are taken from the end of the free list
 * (free_pages[*free_count - 1] first), in request order.  Writes
 *   block_table[r][...]  the entries of the new pages (others untouched)
 *   slots, positions     [num_tokens], requests after one another; places
 *                        behind the last token get slot -1, position 0
 *   cu_q [requests + 1]  prefix sums of new_lens
 *   kv_lens [requests]   ctx + new
 *   free_left, status    [1]: pages left; 0, or 1 the free list is too short,
 *                        2 a request outgrows its table row (width) or
 *                        2^31 - 1 tokens, 3 more new tokens than
 *                        num_tokens.  With a status other
 *                        than 0 nothing is handed out: every slot is -1,
 *                        kv_lens = ctx_lens, free_left = *free_count, the
 *                        table is untouched.
 * Lengths below 0 count as 0.  No output may overlap an input (the table
 * apart).  At most B200FA_MAX_REQUESTS requests.  One launch on `stream`. */
#define B200FA_MAX_REQUESTS 4096
int b200fa_build_tables(const int32_t* ctx_lens, const int32_t* new_lens, int32_t requests, int32_t* block_table,
                        int64_t table_stride, int32_t width, const int32_t* free_pages, int64_t free_capacity,
                        const int32_t* free_count, int32_t page_size, int64_t* slots, int32_t* positions,
                        int64_t num_tokens, int32_t* cu_q, int32_t* kv_lens, int32_t* free_left, int32_t* status,
                        void* stream);

/* Rotary positions.  freq[i] is pair i's angle per position in turns, as a
 * 64-bit binary fraction (0.64 fixed point); the angle of position p is
 * p * freq[i] mod 1 (the product is exact; the frequency's own rounding,
 * 2^-65 turns, counts p times).  layout 0: pair (i, i + rot/2);
 * 1: pair (2i, 2i + 1).  Elements rot.. of a head are copied.  magnitude
 * multiplies the rotated ones; inverse turns by the negative angle. */
typedef struct b200fa_rotary_desc {
    uint32_t        struct_size;
    int32_t         dim;        /* head dim, a multiple of 16, <= 1024          */
    int32_t         rot;        /* rotated elements, a multiple of 16, <= dim   */
    int32_t         layout;
    int32_t         inverse;
    float           magnitude;
    const uint64_t* freq;       /* device, [rot / 2]                            */
} b200fa_rotary_desc;

/* out = rotation of x, both [batch][n][heads][dim] with strides in elements
 * (batch, n, heads; multiples of 16 bytes; the last dimension contiguous).
 * positions: device int32 or int64 (pos_bits 32 / 64), [n] with pos_stride
 * elements between batches (0: shared), or NULL for 0 .. n-1.  out may be x. */
int b200fa_rotary(const void* x, void* out, int64_t batch, int64_t n, int64_t heads, const int64_t* x_strides,
                  const int64_t* out_strides, const void* positions, int32_t pos_bits, int64_t pos_stride,
                  const b200fa_rotary_desc* rotary, int32_t dtype, void* stream);

/* Writes a step's K and V [tokens][heads_kv][dim] into the cache at `slots`
 * (int64; a slot outside [0, num_pages * page_size) is a padded token and
 * skipped; slots of real tokens are distinct), with K rotated by its token's
 * position, and writes the rotated q [tokens][heads_q][dim] to q_out (q NULL:
 * none; q_out may be q).  rotary NULL: plain copies, positions ignored.
 * *_strides: token, head (q, k, v, q_out) or page, token, head (pages). */
int b200fa_append(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides,
                  const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                  void* k_pages, const int64_t* k_page_strides, void* v_pages, const int64_t* v_page_strides,
                  int64_t tokens, int32_t heads_q, int32_t heads_kv, int32_t dim, int64_t num_pages,
                  int32_t page_size, const int64_t* slots, const void* positions, int32_t pos_bits,
                  const b200fa_rotary_desc* rotary, int32_t dtype, void* stream);

/* Attention of new tokens over a paged cache.  Request r's new tokens are rows
 * cu_q[r] .. cu_q[r+1]-1 of q and o; row i of them stands at position
 * p = kv_lens[r] - (cu_q[r+1] - cu_q[r]) + i and attends the cached keys
 * j <= p, with window > 0 only j > p - window or j < sinks.  A row that sees
 * no key gets zeros; rows of o that belong to no request are not written.
 * Pages that no row of a work item sees are not read, nor are values behind a
 * request's last key used, so both may hold anything. */
typedef struct b200fa_paged_args {
    uint32_t    struct_size;    /* sizeof(b200fa_paged_args)                     */
    int32_t     dtype;          /* FP16 or BF16 (q, cache and o alike)           */
    const void* q;              /* [tokens][heads_q][128]                        */
    void*       o;
    const void* k_pages;
    const void* v_pages;
    int64_t     q_strides[2];   /* token, head                                   */
    int64_t     o_strides[2];
    int64_t     k_strides[3];   /* page, token, head                             */
    int64_t     v_strides[3];
    const int32_t* block_table; /* [requests][width]                             */
    int64_t     table_stride;
    const int32_t* kv_lens;     /* [requests]                                    */
    const int32_t* cu_q;        /* [requests + 1]                                */
    int64_t     tokens;
    int64_t     num_pages;
    int32_t     requests, width, page_size;
    int32_t     heads_q, heads_kv;
    int32_t     max_q;          /* the longest chunk (a hint: picks the kernel)  */
    float       scale;
    int32_t     window, sinks;  /* window 0: none                                */
    uint32_t    timeout_us;     /* bound of every device-side wait (to some
                                   milliseconds); 0 = 2 s                        */
    uint32_t    flags;          /* B200FA_PAGED_TEST_WITHHOLD_V or 0             */
    void*       workspace;      /* 256-byte aligned; with status NULL, its first
                                   256 bytes zeroed once                         */
    uint64_t    ws_bytes;
    uint32_t*   status;         /* 256 bytes, zeroed once, kept between calls and
                                   shared by any of them (b200fa_read_status,
                                   b200fa_reset_status); NULL: the first ones of
                                   the workspace.  A struct that ends before this
                                   field is accepted too.                        */
    const int32_t* tables_status; /* b200fa_build_tables' status, or NULL: other
                                   than 0, nothing was handed out for the new
                                   tokens and all their rows become zeros        */
} b200fa_paged_args;

/* Test-only: no V block is loaded, so that the waits for it run out and the
 * kernel reports B200FA_DEV_TIMEOUT (the failure-detection test). */
#define B200FA_PAGED_TEST_WITHHOLD_V 1u

/* Bytes of workspace on the current device (status header + partial results,
 * which live for one call).  Calls that share a workspace must not overlap on
 * the GPU: where streams or graphs may, each call takes one from an allocator
 * that knows its stream, and `status` points elsewhere.  Negative: error. */
int64_t b200fa_paged_workspace_size(void);
int b200fa_paged_fwd(const b200fa_paged_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* B200FA_H_ */
