/*
 * cpu_ops_b200 -- C ABI of the B200 (sm_100a) implementation of the quantized
 * GEMM path of napplesty/cpu_ops.
 *
 * This is the drop-in boundary: the entry points below are what a binding for
 * the reference's
 *     gemm::device::Gemm<uint8_t,LA,int8_t,LB,int32_t,LC,...>::operator()
 *         (include/cpu_ops/gemm/device/gemm.h:99-127, alias GemmU8S8S32 :130-142)
 *     gemm::device::GemmMx<SA,SB,LC,...>::operator()
 *         (include/cpu_ops/gemm/device/gemm_mx.h:78-118, aliases :121-127)
 * forwards to.  Plain C types only: pointers, sizes and PODs; no C++ or torch
 * types cross it.  The C++17 headers under include/cpu_ops/ mirror the
 * reference's templates and flatten their Arguments into the descriptor below.
 *
 * Pointers may be host or device memory (detected per pointer unless
 * `memory_space` says otherwise).  Host operands are staged to the GPU and the
 * result copied back inside the call, so a caller written against the CPU
 * library works unchanged; device operands are used in place.
 *
 * There is no CPU fallback: if no sm_100 device / driver is present the calls
 * return CPUOPS_B200_STATUS_NO_DEVICE.
 */
#ifndef CPU_OPS_B200_H_
#define CPU_OPS_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(_WIN32)
#define CPUOPS_B200_API
#else
#define CPUOPS_B200_API __attribute__((visibility("default")))
#endif

#define CPUOPS_B200_ABI_VERSION 1

/* Return codes.  0..2 are the reference's cpu_ops::Status values
 * (include/cpu_ops/status.h:5-9); the rest are new and only arise from the
 * GPU runtime. */
enum {
  CPUOPS_B200_STATUS_SUCCESS = 0,
  CPUOPS_B200_STATUS_INVALID_PROBLEM = 1,   /* Status::kErrorInvalidProblem   */
  CPUOPS_B200_STATUS_INVALID_ARGUMENTS = 2, /* Status::kErrorInvalidArguments */
  CPUOPS_B200_STATUS_UNSUPPORTED = 3,       /* valid in the reference, not built here */
  CPUOPS_B200_STATUS_NO_DEVICE = 4,         /* no usable sm_100 GPU / driver          */
  CPUOPS_B200_STATUS_CUDA_ERROR = 5,        /* a CUDA call failed (see last_error)     */
  CPUOPS_B200_STATUS_DEVICE_TIMEOUT = 6,    /* a bounded device-side wait gave up      */
  CPUOPS_B200_STATUS_BAD_DESCRIPTOR = 7     /* struct_size / enum value not understood */
};

/* Operand element formats. */
enum {
  CPUOPS_B200_FMT_U8 = 0,   /* uint8_t                      (int8 path, A)   */
  CPUOPS_B200_FMT_S8 = 1,   /* int8_t                       (int8 path, B)   */
  CPUOPS_B200_FMT_E4M3 = 2, /* fp8e4m3_t, mx_formats.h:107-153               */
  CPUOPS_B200_FMT_E5M2 = 3, /* fp8e5m2_t, mx_formats.h:157-199               */
  CPUOPS_B200_FMT_E2M1 = 4  /* fp4e2m1_t, two per byte, even k in low nibble */
};

enum { CPUOPS_B200_KIND_I8 = 0, CPUOPS_B200_KIND_MX = 1 };

/* epilogue::Activation, include/cpu_ops/epilogue/linear_combination.h:12-15 */
enum { CPUOPS_B200_ACT_NONE = 0, CPUOPS_B200_ACT_RELU = 1 };

/* Fused chain ops, include/cpu_ops/epilogue/fusion.h:31-129.  Applied in
 * array order after alpha*acc + beta*C, as epilogue::Chain does (:136-166). */
enum {
  CPUOPS_B200_OP_RELU = 1,          /* Relu        : x < 0 ? 0 : x            */
  CPUOPS_B200_OP_CLAMP = 2,         /* Clamp{lo,hi}: x<lo?lo:(hi<x?hi:x)      */
  CPUOPS_B200_OP_BIAS_ADD = 3,      /* BiasAdd{p}  : x + p[col]               */
  CPUOPS_B200_OP_SCALE_PER_ROW = 4, /* ScalePerRow : x * p[row]               */
  CPUOPS_B200_OP_SCALE_PER_COL = 5, /* ScalePerCol : x * p[col]               */
  CPUOPS_B200_OP_GELU = 6,          /* Gelu (tanh form); f32 accumulators only */
  CPUOPS_B200_OP_SILU = 7           /* Silu;              f32 accumulators only */
};
#define CPUOPS_B200_MAX_OPS 8

enum { CPUOPS_B200_MEM_AUTO = 0, CPUOPS_B200_MEM_HOST = 1, CPUOPS_B200_MEM_DEVICE = 2 };

/* flags */
#define CPUOPS_B200_FLAG_ASYNC 1u /* device operands only: enqueue on `stream` and return \
                                     without synchronising; device-side errors are then   \
                                     reported by cpuops_b200_stream_status()              */
/* Testing/tuning, like tile_n: force or forbid the two-CTA form of the kernel (a cluster
 * of two CTAs per 256-row tile).  Neither flag: the library decides by problem size. */
#define CPUOPS_B200_FLAG_PAIR_ON 2u
#define CPUOPS_B200_FLAG_PAIR_OFF 4u

typedef union cpuops_b200_scalar {
  int32_t i32; /* int8 path: alpha/beta/clamp bounds are s32 */
  float f32;   /* MX path:   f32                            */
} cpuops_b200_scalar;

typedef struct cpuops_b200_epilogue_op {
  int32_t opcode;         /* CPUOPS_B200_OP_*                                       */
  int32_t reserved;       /* 0                                                      */
  const void* ptr;        /* bias / scale vector of the accumulator type, or NULL   */
  cpuops_b200_scalar lo;  /* Clamp only                                             */
  cpuops_b200_scalar hi;
} cpuops_b200_epilogue_op;

/*
 * One GEMM:  D = chain(act(alpha * A*B + beta * C)).
 * Field meaning follows the reference's Arguments (gemm.h:84-94, gemm_mx.h:65-74):
 *   int8: A is m x k, B is k x n, each row- or column-major with leading
 *         dimension lda / ldb in elements (tensor_ref.h:6-27, layout/matrix.h:9-22).
 *   MX:   A is m rows of k, B is n rows of k (k contiguous for both, "TN"),
 *         lda/ldb count ELEMENTS along k (fp4: two per byte, ld must be even),
 *         a_scales[i*ld_scales_a + kk/32], b_scales[j*ld_scales_b + kk/32] are
 *         E8M0 bytes (mx_formats.h:280-295); a_row_major/b_row_major are ignored.
 *   C, D: m x n in the layout c_row_major selects, ldc/ldd in elements; C and D
 *         may be the same buffer; C's values are never read when beta == 0 but
 *         the pointer must be non-null (gemm.h:112-114).
 *   split_k_slices: 0 automatic, 1 never, >1 forced (clamped to the k depth).
 *         Results are bit-identical from run to run for a given slice count,
 *         and for the int8 path identical for every slice count.
 */
typedef struct cpuops_b200_gemm_desc {
  uint32_t struct_size; /* sizeof(cpuops_b200_gemm_desc), checked */
  int32_t kind;         /* CPUOPS_B200_KIND_*                     */
  int32_t a_format;     /* CPUOPS_B200_FMT_*                      */
  int32_t b_format;
  int32_t m, n, k;
  int32_t a_row_major, b_row_major, c_row_major;
  const void* a;
  const void* b;
  const void* a_scales; /* MX only */
  const void* b_scales; /* MX only */
  int32_t lda, ldb;
  int32_t ld_scales_a, ld_scales_b;
  const void* c;
  void* d;
  int32_t ldc, ldd;
  cpuops_b200_scalar alpha, beta;
  int32_t activation; /* CPUOPS_B200_ACT_* */
  int32_t n_ops;      /* 0..CPUOPS_B200_MAX_OPS */
  cpuops_b200_epilogue_op ops[CPUOPS_B200_MAX_OPS];
  int32_t split_k_slices;
  int32_t memory_space; /* CPUOPS_B200_MEM_* for all pointers (AUTO: ask the driver) */
  void* stream;         /* cudaStream_t; NULL = the library's own stream, which is not
                           ordered after the caller's streams: device operands must be
                           complete before the call (a synchronous call returns with D
                           complete)                                                 */
  uint32_t flags;       /* CPUOPS_B200_FLAG_*                                        */
  int32_t device;       /* CUDA device ordinal, or -1 for the current device         */
  int32_t tile_n;       /* 0 = automatic; else force the N tile (testing/tuning)     */
} cpuops_b200_gemm_desc;

/* Replaces Gemm::operator() / GemmMx::operator() (gemm.h:99-127,
 * gemm_mx.h:78-118): validates in the reference's order, runs the GEMM on the
 * GPU, returns a CPUOPS_B200_STATUS_* code.  Synchronous unless FLAG_ASYNC.
 * Thread-safe: calls on the same device are serialised (as the reference serialises
 * on its thread pool, thread_pool.h:93-96), calls on different devices run side by
 * side.  The calling thread's current CUDA device is left as it was.
 * Asynchronous calls are plain kernel launches and may be captured into a CUDA graph,
 * provided the same call ran once on that stream before the capture began (the call
 * then finds its workspace in place; one that would have to allocate during capture
 * returns CPUOPS_B200_STATUS_INVALID_ARGUMENTS instead).  A workspace used under capture
 * is never freed, so graphs stay valid when later calls on the stream need more room.
 * Workspaces belong to streams, not to handles: cudaStreamPerThread is a stream of its own in
 * every thread, and a stream with a destroyed one's handle does not share that one's (that one's
 * graphs stay valid).
 * Large operands in pageable host memory are copied through 16 MB of pinned memory per
 * device and by up to three threads besides the caller's, both kept until the process
 * ends; the threads take no signals, and from then on the library cannot be unloaded. */
CPUOPS_B200_API int cpuops_b200_gemm(const cpuops_b200_gemm_desc* desc);

/* No counterpart in the reference.  u8 x s8 -> s32 GEMM through the two-stage
 * split-k path for callers that must not allocate device memory: a server that
 * gave all device memory to its own pool at start-up, or a latency-critical loop
 * where a cudaMalloc/cudaFree inside the library would stall the whole device.
 * cpuops_b200_gemm() grows a cached workspace with cudaMalloc when a problem first
 * needs one; this entry point never calls cudaMalloc, cudaFree or any allocating
 * routine.  Its split-k partial sums live in a fixed array inside the library image
 * of CPUOPS_B200_NOALLOC_SCRATCH_BYTES (every GPU that loads the library holds it
 * until the process exits).
 *   - Same descriptor and epilogue as cpuops_b200_gemm, kind I8 only, k > 0.
 *   - All pointers must be device memory; A and B must be 16-byte aligned with
 *     leading dimensions that are multiples of 16 (nothing can be staged or repacked).
 *   - split_k_slices: 0 picks as many slices as fit the array, at most
 *     min(8, ceil(k/128)); a forced count whose slices * m * n * 4 bytes of partial sums
 *     do not fit (or m * n * 4 alone) is rejected with
 *     CPUOPS_B200_STATUS_INVALID_ARGUMENTS and a message naming the size and the limit.
 *   - stream == NULL means the legacy default stream (no stream is created).
 *     Synchronous.  FLAG_ASYNC is ignored.
 *   - The first call on a device looks up the array's device address and sets kernel
 *     attributes; make that first call before any stream capture begins.
 *   - All calls share the one array: it keeps the previous call's contents (the
 *     library clears the one word that must start at zero), and two calls whose
 *     kernels overlapped on the GPU would race on it.  The call is synchronous and
 *     serialised per device inside the library, so this only matters to a caller that
 *     loads two copies of the library into one process.
 * Results are bit-identical to cpuops_b200_gemm on the same descriptor. */
#define CPUOPS_B200_NOALLOC_SCRATCH_BYTES (8u << 20)
CPUOPS_B200_API int cpuops_b200_gemm_i8_noalloc(const cpuops_b200_gemm_desc* desc);

/* Rewrites a row-major E8M0 scale array (rows x ceil(k/32) entries, leading
 * dimension ld_scales; the addressing of mx_formats.h:280-295, read by
 * mma_policy_mx.h:213,219,242,248) into the tile-ordered layout the tensor
 * cores consume: for every tile of `tile_rows` rows and every group of
 * `blocks_per_stage` (4 or 8) scale blocks, 512-byte atoms of
 * [32 lanes][4 row groups][4 blocks].  Entries outside the matrix are written
 * as 127 (scale 1.0) so that padding never multiplies by NaN.  `out` must hold
 * cpuops_b200_scale_layout_bytes() bytes of device memory.  Device pointers. */
CPUOPS_B200_API int cpuops_b200_relayout_scales(const void* scales, int32_t rows, int32_t k,
                                                int32_t ld_scales, int32_t tile_rows,
                                                int32_t blocks_per_stage, void* out,
                                                void* stream);
CPUOPS_B200_API size_t cpuops_b200_scale_layout_bytes(int32_t rows, int32_t k, int32_t tile_rows,
                                                      int32_t blocks_per_stage);

/* Row-block sharding of the output across `world` GPUs (one process per GPU):
 * rank `rank` owns rows [*row_begin, *row_begin + *row_count) of A, C and D and
 * needs all of B.  Blocks are balanced to whole 128-row tiles so every rank's
 * arithmetic is identical to the single-GPU run.  Plays the role of the
 * reference's partition_gemm (gemm/threadblock/threadblock_swizzle.h:47-91)
 * across devices. */
CPUOPS_B200_API int cpuops_b200_shard_rows(int32_t m, int32_t world, int32_t rank,
                                           int32_t* row_begin, int32_t* row_count);

/* Status of work enqueued with FLAG_ASYNC on `stream` (synchronises it). */
CPUOPS_B200_API int cpuops_b200_stream_status(void* stream);

/* SMs the GEMM kernels of later calls on `device` (-1: the current one) may occupy; 0 or
 * less = all of them (the default).  No counterpart in the reference.  The kernels are
 * persistent, one CTA per SM, and hold their SMs until they end: a caller that wants a
 * communication kernel to run beside a GEMM (the all-gather of D on a second stream) leaves
 * it some SMs with this setting.  Results do not depend on it for int8; for MX it can change
 * the automatic split-k choice like any change of problem size does, for low-rank adapters of
 * many rows and 16-bit products the parts in which k is summed, and for sums over rows (dbias, dgamma, dbeta, the
 * balance loss) the parts of rows. */
CPUOPS_B200_API int cpuops_b200_set_sm_limit(int32_t device, int32_t sms);

/* Budget of every bounded device-side wait (mbarrier waits of the GEMM kernels' roles), in
 * microseconds; 0 restores the default of one second.  A wait that runs out makes the
 * kernel record a code, unwind and return; the call (or cpuops_b200_stream_status for
 * asynchronous calls) then reports CPUOPS_B200_STATUS_DEVICE_TIMEOUT.  Applies to calls
 * issued after it returns. */
CPUOPS_B200_API int cpuops_b200_set_wait_budget_us(uint32_t microseconds);

/* Self-test of that path (no counterpart in the reference): launches one warp that waits,
 * with a budget of `budget_us` (1..100000) microseconds, on a barrier nothing arrives on.
 * Returns CPUOPS_B200_STATUS_DEVICE_TIMEOUT when the mechanism works -- the wait gave up,
 * the device error word was set, read and cleared -- and the device stays usable.
 * Synchronous; `stream` NULL = the library's own stream. */
CPUOPS_B200_API int cpuops_b200_selftest_wait_timeout(uint32_t budget_us, void* stream);

/* Measurement aid with no counterpart in the reference: while enabled, CUDA
 * events are recorded on the launching stream around every tensor-core GEMM
 * kernel (not the helper kernels).  collect() waits for them, returns the
 * summed device time and the number of timed launches, and forgets them. */
CPUOPS_B200_API int cpuops_b200_profile(int enable);
CPUOPS_B200_API int cpuops_b200_profile_collect(double* total_ms, int32_t* launches);

/* Prepared B (no counterpart in the reference, whose calls are stateless): a decode loop
 * multiplies ever-new activations by the same MX weights.  prepare_b registers the B
 * scale array described by `d` (b_scales, n, k, ld_scales_b; device memory) as unchanged
 * until release_b: later cpuops_b200_gemm calls that pass the same b_scales / n / k /
 * ld_scales_b keep the tile-ordered copy of those scales that the tensor cores need
 * (built on the first such call, one per tile layout) instead of rebuilding it per call.
 * A call with few tiles reads unregistered scales inside the GEMM kernel, with no launch in
 * front; registered, it reads the kept copy of B's and re-lays A's out, which can take longer.
 * The caller must not modify the scale array while it is registered.  release_b
 * synchronises the device and frees the copies. */
CPUOPS_B200_API int cpuops_b200_prepare_b(const cpuops_b200_gemm_desc* d, void** handle);
CPUOPS_B200_API int cpuops_b200_release_b(void* handle);

/* ---- projections whose weights are chosen per row -------------------------------------------
 * No counterpart in the reference: the products of a layer of experts, the routing that picks
 * them, and low-rank adapters beside a shared projection.  Unlike cpuops_b200_gemm these take
 * device memory only (a pointer to host memory, or to another device's, is refused with
 * CPUOPS_B200_STATUS_INVALID_ARGUMENTS), since what they compute depends on index arrays that the
 * host never reads.  `stream`, `flags` (CPUOPS_B200_FLAG_ASYNC), `device` and `memory_space` mean
 * what they mean in cpuops_b200_gemm_desc (MEM_DEVICE skips the check of the pointers), locking
 * and stream capture are the same too.  Calls whose comment says so use the stream's workspace:
 * graphs captured from one stream share it with each other and with that stream's own calls, so replay
 * such graphs one after another, not side by side, nor beside those calls.  Results are
 * bit-identical from run to run, for one setting of cpuops_b200_set_sm_limit (the adapters' products of
 * many rows are summed in parts of k that depend on it).  Outputs must not overlap inputs or one
 * another, except where a comment allows it. */

/* Element types of rows that are not quantised. */
enum { CPUOPS_B200_TYPE_F32 = 0, CPUOPS_B200_TYPE_F16 = 1, CPUOPS_B200_TYPE_BF16 = 2 };

/* How logits become scores. */
enum { CPUOPS_B200_SCORE_SOFTMAX = 0, CPUOPS_B200_SCORE_SIGMOID = 1 };

#define CPUOPS_B200_MAX_GROUPS 1024 /* experts of a route call, groups of a plan */
#define CPUOPS_B200_MAX_TOP_K 32

/* A row plan sorts "pairs" (a row and one of the groups it goes to, numbered row by row: pair
 * q = row * pairs_per_row + slot) by group: offsets[g] .. offsets[g + 1] are the places in
 * `order` of the pairs of group g, in ascending order.  Pairs whose id lies outside [0, groups)
 * belong to no group; as many entries at the end of `order` are -1. */

/* Routing: for every token
 *     score[e]  = softmax(logits)[e]  or  1 / (1 + exp(-logits[e]))
 *     choice[e] = score[e] + bias[e]
 * With n_groups > 1 the experts are cut into n_groups runs of equal length; a run counts as the
 * sum of its `group_best` (1 or 2) best choices, and only the top_groups best runs stay (of
 * equal ones the first).  ids are the top_k experts of those by choice, the best first (of equal
 * ones the first); weights their scores (without bias), divided by their sum if `renormalize`
 * (a sum of zero gives zeros), times `scale`.
 * An expert whose logit or bias is NaN or -inf is out, also of the softmax's sum; where fewer than top_k
 * are left, the remaining ids are -1 and their weights 0.  A logit of +inf counts as the largest
 * number there is (several share the softmax).
 * Choices are made in double precision: which experts a token gets does not hang on rounding.
 * offsets (experts + 1) and order (tokens * top_k): the plan of ids; both NULL: none is made.
 * Uses the stream's workspace when a plan of more than 4096 pairs is made. */
typedef struct cpuops_b200_route_desc {
  uint32_t struct_size; /* sizeof(cpuops_b200_route_desc), checked */
  int32_t tokens, experts, top_k;
  int32_t scoring;      /* CPUOPS_B200_SCORE_*                     */
  int32_t n_groups, top_groups, group_best;
  int32_t renormalize;
  float scale;
  int32_t logits_type;  /* CPUOPS_B200_TYPE_*                      */
  int32_t ld_logits;    /* elements from one token to the next     */
  const void* logits;
  const float* bias;    /* one per expert, or NULL                 */
  int32_t* ids;         /* tokens x top_k, contiguous              */
  float* weights;       /* the same                                */
  int32_t* offsets;
  int32_t* order;
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_route_desc;
CPUOPS_B200_API int cpuops_b200_route(const cpuops_b200_route_desc* desc);

/* The plan of `rows` ids (the second half of cpuops_b200_route, for ids from elsewhere). */
typedef struct cpuops_b200_group_rows_desc {
  uint32_t struct_size;
  int32_t rows, groups;
  const int32_t* ids;   /* rows       */
  int32_t* offsets;     /* groups + 1 */
  int32_t* order;       /* rows       */
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_group_rows_desc;
CPUOPS_B200_API int cpuops_b200_group_rows(const cpuops_b200_group_rows_desc* desc);

/* The experts' products, on MX operands (the formats, scales and leading dimensions of
 * cpuops_b200_gemm_desc).  For every pair q of group g in the plan
 *     acc[j] = sum_k A[q / pairs_per_a_row][k] * B_g[j][k]
 *              (one running f32 sum of the tensor cores, whose roundings grow with k: of random 8-bit
 *              operands 2.5e-6 of the result's norm at k = 4096, 1e-5 at 16384)
 *     y[j]   = acc[j],  or  silu(acc[j]) * acc[n + j]  with `gated`
 *     y[j]  *= row_weights[q]                                              (if given)
 *     D[q]   = y       if pairs_per_d_row == 1; rows of pairs in no group are zeros if `ids` are given
 *              (a layer with one expert per row), and left as they were if they are NULL
 *     D[t]   = the sum of y over t's pairs_per_d_row pairs, ascending, otherwise (pairs in no group
 *              add nothing; a row without any is zero); `ids` are needed then
 * `ids` are the ids the plan was made from.
 * Uses the stream's workspace when it sums (rows * n floats) and when there are 48 pairs per group
 * or more (their rows of A in the plan's order).
 * B_g is n (gated: 2n, the gate's rows first) rows of k, the first of them row g * b_group_rows
 * of B.  A and B: 16-byte aligned, rows a multiple of 16 bytes apart, an even k for e2m1.  A
 * and B may both be 8-bit formats, both e2m1, or e2m1 weights under 8-bit rows (then B 32-byte
 * aligned, its rows a multiple of 32 bytes apart, k a multiple of 128).  The scale arrays may lie
 * anywhere; 16-byte aligned rows of them are read fastest. */
typedef struct cpuops_b200_gemm_grouped_desc {
  uint32_t struct_size;
  int32_t a_format, b_format; /* CPUOPS_B200_FMT_E4M3, _E5M2, _E2M1           */
  int32_t rows;               /* pairs of the plan (length of order)         */
  int32_t n, k, groups;
  int32_t gated;
  int32_t a_rows;             /* rows of A                                   */
  int32_t pairs_per_a_row, pairs_per_d_row;
  int32_t b_group_rows;       /* rows of B from one group to the next        */
  int32_t lda, ldb, ld_scales_a, ld_scales_b;
  int32_t ldd;
  const void* a;
  const void* b;
  const void* a_scales;
  const void* b_scales;
  const int32_t* offsets;     /* groups + 1                                  */
  const int32_t* order;       /* rows                                        */
  const int32_t* ids;         /* rows, or NULL (pairs_per_d_row == 1 only)   */
  const float* row_weights;   /* rows, or NULL                               */
  float* d;                   /* rows / pairs_per_d_row rows of n, row-major */
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_gemm_grouped_desc;
CPUOPS_B200_API int cpuops_b200_gemm_grouped(const cpuops_b200_gemm_grouped_desc* desc);

/* Low-rank adapters of many requests beside a shared projection (whose result is C):
 *     D[t] = C[t] + scales[g] * (X[t] A_g^T) B_g^T     with g = ids[t]
 * and D[t] = C[t] where ids[t] lies outside [0, adapters).  A_g is `rank` rows of k (rows lda,
 * adapters a_stride elements apart), B_g n rows of `rank` (ldb, b_stride).  An adapter of a smaller
 * rank is padded with zeros.  X may be f32 with A and B f16 or bf16, or all three the same
 * 16-bit type; C, D and every sum are f32 (of f16 adapters, where rows are taken in tiles, the elements of
 * X A_g^T are kept to 22 bits, small ones to 2^-39 of the row's largest).  D may be C.  16-byte aligned rows of X, A and B are read
 * fastest.  n and k are at most 2^30.  Uses the stream's workspace where rows are taken in tiles sorted by
 * adapter, which an estimate of both times decides (a few hundred rows and more). */
typedef struct cpuops_b200_adapters_desc {
  uint32_t struct_size;
  int32_t m, n, k, rank, adapters;
  int32_t x_type, w_type;   /* CPUOPS_B200_TYPE_*                   */
  int32_t ldx, lda, ldb, ldc, ldd;
  int64_t a_stride, b_stride;
  const void* x;
  const void* a;
  const void* b;
  const int32_t* ids;       /* m                                    */
  const float* scales;      /* one per adapter, or NULL (all 1)     */
  const float* c;
  float* d;
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_adapters_desc;
#define CPUOPS_B200_MAX_RANK 256
CPUOPS_B200_API int cpuops_b200_adapters(const cpuops_b200_adapters_desc* desc);

/* ---- 16-bit layers and their gradients -------------------------------------------------------
 * What a program that trains the dense parts of a model, or its router, needs beside the quantised products:
 * the reference has 16-bit GEMMs and layer norm on the CPU, no gradients.  As the entry points above, these take
 * device memory only, and `stream`, `flags`, `device`, `memory_space`, locking, stream capture and the
 * stream's workspace mean the same (comments say which calls use the workspace).  Matrices are rows of
 * contiguous elements, ld elements apart; types are CPUOPS_B200_TYPE_*.  Sums are f32 throughout and
 * every stored 16-bit value is rounded once.  Exponentials are exp2 instructions on f32: GELU and SiLU here are within 3e-7 of
 * |z| (in the quantised products' chain they are near their last bit; of z = -inf both give NaN here and there), their slopes
 * within 8e-7 of |dY|, and the balance loss's scores, before they are normalised, within 3e-7 + 8e-8 times the logit's distance
 * from its token's largest (sigmoid: |logit|) of themselves.  Results are bit-identical from run to run, for one setting of
 * cpuops_b200_set_sm_limit (on which the parts that are summed depend).  Outputs must not overlap inputs or
 * one another, except where a comment allows it. */

/* z = alpha * A B + bias,  D = act(z) + beta * C,  Z = z (where Z is given: what cpuops_b200_epilogue_grad wants).
 * A is m x k, B k x n, both f16 or both bf16, each row-major or column-major, so that the products of a backward
 * pass are calls of this entry too: with Y = X W^T (W by rows: B column-major), dX = dY W has B row-major and
 * dW = dY^T X has A column-major and B row-major.  C, D and Z are row-major; C and D f32 or of A's type, Z of D's.
 * activation: 0 or CPUOPS_B200_OP_RELU, _GELU (tanh form), _SILU.  C is not read and may be NULL when beta == 0;
 * D may be C (same ld and type).  k == 0: the product is zero.
 * Sums are the tensor cores' running f32 sums (of up to eight parts of k, added in order, where there are few tiles), which drop
 * low bits, towards zero: 1e-9 of the result's norm per element of k with operands of both signs, 6.5e-9 of the result
 * where all products have one sign.  Where D is f32 they are handed over to f32 additions every 512 elements of k: 7e-7 of the
 * norm up to k = 65536 and 1e-6 at 2^20, 3e-6 of the result with one sign.  Where D has 16 bits they are from k = 16384 (f16)
 * or 131072 (bf16) of a part on, every 8192 elements, so that what is dropped stays below half of the least half step of D's
 * and Z's rounding at any k.
 * 16-byte aligned rows are read and written fastest.  Uses the stream's workspace where rows of A or B are not
 * 16-byte aligned (a copy of them).  m, n and k are at most 2^30. */
typedef struct cpuops_b200_gemm16_desc {
  uint32_t struct_size; /* sizeof(cpuops_b200_gemm16_desc), checked */
  int32_t type;         /* of A and B: CPUOPS_B200_TYPE_F16, _BF16 */
  int32_t c_type, d_type;
  int32_t m, n, k;
  int32_t a_row_major, b_row_major;
  int32_t activation;
  int32_t lda, ldb, ldc, ldd, ldz;
  float alpha, beta;
  const void* a;
  const void* b;
  const float* bias;      /* n, or NULL                              */
  const void* c;
  void* d;
  void* z;                /* or NULL                                 */
  int32_t split_k_slices; /* 0 automatic; else 1, 2, 4 or 8          */
  int32_t tile_n;         /* 0 automatic; else force (testing/tuning, as the FLAG_PAIR_ flags) */
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_gemm16_desc;
CPUOPS_B200_API int cpuops_b200_gemm16(const cpuops_b200_gemm16_desc* desc);

/* The gradient of that epilogue: dZ = dY * act'(Z), dbias[j] = the sum over i of dZ[i][j] before its rounding.
 * dY, Z and dZ are m x n of one type: of an f32 residual stream's gradient the caller makes a 16-bit copy.  (dC of the residual is beta * dY itself; the products' gradients are
 * calls of cpuops_b200_gemm16 on dZ.)  Without an activation Z is not read, and dZ may be NULL.  relu'(z) is 0
 * for z <= 0; where z is infinite gelu' and silu' are their limits, 0 and 1.
 * dZ may be dY or Z.  dbias may be NULL.  Uses the stream's workspace for dbias. */
typedef struct cpuops_b200_epilogue_grad_desc {
  uint32_t struct_size;
  int32_t type;
  int32_t m, n;
  int32_t activation;
  int32_t lddy, ldz, lddz;
  const void* dy;
  const void* z;
  void* dz;
  float* dbias;         /* n, or NULL */
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_epilogue_grad_desc;
CPUOPS_B200_API int cpuops_b200_epilogue_grad(const cpuops_b200_epilogue_grad_desc* desc);

/* Layer norm, row by row (the reference's ops/norm.h layernorm):
 *     mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps),  Y = (x - mean) * rstd * gamma + beta
 * Y is of X's type, or of any type where X is f32.  gamma (NULL: 1) and beta (NULL: 0) hold n floats; mean and rstd
 * (NULL: not wanted) m floats, which cpuops_b200_layer_norm_grad reads.  Y may be X (same ld and type). */
typedef struct cpuops_b200_layer_norm_desc {
  uint32_t struct_size;
  int32_t x_type, y_type;
  int32_t m, n;
  int32_t ldx, ldy;
  float eps;            /* >= 0 */
  const void* x;
  const float* gamma;
  const float* beta;
  void* y;
  float* mean;
  float* rstd;
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_layer_norm_desc;
CPUOPS_B200_API int cpuops_b200_layer_norm(const cpuops_b200_layer_norm_desc* desc);

/* Its gradient, from the mean and rstd that the forward call left: with g = dY * gamma, xhat = (x - mean) * rstd
 *     dX = rstd * (g - sum g / n - xhat * sum(g * xhat) / n) + dR,   dgamma = sum dY * xhat,   dbeta = sum dY
 * (sums of dX's along the row, of dgamma's and dbeta's over the rows).  dR (NULL: 0), of X's type, is the gradient that
 * comes past the norm on the residual stream.  x_type is X's, dR's and dX's, y_type dY's.  dX may be X, dR or
 * (of the same type) dY.  dgamma and dbeta may be NULL.  Uses the stream's workspace for dgamma and dbeta. */
typedef struct cpuops_b200_layer_norm_grad_desc {
  uint32_t struct_size;
  int32_t x_type, y_type;
  int32_t m, n;
  int32_t lddy, ldx, lddr, lddx;
  const void* dy;
  const void* x;
  const void* dr;
  const float* gamma;
  const float* mean;
  const float* rstd;
  void* dx;
  float* dgamma;
  float* dbeta;
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_layer_norm_grad_desc;
CPUOPS_B200_API int cpuops_b200_layer_norm_grad(const cpuops_b200_layer_norm_grad_desc* desc);

/* The balance loss of a router, beside cpuops_b200_route and on its ids:
 *     counts[e] = pairs whose id is e,  f_e = counts[e] / sum counts
 *     p_te = softmax(logits[t])[e],  or with SCORE_SIGMOID s_te / sum_j s_tj of s = 1 / (1 + exp(-logits))
 *     P_e = the mean of p_te over the tokens that have an id in [0, experts)
 *     loss = coefficient * experts * sum_e f_e P_e        (coefficient where the load is even)
 * and dlogits = upstream * d loss / d logits, of the logits' type (counts have no gradient).  Tokens without an id
 * (padding, ids of -1) count nowhere and have a gradient of zero; without any such token the loss is 0.
 * An expert whose logit is NaN or -inf is out of its token's sum; +inf counts as the largest number.
 * dlogits are of the order of coefficient / (tokens * experts) and less: f16, whose numbers end at 6e-8, needs a loss scale in
 * upstream (or f32 logits).
 * upstream: the loss's own gradient, one float on the device (NULL: 1).  counts, loss and dlogits may each be NULL;
 * dlogits may be logits (same ld).  Uses the stream's workspace beyond 32 tokens. */
typedef struct cpuops_b200_balance_loss_desc {
  uint32_t struct_size;
  int32_t tokens, experts, top_k;
  int32_t scoring;       /* CPUOPS_B200_SCORE_*           */
  float coefficient;
  int32_t logits_type;
  int32_t ld_logits, ld_dlogits;
  const void* logits;
  const int32_t* ids;    /* tokens x top_k, contiguous    */
  const float* upstream;
  int32_t* counts;       /* experts                       */
  float* loss;           /* 1                             */
  void* dlogits;
  void* stream;
  uint32_t flags;
  int32_t device;
  int32_t memory_space;
} cpuops_b200_balance_loss_desc;
CPUOPS_B200_API int cpuops_b200_balance_loss(const cpuops_b200_balance_loss_desc* desc);

/* What the calling thread's last cpuops_b200_gemm call that reached a tensor-core kernel
 * launched, or cpuops_b200_gemm16 call (diagnostics for tests and benchmarks): */
typedef struct cpuops_b200_plan {
  int32_t swapped;   /* 1: the caller's B went on the MMA M side (small m)          */
  int32_t tile_n;    /* N tile                                                    */
  int32_t pair;      /* 1: two-CTA clusters, 256-row tiles                         */
  int32_t slices;    /* split-k slices                                            */
  int32_t stages;    /* shared-memory pipeline depth                              */
  int32_t grid;      /* CTAs launched                                             */
  int32_t c_ring;    /* 1: C prefetched by TMA into shared memory                  */
  int32_t prepared_b; /* 1: B's scale atoms came from cpuops_b200_prepare_b        */
  int32_t epilogue_warps; /* 4, or 8 (single-wave launches and short k loops)      */
  int32_t narrow_last;    /* 1: a ragged last tile column ran at its own width     */
  int32_t decode;         /* 1: the small-m MX kernel ran (one launch, raw scales);
                             `slices` is then the most pieces a weight tile was cut into */
} cpuops_b200_plan;
CPUOPS_B200_API int cpuops_b200_last_plan(cpuops_b200_plan* out);

/* Kernels launched by this library in this process so far (all threads). */
CPUOPS_B200_API uint64_t cpuops_b200_launch_count(void);

/* Human-readable description of the last failure on the calling thread. */
CPUOPS_B200_API const char* cpuops_b200_last_error(void);

CPUOPS_B200_API int cpuops_b200_abi_version(void);

/* Number of usable sm_100 devices (0 if none or no driver). */
CPUOPS_B200_API int cpuops_b200_device_count(void);

#ifdef __cplusplus
}
#endif
#endif /* CPU_OPS_B200_H_ */
