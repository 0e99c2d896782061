/* alpaka3_b200 -- C ABI of the B200 (sm_100a) data-parallel primitive library.
 *
 * Plain pointers and sizes only: every device pointer is a CUDA device (or managed) address on the device that is
 * current on the calling thread, every stream is a cudaStream_t passed as void*, and every entry point returns an
 * int status (A3B_OK == 0). On failure a3b_last_error() returns a message for the calling thread. All entry points
 * are asynchronous with respect to the host unless stated otherwise; results are visible after the stream is
 * synchronised.
 *
 * Each entry point names the alpaka3 interface whose backend dispatch it replaces (paths inside the alpaka3 project).
 */
#ifndef ALPAKA3_B200_H
#define ALPAKA3_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define A3B_VERSION 100

#if defined(__GNUC__)
#define A3B_API __attribute__((visibility("default")))
#else
#define A3B_API
#endif

typedef void* a3b_stream_t; /* cudaStream_t */

enum a3b_status
{
    A3B_OK = 0,
    A3B_ERR_INVALID = 1,     /* bad argument (null pointer, unsupported dtype/op combination, bad size) */
    A3B_ERR_CUDA = 2,        /* a CUDA runtime call failed; message has the CUDA error string */
    A3B_ERR_UNSUPPORTED = 3, /* no device / wrong architecture */
    A3B_ERR_TIMEOUT = 4,     /* a bounded device-side wait gave up (reported by a3b_get_device_error) */
    A3B_ERR_NOMEM = 5,
    A3B_ERR_TOO_LARGE = 6
};

enum a3b_dtype
{
    A3B_I32 = 0,
    A3B_U32 = 1,
    A3B_I64 = 2,
    A3B_U64 = 3,
    A3B_F32 = 4,
    A3B_F64 = 5,
    A3B_F16 = 6, /* IEEE half and bfloat16: only for the entry points over logits, rows and gradients that name them */
    A3B_BF16 = 7,
    A3B_E4M3 = 8, /* 8-bit floating point (largest values 448 and 57344): only outputs of a3b_rms_norm */
    A3B_E5M2 = 9
};

/* binary reduce functors: std::plus, ScalarFunc{min}, ScalarFunc{max} (test/unit/algorithm/reduce.cpp:22-56) */
enum a3b_reduce_op
{
    A3B_REDUCE_PLUS = 0,
    A3B_REDUCE_MIN = 1,
    A3B_REDUCE_MAX = 2
};

/* transform functors recognised on the C path: identity (onHost::reduce), x*x, a*b (BabelStream DotMultiplication) */
enum a3b_transform_op
{
    A3B_XFORM_IDENTITY = 0,
    A3B_XFORM_SQUARE = 1,
    A3B_XFORM_PRODUCT = 2
};

/* BabelStream element-wise kernels (benchmark/babelstream/src/babelStreamMainTest.cpp:78-133) */
enum a3b_stream_kind
{
    A3B_STREAM_INIT = 0,   /* a = init[0], b = init[1], c = init[2] */
    A3B_STREAM_COPY = 1,   /* c = a */
    A3B_STREAM_MUL = 2,    /* b = scalar * c */
    A3B_STREAM_ADD = 3,    /* c = a + b */
    A3B_STREAM_TRIAD = 4,  /* a = b + scalar * c */
    A3B_STREAM_NSTREAM = 5 /* a = a + b + scalar * c */
};

/* element-wise transforms for onHost::transform / onHost::concurrent with recognised functors */
enum a3b_map_kind
{
    A3B_MAP_COPY = 0,  /* out = in0 */
    A3B_MAP_SCALE = 1, /* out = alpha * in0 */
    A3B_MAP_ADD = 2,   /* out = in0 + in1 */
    A3B_MAP_MUL = 3,   /* out = in0 * in1 */
    A3B_MAP_AXPY = 4,  /* out = in0 + alpha * in1 (each operation rounded on its own) */
    A3B_MAP_SQUARE = 5 /* out = in0 * in0 */
};

typedef struct a3b_device_info
{
    int ordinal;
    int sm_count;
    int cc_major;
    int cc_minor;
    uint64_t global_mem_bytes;
    uint64_t l2_bytes;
    int max_threads_per_block;
    int warp_size;
    char name[128];
} a3b_device_info;

/* ------------------------------------------------------------------------------------------------- runtime */

A3B_API int a3b_version(void);
A3B_API const char* a3b_last_error(void);
/* onHost::DeviceSelector::getDeviceCount / getDeviceProperties (include/alpaka/onHost/DeviceProperties.hpp:28-56) */
A3B_API int a3b_device_count(int* count);
A3B_API int a3b_device_info_get(int ordinal, a3b_device_info* info);
/* onHost::alloc / allocDeferred: stream-ordered device allocation (include/alpaka/onHost/Queue.hpp:410) */
A3B_API int a3b_malloc_async(void** ptr, size_t bytes, a3b_stream_t stream);
A3B_API int a3b_free_async(void* ptr, a3b_stream_t stream);
/* onHost::memcpy (include/alpaka/onHost/Queue.hpp:237): any direction, one cudaMemcpyAsync */
A3B_API int a3b_memcpy_async(void* dst, void const* src, size_t bytes, a3b_stream_t stream);
/* onHost::wait(queue) (include/alpaka/onHost/interface.hpp:142) */
A3B_API int a3b_stream_synchronize(a3b_stream_t stream);
/* Device scratch for the kernels that the header-only engines (include/alpaka3_b200/simd_engine.cuh) instantiate in
 * the caller's translation unit: at least `bytes`, cached per (device, stream), zero-filled when first allocated or
 * grown. Work ordered on `stream` may use it; the engines leave it as they found it (their tickets are reset by the
 * kernel that drew the last number). No counterpart in alpaka3, whose reductions pre-fill the output instead. */
A3B_API int a3b_engine_scratch(a3b_stream_t stream, size_t bytes, void** ptr);
/* Reads (and with clear != 0 resets) the device-side error word of the current device: bit 0 = a bounded wait timed
 * out (A3B_ERR_TIMEOUT). Synchronises `stream`. */
A3B_API int a3b_get_device_error(a3b_stream_t stream, uint32_t* error_bits, int clear);
/* Limit in nanoseconds for every device-side spin-wait issued afterwards by this process (default 1 s). */
A3B_API int a3b_set_wait_timeout_ns(uint64_t ns);

/* ------------------------------------------------------------------------------- element-wise (transform) */

/* BabelStream kernels: queue.enqueue(FrameSpec, KernelBundle{SimdForEachKernel{}, Simd<Op>{}, a, b, c})
 * (benchmark/babelstream/src/babelStreamMainTest.cpp:285-364). dtype A3B_F32 or A3B_F64. init may be null unless
 * kind == A3B_STREAM_INIT. Every floating-point operation is rounded on its own (no contraction). */
A3B_API int a3b_babelstream(a3b_stream_t stream, int kind, int dtype, void* a, void* b, void* c, uint64_t n, double scalar,
                    double const* init);

/* onHost::transform(queue, out, fn, in0[, in1]) with a recognised fn (include/alpaka/onHost/algo/transform.hpp:50-88).
 * in1 is ignored for unary kinds. Integer dtypes wrap; alpha is converted to dtype first. */
A3B_API int a3b_transform(a3b_stream_t stream, int kind, int dtype, void* out, void const* in0, void const* in1, uint64_t n,
                  double alpha);

/* onHost::fill (include/alpaka/onHost/Queue.hpp:346): value points to one host element of dtype */
A3B_API int a3b_fill(a3b_stream_t stream, int dtype, void* out, uint64_t n, void const* value);

/* onHost::iota (include/alpaka/onHost/algo/iota.hpp:29-85): out[i] = start + i (host start value of dtype) */
A3B_API int a3b_iota(a3b_stream_t stream, int dtype, void* out, uint64_t n, void const* start);

/* nBody drift, onHost::concurrent(..., UpdatePositions{dt}, x, y, z, vx, vy, vz) (example/nBody/src/Kernels.hpp:126-142):
 * x = x + vx*dt per component, fp32 */
A3B_API int a3b_nbody_update_positions(a3b_stream_t stream, float* x, float* y, float* z, float const* vx, float const* vy,
                               float const* vz, uint64_t n, float dt);

/* Seeded Philox4x32-10 streams (counter = start + element index, key = seed), identical to the CPU oracle:
 *   u32: word0 >> shift;   u64: (word1 << 32) | word0;   f32: lo + (hi - lo) * ((word0 >> 8) * 2^-24). */
A3B_API int a3b_random_u32(a3b_stream_t stream, uint32_t* out, uint64_t n, uint64_t seed, uint64_t start, int shift);
A3B_API int a3b_random_u64(a3b_stream_t stream, uint64_t* out, uint64_t n, uint64_t seed, uint64_t start);
A3B_API int a3b_random_f32(a3b_stream_t stream, float* out, uint64_t n, uint64_t seed, uint64_t start, float lo, float hi);

/* ---------------------------------------------------------------------------------------------- reductions */

/* onHost::transformReduce(queue, neutral, out, reduceFn, transformFn, in0[, in1])
 * (include/alpaka/onHost/algo/transformReduce.hpp:59-90; kernel internal/transformReduce.hpp:23-202).
 * out: device pointer to ONE element of dtype, written with the final value (no pre-fill launch needed).
 * neutral: host pointer to one element of dtype. One launch; the final combination runs in the last block in a fixed
 * order, so a given (device, n) always gives the same bits. fp32 inputs are accumulated in fp64 inside the kernel;
 * integer + wraps (two's complement).
 * Ordering: by default the launch is fully ordered after all earlier work of the stream. With a3b_set_early_start
 * enabled on the stream it may start while the previous kernel of the stream still runs (see there). */
A3B_API int a3b_transform_reduce(a3b_stream_t stream, int dtype, int reduce_op, int transform_op, void const* in0,
                         void const* in1, uint64_t n, void const* neutral, void* out);

/* Same, but the per-block partials are left as fp64 (float dtypes) / 64-bit integers in partial_out[0] instead of
 * being rounded to dtype: used to combine shards across GPUs before the final rounding. Ordering as
 * a3b_transform_reduce. */
A3B_API int a3b_transform_reduce_partial(a3b_stream_t stream, int dtype, int reduce_op, int transform_op, void const* in0,
                                 void const* in1, uint64_t n, void const* neutral, void* partial_out);

/* No counterpart in the reference: a3b_transform_reduce for callers that cannot allocate device memory -- a process
 * whose device memory is owned by another allocator's pool, a service that must keep a fixed, accounted memory
 * footprint, a latency-critical loop that cannot afford an allocation's implicit synchronisation. Same arguments as
 * a3b_transform_reduce over a dense 1-D input; it allocates nothing. The result is the same for integer data; for
 * floating-point data it agrees within rounding (its grid is capped at 2024 blocks, so above that size the partials
 * are combined in another order) and is deterministic for a given n. Its scratch is one fixed 16 KB static device
 * array per GPU that loads the library (held until the process exits): the tickets and partials of at most 2024
 * blocks, each of which takes several chunks of a large input (A3B_ERR_TOO_LARGE is kept for a layout that would not
 * fit). The first call on a device (and the first after the device's context was re-created, e.g. by
 * cudaDeviceReset) looks up that array's device address, so make that call before any stream capture. All calls
 * share the array: calls that overlap on the GPU (different streams, devices' own streams in parallel) race and must
 * be serialised by the caller. Always launched fully ordered. */
A3B_API int a3b_transform_reduce_noalloc(a3b_stream_t stream, int dtype, int reduce_op, int transform_op,
                                         void const* in0, void const* in1, uint64_t n, void const* neutral, void* out);

/* Early start of the reductions on `stream` of the current device (a3b_transform_reduce, _partial, a3b_reduce_2d,
 * a3b_transform_reduce_allranks, a3b_reduce_lower_ranks); off by default. No counterpart in alpaka3, whose kernels
 * are plain launches. When enabled, a reduction is launched with programmatic dependent launch: it starts as soon as
 * the previous kernel of the stream lets its dependents launch, reads its input, and waits for that kernel to
 * complete only before it touches its scratch or `out`. The next call thus streams its input while this one combines
 * (and, across ranks, waits for its peers). The library launches fully ordered any call whose input overlaps the
 * output of one of its own reductions that may still run (every reduction started early since the last fully ordered
 * launch). ENABLE IT ONLY IF no other kernel on the stream executes griddepcontrol.launch_dependents
 * (cudaTriggerProgrammaticLaunchCompletion) before its output is written -- e.g. kernels built with programmatic
 * dependent launch by CUTLASS or some cuBLASLt kernels: the reduction could read that output before it is written.
 * Copies, memsets and kernels without that instruction are always complete before the reduction reads its input. */
A3B_API int a3b_set_early_start(a3b_stream_t stream, int enable);

/* onHost::reduce(queue, neutral, out, reduceFn, in) (include/alpaka/onHost/algo/reduce.hpp:28-79) over a pitched
 * 2-D view: `rows` rows of `row_len` elements, consecutive rows `row_pitch_bytes` apart (rows = 1 for 1-D data).
 * N-D alpaka buffers whose slower dimensions are dense multiples of the row pitch map onto this form. Ordering as
 * a3b_transform_reduce. */
A3B_API int a3b_reduce_2d(a3b_stream_t stream, int dtype, int reduce_op, void const* in, uint64_t rows, uint64_t row_len,
                  uint64_t row_pitch_bytes, void const* neutral, void* out);

/* --------------------------------------------------------------------------------------- multi-GPU (one node) */

/* A peer group connects the ranks of one node (one process per GPU) through a small slot buffer per rank that every
 * other rank maps over NVLink (CUDA IPC). Protocol: each rank calls a3b_peer_group_create on its device, exchanges
 * the a3b_ipc_handle_size() bytes written to `local_handle` with all ranks (any host channel), then calls
 * a3b_peer_group_connect with the world handles in rank order. No counterpart in alpaka3, which has no multi-device
 * layer. */
typedef struct a3b_peer_group a3b_peer_group;
A3B_API size_t a3b_ipc_handle_size(void);
A3B_API int a3b_peer_group_create(int world, int rank, a3b_peer_group** group, void* local_handle);
A3B_API int a3b_peer_group_connect(a3b_peer_group* group, void const* handles);
A3B_API int a3b_peer_group_destroy(a3b_peer_group* group);

/* onHost::transformReduce over data sharded across the ranks of a peer group, fused with the all-reduce: one launch
 * per rank reduces the local shard, its last block stores the unrounded partial into every rank's slot (peer stores
 * over NVLink), waits (bounded) for all ranks' partials and combines them in rank order, so every rank writes the
 * same bits to its `out`. All ranks must make the same sequence of calls. A wait that runs out sets bit 0 of the
 * device error word (a3b_get_device_error). Ordering as a3b_transform_reduce: with a3b_set_early_start enabled on the
 * stream, consecutive calls overlap, so a call reads its input while the previous call still waits for the other
 * ranks. */
A3B_API int a3b_transform_reduce_allranks(a3b_stream_t stream, a3b_peer_group* group, int dtype, int reduce_op,
                                          int transform_op, void const* in0, void const* in1, uint64_t n,
                                          void const* neutral, void* out);

/* Carry of a scan split across the ranks of a peer group: sums this rank's shard in one launch, exchanges the shard
 * totals through the peer slots and writes sum(totals of ranks 0 .. rank-1) to carry_out (device pointer, one
 * element of dtype; integers wrap). Feed it to a3b_scan as carry_in. */
A3B_API int a3b_reduce_lower_ranks(a3b_stream_t stream, a3b_peer_group* group, int dtype, void const* in, uint64_t n,
                                   void* carry_out);

/* ------------------------------------------------------------------------------------------------------ scan */

/* onHost::getScanBufferSize<T>(extents) (include/alpaka/onHost/algo/scan.hpp:26-30): bytes of the caller buffer that
 * a3b_scan accepts for n elements of dtype. */
A3B_API size_t a3b_scan_buffer_size(int dtype, uint64_t n);

/* onHost::inclusiveScan / exclusiveScan / *InPlace (include/alpaka/onHost/algo/scan.hpp:45-218), operator +,
 * exclusive identity 0. One cooperative launch of one block per SM that reads every element from HBM once and writes
 * it once (tile aggregates published two rounds ahead of the tiles' scans). in == out is allowed (in-place).
 * buffer: optional caller scratch of at least a3b_scan_buffer_size bytes (any contents; it is cleared on the
 *         stream); null uses a scratch cached by the library per (device, stream).
 * carry_in: optional DEVICE pointer to one element added to every output (the sum of all preceding shards when a
 *         scan is split across GPUs); null means 0. Integer arithmetic wraps (two's complement). */
A3B_API int a3b_scan(a3b_stream_t stream, int dtype, int inclusive, void const* in, void* out, uint64_t n,
             void const* carry_in, void* buffer, size_t buffer_bytes);

/* ---------------------------------------------------------------------------- token log probabilities (rows) */

/* Reductions over every row of logits (vocab values each): with z = scale * x,
 *   lse = ln sum_v e^(z_v),  logp = z_t - lse for the row's token t,  entropy = -sum_v p_v ln p_v, p_v = e^(z_v - lse),
 * and the `top` largest logits of the row, largest first, a tie to the lower index (-0 equals 0; NaN counts as larger
 * than +infinity): their log probabilities and their indices. One launch, every logit read once; the sums are held in
 * fp32. No counterpart in alpaka3, whose reductions give one value for a whole buffer.
 *
 * Rows: logits of dtype A3B_F32, A3B_F16 or A3B_BF16; row r = o * inner + i (o < outer, i < inner) starts at element
 * o * outer_stride + i * inner_stride and is contiguous; any strides, also ones that make rows overlap. The other
 * arrays are dense in row order: targets (index_dtype A3B_I32 or A3B_I64), logp, entropy, lse (fp32), top_logp (fp32)
 * and top_index (index_dtype), `top` of each per row. logp, entropy and lse may be null (not computed); targets may be
 * null if logp is. top: 0 .. 32, at most vocab. scale (the inverse temperature): between 2^-20 and 2^20.
 *
 * A target outside [0, vocab) marks a row without a token: its logp is 0. Logits of -infinity have probability 0 (logp
 * -infinity); a row of nothing else has lse -infinity, entropy 0 and logp -infinity for every token. A NaN in a row
 * makes its lse, logp and entropy NaN. With +infinity in a row its lse is +infinity, its entropy NaN, the logp of a
 * finite logit -infinity and that of +infinity NaN. Logits of any finite size are as good as their own steps allow
 * (masks of -1e9, -1e20 or the lowest value, alone or among others); where scale * logit is beyond fp32's range it is
 * infinite: in a row of nothing but such masks lse is -infinity, and the gradient 0.
 * Repeated calls give the same bits; the order of a row's sums follows from the number of rows, their length and
 * alignment. The outputs may not overlap one another or the inputs.
 * Time: one pass, but alternatives of a row in rising order enter and leave one after another (2048 rows of 50257 bf16
 * logits with 20 alternatives: 64 us in no particular order, 3.7 ms if every row rises from its first to its last).
 * At most 2^31 - 1 rows of at most 2^31 - 65 logits (A3B_ERR_TOO_LARGE). */
A3B_API int a3b_token_logprobs(a3b_stream_t stream, int dtype, void const* logits, uint64_t outer, uint64_t inner,
                               uint64_t vocab, int64_t outer_stride, int64_t inner_stride, double scale, int index_dtype,
                               void const* targets, float* logp, float* entropy, float* lse, uint32_t top,
                               float* top_logp, void* top_index);

/* Gradient of the outputs of a3b_token_logprobs with respect to the logits, one launch:
 *   grad_v = scale * (grad_logp * ([v == t] - p_v) + grad_lse * p_v - grad_entropy * p_v * (ln p_v + entropy)).
 * lse and entropy: as a3b_token_logprobs wrote them for the same logits, targets and scale. grad_logp, grad_entropy,
 * grad_lse: one fp32 value per row, each may be null (zero); targets may be null if grad_logp is, entropy if
 * grad_entropy is. A row without a token (target outside [0, vocab)) gets nothing from grad_logp; a row with lse
 * -infinity gets zeros; with lse +infinity the finite logits get what grad_logp gives their own token, else 0, and the
 * infinite ones NaN; with lse NaN all are NaN. Above |lse| = 2^24, where lse's own steps are 2 and more, scale * x is rounded to fp32 before lse
 * is taken off, as it was when lse was rounded: p stays at most 1. The alternatives have no gradient. grad_logits has the
 * logits' dtype, rounded once, and its own strides; its rows may not overlap. It may be the logits themselves (same
 * address and strides: in place) or must lie wholly before or behind them; it may not overlap the arrays of one value per
 * row. */
A3B_API int a3b_token_logprobs_backward(a3b_stream_t stream, int dtype, void const* logits, uint64_t outer, uint64_t inner,
                                        uint64_t vocab, int64_t outer_stride, int64_t inner_stride, double scale,
                                        int index_dtype, void const* targets, float const* lse, float const* entropy,
                                        float const* grad_logp, float const* grad_entropy, float const* grad_lse,
                                        void* grad_logits, int64_t grad_outer_stride, int64_t grad_inner_stride);

/* --------------------------------------------------------------------- norm and clipping of a list of gradients */

/* A list of dense device tensors on the device that is current when it is used: count pairs of an input and an output
 * address with the number of elements (0 is allowed) and dtype (A3B_F32, A3B_F64, A3B_F16 or A3B_BF16, mixed within a
 * list as needed). `out` may be null (every tensor in place), as may single entries of it. The list holds addresses
 * and sizes only: the caller keeps the memory alive while calls on it are pending, and makes a new list when an
 * address changes. It may be destroyed as soon as the calls that use it have returned, and used by several streams
 * and threads at once. No counterpart in alpaka3, whose algorithms take one buffer each. */
typedef struct a3b_tensor_list a3b_tensor_list;
A3B_API int a3b_tensor_list_create(void const* const* in, void* const* out, uint64_t const* n, int const* dtype,
                                   uint64_t count, a3b_tensor_list** list);
A3B_API int a3b_tensor_list_destroy(a3b_tensor_list* list);

/* norm over all elements x of a list: sqrt(sum x^2), sum |x|, max |x| (NaN if any element is) */
enum a3b_norm_kind
{
    A3B_NORM_L2 = 0,
    A3B_NORM_L1 = 1,
    A3B_NORM_MAX = 2
};

/* Bytes of device scratch that a3b_grad_norm and a3b_clip_grad_norm need for this list on the current device (any
 * contents; nothing is kept in it between calls). Calls that overlap on the GPU need one each. 0 on failure. */
A3B_API size_t a3b_grad_norm_workspace(a3b_tensor_list const* list);

/* Norm of the whole list, held in fp64 and rounded once to norm (one element of norm_dtype, A3B_F32 or A3B_F64).
 * partial: null, or one double that receives sum x^2, sum |x| or max |x| unrounded, to be combined across ranks (sum,
 * sum, max) before a3b_clip_grads. Either of norm and partial may be null. Squares that leave fp32's range are formed
 * in fp64. The order of the sum depends on the list and the device alone: repeated calls give the same bits. Here and
 * below norm, partial and the workspace lie apart from one another (A3B_ERR_INVALID) and from the tensors. */
A3B_API int a3b_grad_norm(a3b_stream_t stream, a3b_tensor_list const* list, int kind, void* workspace,
                          size_t workspace_bytes, double* partial, int norm_dtype, void* norm);

/* out = in * min(1, max_norm / (norm + 1e-6)) for every tensor of the list, with the norm that `partial` (one double on
 * the device, as a3b_grad_norm leaves it or combined over ranks) stands for; the product is formed in fp32 (fp64 for
 * A3B_F64, and for a factor below 2^-126) and rounded once. Tensors in place are not touched where the factor is 1. norm:
 * null, or one element that receives the norm. A NaN norm makes every output NaN. The outputs may not overlap one
 * another, and each must be its own input or overlap no input (A3B_ERR_INVALID). max_norm: not negative, not NaN. */
A3B_API int a3b_clip_grads(a3b_stream_t stream, a3b_tensor_list const* list, int kind, double const* partial,
                           double max_norm, int norm_dtype, void* norm);

/* a3b_grad_norm and a3b_clip_grads in one call. */
A3B_API int a3b_clip_grad_norm(a3b_stream_t stream, a3b_tensor_list const* list, int kind, double max_norm,
                               void* workspace, size_t workspace_bytes, int norm_dtype, void* norm);

/* Rows of an array: row o * inner + i (o < outer, i < inner, as the call says) starts at element o * outer_stride + i *
 * inner_stride of data and is contiguous. data null: the array is left out. */
typedef struct a3b_rows
{
    void* data;
    int64_t outer_stride;
    int64_t inner_stride;
} a3b_rows;

/* --------------------------------------------------------------------------------- root-mean-square norm (rows) */

/* Over every row of n elements: h = x + residual (rounded to dtype), r = 1 / sqrt(mean h^2 + eps), out = h * r * weight.
 * No counterpart in alpaka3: transformReduce with one result a row, and a transform with that result.
 *
 * Rows of dtype A3B_F32, A3B_F16 or A3B_BF16. residual: null or rows that are added; total: null or rows that
 * receive h (needs a residual). Rounded or not stored, it is the rounded h that is normed, so that a gradient which reads
 * `total` is that of what was computed. weight: n elements of dtype or A3B_F32, null: ones. rstd: null or one fp32 value a
 * row that receives r, for the gradient. The sum of squares is held in fp32, or in fp64 where that leaves fp32's range
 * (elements beyond 1e19, or below 1e-15 with an eps below 2^-60); every stored value is rounded once.
 *
 * out has dtype, or A3B_E4M3 or A3B_E5M2 with scales: groups of `group` elements of a row (32, 64 or 128, the last of a row
 * may be shorter; 0: the whole row) share the scale s = max |y| * (1 / L), L = 448 or 57344, y = h * r * weight in fp32, and
 * out = y * (1 / s) rounded to the nearest 8-bit value, at most L; both reciprocals and both products are the nearest fp32
 * values (an s below 2^-126 divides instead). scales: fp32, dense, ceil(n / group) (or 1) a row. A group of
 * zeros, or one whose s rounds to 0, has scale 0 and zeros.
 *
 * NaN in a row makes its out and rstd NaN; an infinity makes rstd 0, itself NaN and the others 0. A row of zeros with eps 0
 * has rstd infinity and NaN as output; one whose r is beyond fp32 (magnitudes below 2^-128 with eps 0) has rstd infinity and
 * infinities, NaN where it is 0. A group with a NaN has scale NaN and NaN throughout; one with an infinite y has scale infinity,
 * NaN there and 0 elsewhere.
 * An output may be an input of the same type in place (same address and strides: total = residual, out = x, ...); otherwise
 * outputs must lie apart from the inputs and from one another: wholly before or behind, or beside them in rows whose steps
 * are all multiples of one length that holds both (parts of one wider row). Rows of an output may not overlap. The order of
 * a row's sums follows from its length, alignment and the number of rows. At most 2^31 - 1 rows of 2^31 - 65 elements
 * (A3B_ERR_TOO_LARGE). One launch. */
typedef struct a3b_rms_norm_args
{
    uint64_t outer, inner, n;
    a3b_rows x, residual, total, out; /* x and residual are read */
    void const* weight;
    float* rstd;
    float* scales;
    double eps; /* 0 .. 2^100 */
    int32_t dtype, out_dtype, weight_dtype;
    uint32_t group;
} a3b_rms_norm_args;
A3B_API int a3b_rms_norm(a3b_stream_t stream, a3b_rms_norm_args const* args);

/* Bytes of device scratch that a3b_rms_norm_backward needs for grad_weight on the current device (any contents; nothing is
 * kept in it between calls). Calls that overlap on the GPU need one each. 0 on failure. */
A3B_API size_t a3b_rms_norm_backward_workspace(uint64_t rows, uint64_t n);

/* Gradient of a3b_rms_norm's out (as if not rounded to 8 bits): with d = grad_out * weight and k = x * rstd,
 *   grad_x = rstd * (d - k * mean(d * k)) + grad_total,   grad_weight = sum over rows of grad_out * k.
 * x: the rows that were normed (`total`, where there was a residual; grad_x is then the gradient of x and of residual
 * alike), rstd: as a3b_rms_norm wrote it; grad_total: null or the gradient that reaches `total` itself. grad_out, x,
 * grad_total and grad_x have dtype and each its strides. grad_weight: null or n elements of the weight's type (dtype or
 * A3B_F32 without a weight); it needs a workspace of a3b_rms_norm_backward_workspace bytes, 16-byte aligned. All sums are
 * held in fp32 (a row's positions and the rows in a fixed order: repeated calls give the same bits) and rounded once.
 * grad_x may be grad_out, x or grad_total in place. No rows: grad_weight is set to zero. */
typedef struct a3b_rms_norm_backward_args
{
    uint64_t outer, inner, n;
    a3b_rows grad_out, x, grad_total, grad_x; /* all but grad_x are read */
    void const* weight;
    float const* rstd;
    void* grad_weight;
    void* workspace;
    uint64_t workspace_bytes;
    int32_t dtype, weight_dtype, grad_weight_dtype;
    int32_t reserved; /* 0 */
} a3b_rms_norm_backward_args;
A3B_API int a3b_rms_norm_backward(a3b_stream_t stream, a3b_rms_norm_backward_args const* args);

/* ------------------------------------------------------------------------------- rows of a table, by tokens */

/* out_i = scale * row t_i of the table, for count = outer * inner tokens t (A3B_I32 or A3B_I64, dense): a transform whose
 * input is picked by an index. The table holds the rows of the tokens [first, first + vocab), n elements each, row_stride
 * apart; a token outside it gives a row of zeros (as a table cut over ranks wants, and as -100 for padding). Types: A3B_F32, A3B_F16 or A3B_BF16, both
 * alike, or one of them A3B_F32; the product is formed in fp32 and rounded once. scale: any finite fp32 value. The output's
 * rows may not overlap one another, the table or the tokens (beside them in rows of steps that are all multiples of one
 * length is apart). At most 2^31 - 65 tokens, rows of the table and elements a row (A3B_ERR_TOO_LARGE; rows of more than
 * 65535 * 512 accesses too, of one element, or of 4 or 8 where rows begin at 16 bytes and are whole packs). One launch. */
typedef struct a3b_embedding_args
{
    uint64_t outer, inner, n, vocab;
    int64_t first;
    void const* table;
    int64_t table_stride;
    void const* tokens;
    a3b_rows out;
    double scale;
    int32_t table_dtype, index_dtype, out_dtype;
    int32_t reserved; /* 0 */
} a3b_embedding_args;
A3B_API int a3b_embedding(a3b_stream_t stream, a3b_embedding_args const* args);

/* Bytes of device scratch that a3b_embedding_backward needs for `count` tokens on the current device (any contents; nothing
 * is kept in it between calls). Calls that overlap on the GPU need one each. 0 on failure. */
A3B_API size_t a3b_embedding_backward_workspace(uint64_t count, uint64_t n, uint64_t vocab);

/* Gradient of a3b_embedding with respect to the table: row v of grad_table = add_v + scale * the sum of grad_out_i over the
 * positions i whose token is first + v, zero (add_v) for tokens that do not occur. add: null, or rows of grad_table's type
 * that are added (the gradient from the table's other use as a head); add may be grad_table itself, of which then only the
 * rows of tokens that occur are touched. Types as in a3b_embedding: grad_out is of its out_dtype, the table of its
 * table_dtype. Sums are held in fp32 and rounded once; their order follows from count, n and vocab (and the device) alone:
 * repeated calls give the same bits. grad_out's rows may have any strides; grad_table's may not overlap. workspace: 16-byte
 * aligned, of a3b_embedding_backward_workspace bytes. grad_table and workspace lie apart from all inputs. A call of more
 * blocks than one launch holds (a table of some 2^44 elements and more) is refused before anything is launched
 * (A3B_ERR_TOO_LARGE). */
typedef struct a3b_embedding_backward_args
{
    uint64_t outer, inner, n, vocab;
    int64_t first;
    a3b_rows grad_out;
    void const* tokens;
    void const* add;
    int64_t add_stride;
    void* grad_table;
    int64_t table_stride;
    void* workspace;
    uint64_t workspace_bytes;
    double scale;
    int32_t grad_dtype, index_dtype, table_dtype;
    int32_t reserved; /* 0 */
} a3b_embedding_backward_args;
A3B_API int a3b_embedding_backward(a3b_stream_t stream, a3b_embedding_backward_args const* args);

/* ------------------------------------------------------------------------------- verification of drafted tokens */

/* For every sequence b of a batch, `length` drafted tokens t (A3B_I32 or A3B_I64; the first one outside [0, vocab) ends the
 * sequence's draft) against the target's logits (length + 1 rows a sequence: position i's row predicts draft i) and the
 * draft's own (length rows; null: the drafts were certain, q is 1 at t and 0 elsewhere):
 *   p_v = e^(scale * z_v - lse),  q_v = e^(draft_scale * z'_v - draft_lse), lse and draft_lse as a3b_token_logprobs writes
 * them. Draft i stands while uniform_i * q(t_i) < p(t_i). At the first that does not, one token is drawn from the rates
 * (p_v - q_v)+, behind the last one that stands from the rates p_v (also where no rate is left otherwise): the token with
 * the largest rate_v / noise_v, a tie to the lowest. With uniform in [0, 1) and noise independent exponential variates the
 * tokens are distributed as if drawn from the target one by one. Comparisons and quotients are those of the formula in 64
 * bits, every operation rounded by itself.
 *
 * tokens (length + 1 a sequence): the drafts that stand, the drawn token, -1 behind it; accepted: how many stand. A row with
 * nothing left (lse -infinity), a NaN or +infinity draws -1. A NaN in the draft's row refuses its draft and takes nothing
 * away. noise is positive; at 0 it wins where its rate is positive, and a token whose noise is negative or NaN is not drawn
 * (its rate still counts as one that is left: where no other is, -1 is drawn).
 *
 * Greedy sequences: top_index (null: none; length + 1 a sequence) holds the target's most likely token for every row, as
 * a3b_token_logprobs gives with one alternative. A sequence whose first entry is a token is verified greedily: draft i stands
 * while it equals top_index i, and the next entry follows. logits may be null if all sequences are greedy; then lse, uniform
 * and noise may be, too.
 *
 * noise: row b starts at element b * noise_stride; everything else but the logits is dense. index_dtype is that of drafts, top_index, tokens and
 * accepted. scale, draft_scale: between 2^-20 and 2^20. The outputs lie apart from one another and from the inputs. One
 * launch. At most 2^31 - 1 rows of 2^31 - 65 logits (A3B_ERR_TOO_LARGE). */
typedef struct a3b_verify_drafts_args
{
    uint64_t batch, length, vocab;
    a3b_rows logits, draft_logits; /* read; outer: the sequence, inner: the position */
    float const* lse;
    float const* draft_lse;
    double scale, draft_scale;
    void const* drafts;
    void const* top_index;
    float const* uniform;
    float const* noise;
    int64_t noise_stride;
    void* tokens;
    void* accepted;
    int32_t dtype, index_dtype;
} a3b_verify_drafts_args;
A3B_API int a3b_verify_drafts(a3b_stream_t stream, a3b_verify_drafts_args const* args);

/* ----------------------------------------------------------------------------------------------------- nBody */

/* UpdateVelocitiesKernel (example/nBody/src/Kernels.hpp:24-124) for the i-bodies [i_begin, i_begin + i_count) against
 * all n_all j-bodies: v_i += dt * sum_j m_j d_ij / ((|d_ij|^2 + eps)^3)^(1/2), d_ij = p_j - p_i.
 * m, x, y, z hold all n_all bodies; vx, vy, vz hold the i_count local velocities. fp32, SoA. */
A3B_API int a3b_nbody_update_velocities(a3b_stream_t stream, float const* m, float const* x, float const* y, float const* z,
                                uint64_t n_all, uint64_t i_begin, uint64_t i_count, float* vx, float* vy, float* vz,
                                float dt, float eps);

/* One full nBody time step for the local bodies (nBody.cpp:188-205): the velocity kick above for [i_begin,
 * i_begin + i_count), then the drift x += v*dt of those bodies' positions (x + i_begin ...), in one call. The positions
 * of all n_all bodies are read before any is moved (the drift runs after every force is known). */
A3B_API int a3b_nbody_step(a3b_stream_t stream, float const* m, float* x, float* y, float* z, uint64_t n_all,
                   uint64_t i_begin, uint64_t i_count, float* vx, float* vy, float* vz, float dt, float eps);

/* --------------------------------------------------------------------------------------------------- HACCmk */

/* HACCmk's short-range force step (benchmark/HACCmk/src/main_alpaka.cpp:47-123 Step10Kernel, CPU gold
 * helper.hpp:19-66): for the first n1 particles (targets) against all n2 particles (sources),
 *   d = p_j - p_i, r2 = |d|^2, m = (r2 < fsrrmax2) ? mass_j : 0, f = r2 + mp_rsm2,
 *   f = m * (1 / (f * sqrt f) - poly(r2)),  v_i = fcoeff * sum_j f * d   (written to vx2/vy2/vz2[i], i < n1).
 * fp32, SoA; 0 <= n1 <= n2. */
A3B_API int a3b_haccmk_step10(a3b_stream_t stream, float const* xx, float const* yy, float const* zz, float const* mass,
                              int n1, int n2, float fsrrmax2, float mp_rsm2, float fcoeff, float* vx2, float* vy2,
                              float* vz2);

/* ------------------------------------------------------------------------------------------------------ heat */

/* StencilKernel (example/heatEquation2D/src/StencilKernel.hpp:26-86): one explicit 5-point Jacobi step on a row-major
 * fp64 grid of (rows + 2) x (cols + 2) cells (1-cell halo ring), consecutive rows `pitch_elems` apart. Updates interior
 * rows [row_begin, row_end) (1 <= row_begin <= row_end <= rows + 1) and all interior columns:
 *   next = cur*(1 - 2rX - 2rY) + west*rX + east*rX + north*rY + south*rY   (left to right, each op rounded).
 * The halo ring of `next` is not written. */
A3B_API int a3b_heat_step(a3b_stream_t stream, double const* cur, double* next, uint64_t rows, uint64_t cols,
                  uint64_t pitch_elems, uint64_t row_begin, uint64_t row_end, double rX, double rY);

/* Initial field of the heat workload: interior sin(pi*j*dx)*sin(pi*(i + row_offset)*dy), ring set to 0 only at the
 * global boundary (row i of this slab is global row i + row_offset). grid as in a3b_heat_step, rows = local rows. */
A3B_API int a3b_heat_init(a3b_stream_t stream, double* u, uint64_t rows, uint64_t cols, uint64_t pitch_elems,
                  uint64_t row_offset, uint64_t global_rows, double dx, double dy);

/* The heatEquation2D example's own problem (example/heatEquation2D/src/analyticalSolution.hpp:17-78,
 * BoundaryKernel.hpp:23-57): writes the exact solution e^{-pi^2 t}(sin pi x + sin pi y), x = col*dx, y = row*dy, to
 * every cell (ring_only == 0, the initial field initalizeBuffer writes) or only to the cells on the global ring
 * (ring_only != 0, the time-dependent Dirichlet boundary applied after each step). Grid as in a3b_heat_step. */
A3B_API int a3b_heat_exact(a3b_stream_t stream, double* u, uint64_t rows, uint64_t cols, uint64_t pitch_elems,
                           uint64_t row_offset, uint64_t global_rows, double t, double dx, double dy, int ring_only);

/* Row slabs of the heat grid across the ranks of one node, halo exchange fused into the stencil step. alpaka3's
 * heatEquation2D example runs on one device (example/heatEquation2D/src/heatEquation2D.cpp:97-214); the row
 * decomposition with one ghost row per side is new here.
 *
 * Each rank owns a halo mailbox (a small cudaMalloc'd buffer: two ghost rows per side, double-buffered by step
 * parity, and one step flag per column block) that its upper and lower neighbours map through CUDA IPC. Create it
 * on every rank, exchange the a3b_ipc_handle_size()-byte handles (rank order), connect. */
typedef struct a3b_halo a3b_halo;
A3B_API size_t a3b_halo_bytes(uint64_t cols);
A3B_API int a3b_halo_create(int world, int rank, uint64_t cols, a3b_halo** halo, void* local_handle);
A3B_API int a3b_halo_connect(a3b_halo* halo, void const* handles);
/* Call only when no neighbour is still writing into this mailbox (after a barrier that follows the last step). */
A3B_API int a3b_halo_destroy(a3b_halo* halo);

/* Sends this rank's first and last interior rows of u (the initial field) to the neighbours' mailboxes; call once on
 * every rank after a3b_heat_init and before the first a3b_heat_step_halo. u: (rows + 2) x pitch_elems fp64, rows
 * 16-byte aligned (even pitch). */
A3B_API int a3b_heat_halo_publish(a3b_stream_t stream, a3b_halo* halo, double const* u, uint64_t rows, uint64_t cols,
                                  uint64_t pitch_elems);

/* One a3b_heat_step over the whole slab (rows 1..rows) in one launch, with the ghost rows taken from this rank's
 * mailbox (the neighbours' boundary rows of the previous step; a rank without an upper / lower neighbour uses its
 * own ghost row, the global Dirichlet ring) and its own boundary rows stored into the neighbours' mailboxes over
 * NVLink. The bands holding rows 1 and `rows` run first and wait, bounded by a3b_set_wait_timeout_ns, for the
 * neighbours' flags (a timeout raises bit 0 of the device error word); the other bands never wait. Every rank makes
 * the same sequence of publish / step calls. */
A3B_API int a3b_heat_step_halo(a3b_stream_t stream, a3b_halo* halo, double const* cur, double* next, uint64_t rows,
                               uint64_t cols, uint64_t pitch_elems, double rX, double rY);

#ifdef __cplusplus
}
#endif

#endif /* ALPAKA3_B200_H */
