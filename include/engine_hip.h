/*
 * engine_hip.h -- C-ABI of the MI355X (gfx950) matrix-multiply engine.
 *
 * This is the drop-in boundary. It is plain C: no HIP, torch or C++ types
 * cross it. Device pointers are `void*`/typed pointers to device memory,
 * streams and events are opaque handles (a HIP stream handle may be passed
 * where an `eng_stream` is expected; NULL is the legacy default stream),
 * dimensions are signed 64-bit, and every function returns a status code:
 *
 *   ENG_OK (0)                 success
 *   ENG_INVALID_ARGUMENT (1)   a precondition failed; nothing was launched
 *   ENG_DEVICE_ERROR (2)       the HIP runtime reported an error
 *
 * After a non-zero status, eng_last_error() returns the message of the
 * failure on the calling thread, formatted like the reference's EngineError:
 *   "[engine] <file>:<line>\n  check failed: <expr>\n  <message>"
 * and containing the same substrings the reference's contract tests match
 * ("null", "non-negative", "negative", "eps").
 *
 * The C++17 launch API of the reference (namespace engine::cuda, header
 * include/engine/kernels.hpp) is restated on top of this ABI by the headers
 * under include/engine/ in this repository.
 *
 * Layout convention (reference include/engine/cpu_ref.hpp:14-17): all 2-D
 * data is row-major and contiguous. GEMV/RMSNorm+linear weights are stored
 * [K x N] and out = x . W (reference include/engine/kernels.hpp:83-99).
 */
#ifndef ENGINE_HIP_H
#define ENGINE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ENG_OK 0
#define ENG_INVALID_ARGUMENT 1
#define ENG_DEVICE_ERROR 2

/* IEEE-754 binary16 bit pattern (the reference's engine::half). */
typedef uint16_t eng_half;
/* Opaque stream / event handles (hipStream_t / hipEvent_t underneath). */
typedef void* eng_stream;
typedef void* eng_event;
/* Opaque pooled-allocator handle. */
typedef struct eng_pool_s* eng_pool;

/* Device kinds, numbered like the reference's engine::Device
 * (include/engine/tensor.hpp:50-53): 0 = host, 1 = the GPU. */
#define ENG_DEVICE_CPU 0
#define ENG_DEVICE_GPU 1

/* Stream / event flags (values of hipStreamNonBlocking / hipEventDisableTiming). */
#define ENG_STREAM_DEFAULT 0u
#define ENG_STREAM_NON_BLOCKING 1u
#define ENG_EVENT_DEFAULT 0u
#define ENG_EVENT_DISABLE_TIMING 2u

/* Message of the last failed call on this thread ("" if none). */
const char* eng_last_error(void);
/* Library build string: "engine_hip <version> gfx950 <build flags> git <source revision>". */
const char* eng_build_info(void);

/* ------------------------------------------------------------------------
 * Device queries. Replace engine::cuda_device_count / cuda_device_summary /
 * cuda_peak_bandwidth_gbs / cuda_driver_version / cuda_clock_rate_khz /
 * cuda_live_sm_clock_mhz / cuda_live_mem_clock_mhz
 * (reference include/engine/cuda_device.hpp:20-48, src/cuda_device.cpp:51-222).
 * Like the reference, the count answers 0 (not an error) when no device or
 * driver is present.
 * ---------------------------------------------------------------------- */
int eng_device_count(int* count);
int eng_device_summary(char* buf, size_t len);
/* Theoretical peak HBM bandwidth from the device's memory clock and bus
 * width (clock x bus bytes x 2), in GB/s. */
int eng_peak_bandwidth_gbs(double* gbs);
int eng_driver_version(char* buf, size_t len);
int eng_clock_rate_khz(int* khz);
/* Live clocks in MHz, read on each call from the amdgpu driver's sysfs node
 * of the device's PCI function: the current level of pp_dpm_sclk /
 * pp_dpm_mclk, else the hwmon freq1_input / freq2_input. Without either, the
 * engine clock falls back to the nominal clock and the memory clock reports 0,
 * as the reference does without NVML (src/cuda_device.cpp:196-222).
 * eng_live_clock_source names the files read ("unavailable" for a fallback). */
int eng_live_sm_clock_mhz(int* mhz);
int eng_live_mem_clock_mhz(int* mhz);
int eng_live_clock_source(char* buf, size_t len);
/* Architecture the device reports (e.g. "gfx950:sramecc+:xnack-"). */
int eng_device_arch(char* buf, size_t len);
int eng_device_cu_count(int* cus);

/* ------------------------------------------------------------------------
 * Memory. Replace the cudaMalloc / cudaFree / cudaMemcpy / cudaMemset calls
 * behind engine::DeviceBuffer<T> (reference include/engine/device_buffer.hpp:
 * 33-92) and Storage (src/tensor.cpp:56-95).
 * ---------------------------------------------------------------------- */
int eng_malloc(void** ptr, size_t bytes);
int eng_free(void* ptr);
/* The blocking calls (eng_memcpy_h2d / _d2h / _d2d, eng_memset) have finished
 * on the device when they return, so work queued afterwards on any stream,
 * non-blocking ones included, sees their bytes. */
int eng_memcpy_h2d(void* dst, const void* src, size_t bytes);
int eng_memcpy_d2h(void* dst, const void* src, size_t bytes);
int eng_memcpy_d2d(void* dst, const void* src, size_t bytes);
int eng_memcpy_h2d_async(void* dst, const void* src, size_t bytes, eng_stream stream);
int eng_memcpy_d2h_async(void* dst, const void* src, size_t bytes, eng_stream stream);
int eng_memset(void* ptr, int value, size_t bytes);
/* The low byte of `value` into `bytes` bytes, ordered on `stream`. A fill
 * kernel (not hipMemsetAsync), so it may be captured into a HIP graph. */
int eng_memset_async(void* ptr, int value, size_t bytes, eng_stream stream);
int eng_device_sync(void);
/* hipGetLastError(), cleared; ENG_DEVICE_ERROR with its text if set. */
int eng_check_last_launch(void);

/* ------------------------------------------------------------------------
 * Streams and events. Replace engine::CudaStream / CudaEvent
 * (reference include/engine/cuda_stream.hpp:21-124, src/cuda_stream.cpp:11-38).
 * Streams are created at the default priority. eng_stream_destroy waits for
 * the stream's work and releases the stream's scratch arena (the device
 * memory the split-K GEMV, split-KV attention, rmsnorm_linear at M > 1, the
 * FFN launchers and matrix products split by K reuse on that stream; it grows to
 * the largest request). Arenas are found by (device, stream handle): streams
 * created elsewhere keep theirs until the process ends, and hipStreamPerThread is
 * one handle for all host threads, so there calls that need scratch have to be
 * ordered by the caller (eng_matmul_f32, and the plain FP32 product inside the
 * other entries, uses no scratch there).
 * ---------------------------------------------------------------------- */
int eng_stream_create(eng_stream* stream, unsigned int flags);
int eng_stream_destroy(eng_stream stream);
int eng_stream_sync(eng_stream stream);
int eng_stream_wait_event(eng_stream stream, eng_event event, unsigned int flags);
/* Holds `stream` for `microseconds` of GPU time (at most 1,000,000): one
 * one-wave kernel that sleeps until the device's constant-rate clock has
 * advanced that far, then exits. A timing harness issues it before a window
 * of launches so that every launch of the window is queued before the first
 * one starts and the window measures the GPU's back-to-back rate, not the
 * host's issue rate (no reference counterpart; the reference's harness times
 * launches as the host issues them, bench/bench_harness.hpp:205-348). */
int eng_stream_delay(eng_stream stream, unsigned int microseconds);
int eng_event_create(eng_event* event, unsigned int flags);
int eng_event_destroy(eng_event event);
int eng_event_record(eng_event event, eng_stream stream);
/* *done = 1 when complete, 0 when still pending. */
int eng_event_query(eng_event event, int* done);
int eng_event_sync(eng_event event);
int eng_event_elapsed_ms(float* ms, eng_event start, eng_event end);

/* ------------------------------------------------------------------------
 * HIP graph capture of a stream. No counterpart in the reference: for decode
 * loops that issue the same launches every token (capture once, replay per
 * token). eng_graph_capture_begin starts recording the work issued on
 * `stream` (a stream from eng_stream_create, not the null stream) without
 * running it; eng_graph_capture_end stops, instantiates and returns the graph;
 * eng_graph_launch replays it on any stream. Every launcher here is
 * capture-safe once it has run eagerly on that stream at least once with
 * shapes at least as large (the stream's scratch arena is sized outside the
 * capture -- a call that would have to grow it during capture fails with a
 * message saying so; zero fills are kernels, not memsets). A failed capture
 * returns an error and leaves no graph; the stream is no longer capturing
 * either way.
 * Scratch: at capture end the call waits for the capture stream's earlier
 * (eager) work, then the graph takes over the blocks of the capture stream's
 * scratch arenas that launches captured in it leased, and the stream continues
 * on fresh blocks of the same sizes. A replay therefore shares no scratch with
 * eager calls on the capture stream or with any other graph, may run on any
 * stream, and stays valid after the capture stream is destroyed. Replays of
 * one graph share its blocks: they must not overlap (issue them on one
 * stream, or order them with events). A graph captured with HIP's own calls
 * takes no blocks over: launchers that need scratch leave the stream's arena in
 * it, so its replays have to be ordered with that stream's other work and end
 * before the stream is destroyed. The plain FP32 product (eng_matmul_f32) uses
 * no scratch in such a capture, nor in one here whose stream's arena is too small
 * for it, and then sums in another order than its eager call. eng_graph_destroy waits for the device
 * before freeing the graph's blocks.
 * ---------------------------------------------------------------------- */
typedef void* eng_graph;
int eng_graph_capture_begin(eng_stream stream);
int eng_graph_capture_end(eng_stream stream, eng_graph* graph);
int eng_graph_launch(eng_graph graph, eng_stream stream);
int eng_graph_destroy(eng_graph graph);

/* ------------------------------------------------------------------------
 * Pooled allocator. Replaces engine::PoolAllocator / pool_allocator(Device) /
 * AllocStats (reference include/engine/pool_allocator.hpp:27-148,
 * include/engine/allocator.hpp:34-63, src/pool_allocator.cpp:38-271):
 * power-of-two buckets of at least 256 B, 256-B alignment, slabs carved
 * most-recent-first, slab size doubling from the initial size and capped at
 * 64 MiB, stream-ordered reuse of GPU blocks through a per-block event,
 * mutex-guarded, exact statistics.
 * ---------------------------------------------------------------------- */
typedef struct eng_alloc_stats {
  uint64_t bytes_in_use;
  uint64_t bytes_reserved;
  uint64_t peak_bytes_in_use;
  uint64_t num_allocs;
  uint64_t num_driver_allocs;
} eng_alloc_stats;

int eng_pool_create(eng_pool* pool, int device, size_t initial_slab_bytes);
int eng_pool_destroy(eng_pool pool);
/* The process-wide pool of a device kind (created on first use). */
int eng_pool_default(eng_pool* pool, int device);
/* bytes == 0 yields *ptr == NULL and ENG_OK, like the reference. */
int eng_pool_allocate(eng_pool pool, size_t bytes, void** ptr);
/* Host pools: immediate. GPU pools: reuse deferred until the work queued on
 * `stream` so far completes (an event is recorded on `stream`). */
int eng_pool_deallocate(eng_pool pool, void* ptr, eng_stream stream);
int eng_pool_stats(eng_pool pool, eng_alloc_stats* stats);
int eng_pool_reset(eng_pool pool);
/* Passthrough allocator of a device kind (reference src/allocator.cpp:42-118). */
int eng_passthrough_allocate(int device, size_t bytes, void** ptr);
int eng_passthrough_deallocate(int device, void* ptr);
int eng_passthrough_stats(int device, eng_alloc_stats* stats);

/* ------------------------------------------------------------------------
 * Host fp16 conversions (IEEE-754 round-to-nearest-even; replaces the
 * host half_to_float / float_to_half of reference include/engine/half.hpp:
 * 27-105, whose non-CUDA float->half truncates).
 * ---------------------------------------------------------------------- */
int eng_f32_to_f16_host(const float* in, eng_half* out, size_t n);
int eng_f16_to_f32_host(const eng_half* in, float* out, size_t n);

/* ------------------------------------------------------------------------
 * Kernels. All pointers are DEVICE pointers; launches are asynchronous on
 * `stream`. Preconditions, messages and zero-size behaviour follow the
 * reference launchers exactly:
 *   - null pointer           -> ENG_INVALID_ARGUMENT, "... is null" / "null device pointer"
 *   - negative dimension     -> ENG_INVALID_ARGUMENT, "... must be non-negative" / "negative dimension"
 *   - GEMV/GEMM with K == 0  -> output zero-filled on `stream`
 *   - N == 0 (GEMV), M or N == 0 (GEMM) -> no-op
 *   - rmsnorm_linear with any dimension 0 -> no-op (nothing written)
 * ---------------------------------------------------------------------- */

/* C[M x N] = A[M x K] . B[K x N], fp32 accumulate: three exact bf16 terms
 * per value on the bf16 matrix cores, small calls on the FP32 instruction.
 * Replaces engine::cuda::matmul_register_tiled
 * (reference include/engine/kernels.hpp:77-81, kernels/matmul_register_tiled.cu:176-199). */
int eng_matmul_f32(const float* A, const float* B, float* C, int64_t M, int64_t N, int64_t K,
                   eng_stream stream);

/* out[N] = x[K] . A[K x N], fp32. Replaces engine::cuda::gemv
 * (reference include/engine/kernels.hpp:83-86, kernels/gemv.cu:114-147). */
int eng_gemv_f32(const float* A, const float* x, float* out, int64_t N, int64_t K,
                 eng_stream stream);

/* out[N] = x[K] . A[K x N] with half A, x and out, fp32 accumulate, out
 * rounded to nearest even. Replaces engine::cuda::gemv_fp16
 * (reference include/engine/kernels.hpp:118-121, kernels/gemv_fp16.cu:117-149). */
int eng_gemv_f16(const eng_half* A, const eng_half* x, eng_half* out, int64_t N, int64_t K,
                 eng_stream stream);

/* out[N] = x[K] . A[K x N] with half A and fp32 x / out, fp32 accumulate.
 * Additive overload of engine::cuda::gemv_fp16 for fp16-weight decode with
 * fp32 activations (no reference counterpart; same contract as gemv_fp16). */
int eng_gemv_f16w(const eng_half* A, const float* x, float* out, int64_t N, int64_t K,
                  eng_stream stream);

/* out[r][c] = in[r][c] / sqrt(mean(in[r][:]^2) + eps) * weight[c]; weight may
 * be NULL (no gain). Replaces engine::cuda::rmsnorm
 * (reference include/engine/kernels.hpp:61-63, kernels/rmsnorm.cu:171-192). */
int eng_rmsnorm_f32(const float* in, const float* weight, float* out, int64_t rows,
                    int64_t cols, float eps, eng_stream stream);

/* out[M x N] = RMSNorm(in[M x K], rms_weight, eps) . W[K x N]; rms_weight may be
 * NULL. One fused kernel: the sum of squares is reduced inside the GEMV/GEMM.
 * Replaces engine::cuda::rmsnorm_linear
 * (reference include/engine/kernels.hpp:92-99, kernels/rmsnorm_linear.cu:173-201). */
int eng_rmsnorm_linear_f32(const float* in, const float* rms_weight, const float* W, float* out,
                           int64_t M, int64_t N, int64_t K, float eps, eng_stream stream);

/* As eng_rmsnorm_linear_f32 with an fp16 weight matrix W[K x N] (fp32 in / out).
 * Additive overload (no reference counterpart; same contract). */
int eng_rmsnorm_linear_f16w(const float* in, const float* rms_weight, const eng_half* W,
                            float* out, int64_t M, int64_t N, int64_t K, float eps,
                            eng_stream stream);

/* eng_rmsnorm_linear_f16w for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc): no counterpart in the reference. Same arguments, kernels and
 * bits as eng_rmsnorm_linear_f16w, for M <= 16 rows (decode and small
 * batches); the split-K partial sums live in a static device buffer of
 * 8 MiB + 64 KiB per GPU, held until the process ends, instead of the stream's
 * scratch arena. Nothing is allocated. Fails with a message (status 1) for
 * M > 16 or a shape whose partial sums would exceed the buffer. Every call on
 * a GPU shares that GPU's buffer: calls that overlap on one GPU (different
 * streams or host threads without ordering) race, so order them. */
int eng_rmsnorm_linear_f16w_noalloc(const float* in, const float* rms_weight, const eng_half* W,
                                    float* out, int64_t M, int64_t N, int64_t K, float eps,
                                    eng_stream stream);

/* Output-major weights (no reference counterpart; additive). W is row-major
 * [N x K] -- one contiguous row of K weights per output, the layout of the
 * decode configurations "y = W.x, W [out x in]" -- and
 *   y[N] = W[N x K] . x[K]                                 (eng_gemv_*_nk)
 *   out[M x N] = RMSNorm(in[M x K], rms_weight, eps) . W^T  (eng_rmsnorm_linear_*_nk)
 * Same preconditions, messages and zero-size rules as the reference-layout
 * functions above (K == 0: the GEMVs zero-fill, rmsnorm_linear writes nothing).
 * Each output row is one contiguous stream, so M == 1 needs no split-K
 * reduction; M > 1 takes the few-row kernels and the GEMMs with B read as B^T. */
int eng_gemv_f16w_nk(const eng_half* W, const float* x, float* y, int64_t N, int64_t K,
                     eng_stream stream);
int eng_gemv_f32_nk(const float* W, const float* x, float* y, int64_t N, int64_t K,
                    eng_stream stream);
int eng_rmsnorm_linear_f16w_nk(const float* in, const float* rms_weight, const eng_half* W,
                               float* out, int64_t M, int64_t N, int64_t K, float eps,
                               eng_stream stream);
int eng_rmsnorm_linear_f32_nk(const float* in, const float* rms_weight, const float* W,
                              float* out, int64_t M, int64_t N, int64_t K, float eps,
                              eng_stream stream);

/* Replaces engine::cuda::rmsnorm_linear_fused_direct
 * (reference include/engine/kernels.hpp:101-104, kernels/rmsnorm_linear.cu:143-171),
 * the benchmarking entry that forces the fused kernel for every M. Here every
 * M is served by fused kernels already, so it runs the same code as
 * eng_rmsnorm_linear_f32. */
int eng_rmsnorm_linear_fused_direct_f32(const float* in, const float* rms_weight,
                                        const float* W, float* out, int64_t M, int64_t N,
                                        int64_t K, float eps, eng_stream stream);

/* ------------------------------------------------------------------------
 * The ops either side of the linear layers (SwiGLU FFN, residual stream).
 * ---------------------------------------------------------------------- */

/* out[i] = a[i] + b[i], bit-exact fp32 addition. n < 0 -> "n must be
 * non-negative"; n == 0 returns before the pointer check; null -> "null device
 * pointer". Replaces engine::cuda::vector_add
 * (reference include/engine/kernels.hpp:47-50, kernels/vector_add.cu:119-149). */
int eng_vector_add_f32(const float* a, const float* b, float* out, int64_t n, eng_stream stream);

/* sum_out = x + residual (bit-exact); norm_out = sum_out / sqrt(mean(sum_out^2)
 * + eps) * weight, per row of [rows x cols]; weight may be NULL, the other
 * pointers may not ("null device pointer"); "negative dimension"; "eps must be
 * non-negative"; rows or cols == 0 writes nothing. Replaces
 * engine::cuda::residual_rmsnorm (reference include/engine/kernels.hpp:106-112,
 * kernels/residual_rmsnorm.cu:124-150). */
int eng_residual_rmsnorm_f32(const float* x, const float* residual, const float* weight,
                             float* norm_out, float* sum_out, int64_t rows, int64_t cols,
                             float eps, eng_stream stream);

/* out[i] = SiLU(gate[i]) * up[i], SiLU(g) = g / (1 + exp(-g)), fp32 (and half
 * in / out with fp32 arithmetic, rounded to nearest even). "gate is null" /
 * "up is null" / "out is null"; "n must be non-negative"; n == 0 is a no-op.
 * Replace engine::cuda::swiglu / swiglu_fp16
 * (reference include/engine/kernels.hpp:138-142, kernels/swiglu.cu:155-227). */
int eng_swiglu_f32(const float* gate, const float* up, float* out, int64_t n, eng_stream stream);
int eng_swiglu_f16(const eng_half* gate, const eng_half* up, eng_half* out, int64_t n,
                   eng_stream stream);

/* act[M x N] = SiLU(xn . Wg^T) * (xn . Wu^T), xn = RMSNorm(in[M x K], rms_weight,
 * eps), with output-major W_gate, W_up [N x K]: the gate / up half of a SwiGLU
 * FFN in one call (no reference counterpart: the reference composes rmsnorm,
 * two GEMV / GEMMs and swiglu, tests/test_kernels.cu:2867-2898). Decode
 * (M == 1) is a single fused launch; other shapes use scratch for gate
 * and up. rms_weight may be NULL. Messages: "negative dimension", "null device
 * pointer", "eps must be non-negative"; any zero dimension writes nothing. */
int eng_rmsnorm_linear_swiglu_f16w_nk(const float* in, const float* rms_weight,
                                      const eng_half* W_gate, const eng_half* W_up, float* act,
                                      int64_t M, int64_t N, int64_t K, float eps,
                                      eng_stream stream);
int eng_rmsnorm_linear_swiglu_f32_nk(const float* in, const float* rms_weight,
                                     const float* W_gate, const float* W_up, float* act,
                                     int64_t M, int64_t N, int64_t K, float eps,
                                     eng_stream stream);

/* The same with reference-layout W_gate, W_up [K x N] (the layout of
 * rmsnorm_linear, include/engine/kernels.hpp:92-99; no reference counterpart:
 * the reference composes two rmsnorm_linear calls and swiglu,
 * tests/test_kernels.cu:2867-2898). Decode (up to 16 rows, N a multiple of 8
 * fp16 / 4 fp32 elements, 16-byte aligned weights) is, per pass of up to 4
 * rows, one split-K launch over both matrices and one reduce launch with the
 * SwiGLU epilogue; its result equals that composition bit for bit. Same
 * messages as the _nk form. */
int eng_rmsnorm_linear_swiglu_f16w(const float* in, const float* rms_weight,
                                   const eng_half* W_gate, const eng_half* W_up, float* act,
                                   int64_t M, int64_t N, int64_t K, float eps,
                                   eng_stream stream);
int eng_rmsnorm_linear_swiglu_f32(const float* in, const float* rms_weight,
                                  const float* W_gate, const float* W_up, float* act, int64_t M,
                                  int64_t N, int64_t K, float eps, eng_stream stream);

/* ------------------------------------------------------------------------
 * Decode attention over an fp16 KV cache, and its bridge kernels.
 * ---------------------------------------------------------------------- */

/* Single-token decode attention with split-KV FlashDecoding: for each query
 * head h, out[h] = softmax(scale * K_g . q[h]) . V_g over keys 0..kv_len-1 of
 * KV head g = h / (n_heads / n_kv_heads). q / out [n_heads, head_dim] half;
 * K / V head-major, key j of KV head g at g * kv_head_stride + j * head_dim.
 * split_kv = 0 picks the split count; the query heads of a GQA group share
 * each K / V load. Messages (order as the reference): "q is null", "k is
 * null", "v is null", "out is null", "kv_len must be non-negative", "n_heads
 * must be positive", "n_kv_heads must be positive", "n_heads must be divisible
 * by n_kv_heads", "head_dim must be 64 or 128", "scale must be finite",
 * "split_kv must be non-negative", "kv_head_stride < kv_len * head_dim";
 * kv_len == 0 zero-fills out. Replaces engine::cuda::attention_decode
 * (reference include/engine/kernels.hpp:190-194, kernels/attention_decode.cu:
 * 632-715); the _with_mode form replaces detail::attention_decode_with_mode
 * (kernels.hpp:169-174), share_gqa_kv = 0 giving one query head per workgroup. */
int eng_attention_decode_f16(const eng_half* q, const eng_half* k, const eng_half* v,
                             eng_half* out, int64_t kv_len, int64_t n_heads, int64_t n_kv_heads,
                             int64_t head_dim, int64_t kv_head_stride, float scale, int split_kv,
                             eng_stream stream);
int eng_attention_decode_with_mode_f16(const eng_half* q, const eng_half* k, const eng_half* v,
                                       eng_half* out, int64_t kv_len, int64_t n_heads,
                                       int64_t n_kv_heads, int64_t head_dim,
                                       int64_t kv_head_stride, float scale, int split_kv,
                                       int share_gqa_kv, eng_stream stream);

/* Elementwise fp32 <-> fp16 (round to nearest even); n < 0 -> "n must be
 * non-negative", n == 0 returns before the pointer checks. Replace
 * engine::cuda::detail::cast_f32_to_f16 / cast_f16_to_f32
 * (reference include/engine/kernels.hpp:176-180, kernels/attention_bridge.cu:64-84). */
int eng_cast_f32_to_f16(const float* in, eng_half* out, int64_t n, eng_stream stream);
int eng_cast_f16_to_f32(const eng_half* in, float* out, int64_t n, eng_stream stream);

/* Scatter token-major k_new / v_new [s_new, n_kv_heads, head_dim] into
 * head-major caches [n_kv_heads, kv_max_seq_len, head_dim] at positions
 * pos_offset .. pos_offset + s_new - 1. Replaces engine::cuda::detail::kv_cache_write
 * (reference include/engine/kernels.hpp:182-188, kernels/attention_bridge.cu:86-110). */
int eng_kv_cache_write_f16(const eng_half* k_new, const eng_half* v_new, eng_half* k_cache,
                           eng_half* v_cache, int64_t s_new, int64_t n_kv_heads, int64_t head_dim,
                           int64_t pos_offset, int64_t kv_max_seq_len, eng_stream stream);

/* Weight layout conversion: dst [cols x rows] = src [rows x cols] transposed,
 * bit patterns copied unchanged. Converts reference-layout weights A [K x N]
 * (out = x . A, reference include/engine/kernels.hpp:83-99) once, at load
 * time, into the output-major W [N x K] that eng_gemv_f16w_nk /
 * eng_rmsnorm_linear_f16w_nk (and the _f32 forms) stream fastest. No
 * reference counterpart (the reference has one weight layout). Messages:
 * "negative dimension", "null device pointer", "src and dst overlap"; a zero
 * dimension is a no-op. */
int eng_transpose_f16(const eng_half* src, eng_half* dst, int64_t rows, int64_t cols,
                      eng_stream stream);
int eng_transpose_f32(const float* src, float* dst, int64_t rows, int64_t cols,
                      eng_stream stream);

/* ------------------------------------------------------------------------
 * Weights in microscaled 4-bit floating point (MXFP4 of the OCP Microscaling
 * Formats specification v1.0; additive, no reference counterpart).
 *
 * A matrix [rows x cols] is two buffers. Each run of 32 values along a row (a
 * block; the last one of a row is filled with zeros) shares a scale 2^(s - 127)
 * held as the byte s, 255 standing for NaN; a value is a 4-bit code: sign and
 * one of 0, 0.5, 1, 1.5, 2, 3, 4, 6. With nb = ceil(cols / 32):
 *   codes   rows * nb * 16 bytes, 16-byte aligned: row r's at r * nb * 16, two
 *           values a byte, the even one in the low four bits
 *   scales  rows * nb bytes: row r's at r * nb
 *
 * eng_mx4_quantize_*: the scale's exponent is floor(log2(largest magnitude of
 * the block)) - 2, at least -127 (s = 0, also for a block of zeros); values are
 * divided by the scale and rounded to the nearest code, ties to the even one,
 * magnitudes above 6 to 6. A block that holds a NaN or an infinity gets s = 255
 * and zero codes. Output-major weights [N x K] (eng_transpose_* makes them) are
 * quantised along K, as the products below take them.
 * eng_mx4_dequantize_*: the values again, rounded to nearest even where fp16
 * does not hold them (infinity past its range).
 * rows == 0 or cols == 0 is a no-op. src / dst need no more than their type's
 * alignment; at 16 bytes and rows of whole 16 bytes they move in 16-byte pieces.
 *
 * eng_linear_mx4w_nk: y[M x N] = x[M x K] . W^T, fp32 x and y, W [N x K] as
 * above, for any M (M == 1 is the decode GEMV). K == 0 zero-fills y.
 * eng_rmsnorm_linear_mx4w_nk: out = RMSNorm(in, rms_weight, eps) . W^T, rms_weight
 * may be NULL; as for eng_rmsnorm_linear_* any zero dimension is a no-op.
 * Products are exact and sums fp32, as for fp16 weights: every fp32 activation
 * enters the matrix cores as three bf16 terms that add up to it (but for its bits
 * below 2^-133, which are dropped). Weights of 2^128 and more, 4 and 6 under the
 * scale bytes 253 and 254, are infinities: the sums they enter are infinite or NaN.
 * K is at most 2^23. The same call gives the same bits; the kernel, and with it the
 * order of the sums, depends on M, N and K. From 5 rows (below that, where X does
 * not fit the LDS: M K past 20000 or so) the stream's scratch arena is used: at 5 to
 * 64 rows up to 128 M N bytes, past them 6 bytes for each activation of a pass (as
 * many rows as make 256 MiB, at least 128) and up to 64 M N bytes.
 * ---------------------------------------------------------------------- */
int eng_mx4_quantize_f32(const float* src, uint8_t* codes, uint8_t* scales, int64_t rows,
                         int64_t cols, eng_stream stream);
int eng_mx4_quantize_f16(const eng_half* src, uint8_t* codes, uint8_t* scales, int64_t rows,
                         int64_t cols, eng_stream stream);
int eng_mx4_dequantize_f32(const uint8_t* codes, const uint8_t* scales, float* dst, int64_t rows,
                           int64_t cols, eng_stream stream);
int eng_mx4_dequantize_f16(const uint8_t* codes, const uint8_t* scales, eng_half* dst,
                           int64_t rows, int64_t cols, eng_stream stream);
int eng_linear_mx4w_nk(const float* x, const uint8_t* codes, const uint8_t* scales, float* y,
                       int64_t M, int64_t N, int64_t K, eng_stream stream);
int eng_rmsnorm_linear_mx4w_nk(const float* in, const float* rms_weight, const uint8_t* codes,
                               const uint8_t* scales, float* out, int64_t M, int64_t N, int64_t K,
                               float eps, eng_stream stream);

/* ------------------------------------------------------------------------
 * A KV cache in 8 bits for batches of sequences (additive; the fp16 cache of one
 * sequence is eng_kv_cache_write_f16 / eng_attention_decode_f16).
 *
 * Caches are e4m3 bytes (OCP FP8: no infinity, largest value 448), head-major,
 * [batch, n_kv_heads, kv_max_seq_len, head_dim], 16-byte aligned; every block of
 * ENG_KV_Q8_BLOCK tokens of a (sequence, KV head) has one fp32 scale for K and
 * one for V, [batch, n_kv_heads, ceil(kv_max_seq_len / ENG_KV_Q8_BLOCK)]. The
 * value of a code is its e4m3 value times its block's scale. A cache written by
 * other means may have any scales from zero to 2^24; V scales below 2^-40 count as
 * 2^-40, whose values an fp16 output cannot show. head_dim is 64 or 128. Positions
 * and lengths are read on the device (int32 arrays of `batch`), so a captured decode
 * step is replayed for every token.
 *
 * eng_kv_cache_write_q8: rows k_new / v_new [batch, s_new, n_kv_heads, head_dim]
 * (16-byte aligned) become tokens pos[b] .. of sequence b; the first n_new[b] of
 * its s_new rows where n_new is given, all of them where it is NULL. A block's
 * scale is the least power of two from 2^-15 to 2^8 that brings its largest
 * finite new magnitude to 448 or below, or its present scale if that is larger
 * and the block holds tokens before pos[b]; if the scale grows, the codes of
 * those tokens are rounded to it. Values are rounded to nearest even; infinities
 * and NaN become NaN codes and do not count for the scale. Tokens at or past
 * kv_max_seq_len are dropped, and a sequence with pos[b] < 0 or n_new[b] <= 0 is
 * left as it is. What a block holds behind the last new token is no longer
 * defined: those tokens are not part of the sequence. s_new <= kv_max_seq_len.
 *
 * eng_attention_decode_q8: for each sequence b and query head h,
 *   out[b][h] = softmax(scale q[b][h] . K[b][h / (n_heads / n_kv_heads)]^T) . V
 * over its first kv_len[b] tokens, q and out fp16 [batch, n_heads, head_dim]; a
 * sequence without tokens (kv_len[b] <= 0) gets zeros. max_kv_len is the caller's
 * bound on kv_len: it chooses the launch, lengths above it are taken as
 * max_kv_len. split_kv = 0 chooses the number of splits of a sequence; a
 * positive value asks for as many (at most 256, and at least one block each).
 * Blocks that a sequence's length reaches must have been written. Scores, softmax
 * and sums are fp32. More than one split uses the stream's scratch arena.
 * ---------------------------------------------------------------------- */
#define ENG_KV_Q8_BLOCK 32
int eng_kv_cache_write_q8(const eng_half* k_new, const eng_half* v_new, uint8_t* k_cache,
                          uint8_t* v_cache, float* k_scale, float* v_scale, const int32_t* pos,
                          const int32_t* n_new, int64_t batch, int64_t s_new, int64_t n_kv_heads,
                          int64_t head_dim, int64_t kv_max_seq_len, eng_stream stream);
int eng_attention_decode_q8(const eng_half* q, const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* k_scale, const float* v_scale, eng_half* out,
                            const int32_t* kv_len, int64_t batch, int64_t n_heads,
                            int64_t n_kv_heads, int64_t head_dim, int64_t max_kv_len,
                            int64_t kv_max_seq_len, float scale, int split_kv, eng_stream stream);

/* ------------------------------------------------------------------------
 * Attention over long contexts (additive, no reference counterpart): new tokens of
 * a batch with a sliding window, and single tokens of sequences that share a prefix.
 * Caches are head-major, [batch, n_kv_heads, kv_max_seq_len, head_dim], 16-byte
 * aligned: fp16 (each sequence's as eng_kv_cache_write_f16 fills it) or 8-bit with
 * scales (eng_kv_cache_write_q8's). head_dim is 64 or 128. Positions, counts and
 * lengths are int32 arrays on the device. Scores, softmax and sums are fp32. Weights
 * enter their products with V as two fp16 terms (22 bits) for single tokens (s_new ==
 * 1), and over a prefix for up to 128 query rows of a KV head (sequences of a group
 * times n_heads / n_kv_heads), and rounded to fp16 once past that and for more new
 * tokens. A row that sees no key, or none whose score is above -inf, gets zeros. What
 * a query does not see does not reach its result, infinities and NaN included; what it
 * sees of them in V does: an infinity stays one, two of unlike signs give NaN.
 *
 * eng_attention_window_*: q and out [batch, s_new, n_heads, head_dim]. Query i of
 * sequence b stands at position p = pos[b] + i, and its K and V rows and all before
 * them are in the caches (write them first). It sees the keys j <= p, of these with
 * window > 0 those with j > p - window or j < sinks; window == 0 is no window. s_new
 * is a prompt's length, a piece's or 1. The first n_new[b] of a sequence's s_new
 * queries are computed (all of them where n_new is NULL, none where n_new[b] or pos[b]
 * is below zero) and the rows of out behind them left as they were. Keys at or past
 * max_kv_len, the caller's bound on pos + n_new, are not seen; it and s_new choose the
 * launch. Single tokens over 8-bit caches without a window are eng_attention_decode_q8's
 * too: that one is the faster where lengths come near their bound, this one where they
 * are far below.
 *
 * eng_attention_prefix_*: one query of each sequence, q and out [batch, n_heads,
 * head_dim], over the first prefix_len[g] tokens of prefix g, shared by the batch /
 * n_prefix sequences of group g = b / (batch / n_prefix), and then the first
 * kv_len[b] of its own, in one softmax. The prefixes are caches of their own,
 * [n_prefix, n_kv_heads, prefix_max_seq_len, head_dim], each read from memory once
 * for its group (past 16 query rows of a KV head again from the L2). Lengths past
 * max_prefix_len / max_kv_len are taken as these, lengths below zero as zero.
 *
 * split_kv = 0 chooses the number of pieces that a row's keys are computed in; a
 * positive value asks for as many (at most 256, prefix and own keys 128 each). More
 * than one uses the stream's scratch arena (eng_attention_prefix_* always does). The
 * same call gives the same bits; the order of the sums, and with it the last bits,
 * depends on the shape, on max_kv_len and on split_kv.
 * ---------------------------------------------------------------------- */
int eng_attention_window_f16(const eng_half* q, const eng_half* k_cache, const eng_half* v_cache,
                             eng_half* out, const int32_t* pos, const int32_t* n_new, int64_t batch,
                             int64_t s_new, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                             int64_t window, int64_t sinks, int64_t max_kv_len,
                             int64_t kv_max_seq_len, float scale, int split_kv, eng_stream stream);
int eng_attention_window_q8(const eng_half* q, const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* k_scale, const float* v_scale, eng_half* out,
                            const int32_t* pos, const int32_t* n_new, int64_t batch, int64_t s_new,
                            int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t window,
                            int64_t sinks, int64_t max_kv_len, int64_t kv_max_seq_len, float scale,
                            int split_kv, eng_stream stream);
int eng_attention_prefix_f16(const eng_half* q, const eng_half* k_prefix, const eng_half* v_prefix,
                             const int32_t* prefix_len, const eng_half* k_cache,
                             const eng_half* v_cache, const int32_t* kv_len, eng_half* out,
                             int64_t n_prefix, int64_t batch, int64_t n_heads, int64_t n_kv_heads,
                             int64_t head_dim, int64_t max_prefix_len, int64_t prefix_max_seq_len,
                             int64_t max_kv_len, int64_t kv_max_seq_len, float scale, int split_kv,
                             eng_stream stream);
int eng_attention_prefix_q8(const eng_half* q, const uint8_t* k_prefix, const uint8_t* v_prefix,
                            const float* k_prefix_scale, const float* v_prefix_scale,
                            const int32_t* prefix_len, const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* k_scale, const float* v_scale, const int32_t* kv_len,
                            eng_half* out, int64_t n_prefix, int64_t batch, int64_t n_heads,
                            int64_t n_kv_heads, int64_t head_dim, int64_t max_prefix_len,
                            int64_t prefix_max_seq_len, int64_t max_kv_len, int64_t kv_max_seq_len,
                            float scale, int split_kv, eng_stream stream);

/* ------------------------------------------------------------------------
 * Beam search over a batch of groups of `beams` sequences (additive, no reference
 * counterpart): the next candidates, and the caches brought in line with them.
 *
 * eng_beam_select_*: logits [batch * beams rows of ld], the first `vocab` of a row
 * counting; scores [batch, beams], the beams' sums of log-probabilities so far.
 * Candidate (b, t) scores scores[b] + logits[b][t] - log sum_u exp logits[b][u]. The
 * n_out best of a group's beams * vocab candidates come out in descending order:
 * out_scores, out_parent (the beam, 0 .. beams - 1) and out_token [batch, n_out].
 * Candidates of one beam are compared by their logits, those of unlike beams by
 * their scores in 64 bits; ties go to the lower beam, then the lower token. The sums
 * of exponentials are fp32, and out_scores with them good to 2e-6 and their own
 * rounding; a group in which that leaves an order open has them formed again in 64
 * bits, which takes it longer (not for beams of equal logits: sums that agree in every
 * bit count as equal). finished
 * [batch, beams] (bytes; NULL: none) marks beams that have ended: such a beam has
 * one candidate, token eos with its score unchanged, whatever its logits are. out_finished
 * [batch, n_out] (may be NULL) is 1 where the parent has ended or the token is eos
 * (eos < 0: no token is). A candidate whose score is -inf or no number ranks last, as
 * -inf: all of a beam's whose score is not finite or whose row holds a NaN, +inf or
 * only -inf, and all but one of a finished beam's. beams is 1 to 32, n_out 1 to 64 and
 * at most beams * vocab. Outputs must not overlap inputs. Uses the stream's scratch
 * arena.
 *
 * eng_kv_cache_reorder_*: sequence (g, j) of the caches [batch * beams, n_kv_heads,
 * kv_max_seq_len, head_dim] gets the first kv_len[g beams + p] tokens of sequence
 * (g, p), p = parent[g][j] (out_parent with n_out == beams), into buffers of the
 * same shape, or, with the same pointers as source and destination, in place: beams
 * that keep their place (p == j) are then not touched. 8-bit caches move with the
 * scales of the blocks that the tokens reach. What lies behind the length stays as it
 * was, fp16 values or 8-bit codes, and so does a sequence whose p is outside 0 ..
 * beams - 1; codes in the last block that is reached are under the new scale then, so
 * what they stood for is lost. Lengths past max_kv_len are taken as it. kv_len itself
 * is not reordered: where a group's lengths differ, the next step needs it gathered by
 * parent. Source and destination
 * buffers are the same or do not overlap; beams is 1 to 32, head_dim 64 or 128, caches
 * are 16-byte aligned.
 * ---------------------------------------------------------------------- */
int eng_beam_select_f32(const float* logits, int64_t ld, const float* scores, const uint8_t* finished,
                        float* out_scores, int32_t* out_parent, int32_t* out_token,
                        uint8_t* out_finished, int64_t batch, int64_t beams, int64_t n_out,
                        int64_t vocab, int64_t eos, eng_stream stream);
int eng_beam_select_f16(const eng_half* logits, int64_t ld, const float* scores, const uint8_t* finished,
                        float* out_scores, int32_t* out_parent, int32_t* out_token,
                        uint8_t* out_finished, int64_t batch, int64_t beams, int64_t n_out,
                        int64_t vocab, int64_t eos, eng_stream stream);
int eng_kv_cache_reorder_f16(const eng_half* k_src, const eng_half* v_src, eng_half* k_dst, eng_half* v_dst,
                             const int32_t* parent, const int32_t* kv_len, int64_t batch, int64_t beams,
                             int64_t n_kv_heads, int64_t head_dim, int64_t max_kv_len,
                             int64_t kv_max_seq_len, eng_stream stream);
int eng_kv_cache_reorder_q8(const uint8_t* k_src, const uint8_t* v_src, const float* k_scale_src,
                            const float* v_scale_src, uint8_t* k_dst, uint8_t* v_dst, float* k_scale_dst,
                            float* v_scale_dst, const int32_t* parent, const int32_t* kv_len,
                            int64_t batch, int64_t beams, int64_t n_kv_heads, int64_t head_dim,
                            int64_t max_kv_len, int64_t kv_max_seq_len, eng_stream stream);

/* ------------------------------------------------------------------------
 * ENGREF01 tensor files and device weight slabs.
 *
 * The container is the reference's golden format (tools/gen_reference.py:
 * 56-83, tests/golden.hpp:21-33): "ENGREF01", int32 count, then per tensor
 * int32 name length, name, int32 dtype, int32 ndim, int64 dims, int64 byte
 * count, data. The reference reader (tests/golden.cpp:104-209, which these
 * functions replace) accepts dtype 0 only; here 1 stores IEEE binary16
 * weights at native size and 2 float64. A file is memory-mapped and checked
 * as the reference checks it (messages: "bad magic", "implausible tensor
 * count", "implausible name length", "truncated tensor name", "has dtype",
 * "implausible ndim", "negative dimension", "header says ... bytes but its
 * shape implies", "truncated data", "duplicate tensor name", "unexpected
 * trailing bytes", "unexpected end of file while reading"); a missing
 * tensor name reports the names present ("not found. Available:", as
 * tests/golden.cpp:197-205). The slab is the on-disk-to-HBM step of the
 * reference's planned mmap weight loader (README.md:247): every tensor at a
 * 256-byte aligned offset, in file order, in one device allocation.
 * ---------------------------------------------------------------------- */

#define ENG_ENGREF_F32 0
#define ENG_ENGREF_F16 1
#define ENG_ENGREF_F64 2

typedef struct eng_engref_s* eng_engref;

/* Maps and validates `path`; *file is NULL on failure. A handle is
 * read-only after open and may be shared by threads. */
int eng_engref_open(const char* path, eng_engref* file);
/* Unmaps the file; pointers returned for it become invalid. NULL is a no-op. */
int eng_engref_close(eng_engref file);
int eng_engref_count(eng_engref file, int32_t* count);
/* Index of the tensor called `name` (unknown name: ENG_INVALID_ARGUMENT). */
int eng_engref_find(eng_engref file, const char* name, int32_t* index);
/* Tensor `index` (0 .. count-1, file order). Any output pointer may be NULL.
 * name (NUL-terminated), dims[ndim] and host_data (the mapped bytes,
 * little-endian, not necessarily aligned) live until eng_engref_close;
 * slab_offset is the tensor's byte offset in the slab. */
int eng_engref_tensor(eng_engref file, int32_t index, const char** name, int32_t* dtype,
                      int32_t* ndim, const int64_t** dims, int64_t* nbytes,
                      const void** host_data, int64_t* slab_offset);
/* Bytes of device memory the slab needs (a multiple of 256). */
int eng_engref_slab_bytes(eng_engref file, int64_t* bytes);
/* Copies every tensor into the caller's device allocation `slab` (256-byte
 * aligned, `capacity` >= eng_engref_slab_bytes) through pinned staging
 * buffers on `stream`; returns when the copies are complete. Padding bytes
 * between tensors are left as they were. Messages: "capacity must be
 * non-negative", "slab capacity ... bytes needed", "slab is null", "slab must
 * be 256-byte aligned". */
int eng_engref_upload(eng_engref file, void* slab, int64_t capacity, eng_stream stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* ENGINE_HIP_H */
