/* Plain-C entry points for the parts of the reference API that exist only as
 * C++ (namespace cumpsgemm, include/cumpsgemm/cumpsgemm.hpp:45-129, and
 * namespace cumpsgemm::hijack_control, include/cumpsgemm/hijack_control.hpp:7-34),
 * so that ctypes / cgo / JNI style bindings can reach them without C++ name
 * mangling.  Suffix _s = float, _c = cuComplex.  Every function forwards to
 * the C++ function named in its comment; argument meaning is identical.
 *
 * The last section adds what a multi-GPU caller needs to make the AUTO /
 * FP16TCEC_SCALING decisions global across ranks; it has no counterpart in
 * the reference, which is single-GPU.
 */
#ifndef CUMPSGEMM_B200_CUMPSGEMM_EXT_H
#define CUMPSGEMM_B200_CUMPSGEMM_EXT_H
#include "cumpsgemm.h"
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- exponent statistics ------------------------------------------------ */
/* cumpsgemm::exp_stats_ext<T>  (reference: src/exp_stats.cu:502-525) */
unsigned cuMpSGEMM_exp_stats_ext_s(cuMpSGEMM_handle_t handle, unsigned m, unsigned n,
                                   const float *ptr, unsigned ld, unsigned batch_size,
                                   unsigned stride);
unsigned cuMpSGEMM_exp_stats_ext_c(cuMpSGEMM_handle_t handle, unsigned m, unsigned n,
                                   const cuComplex *ptr, unsigned ld, unsigned batch_size,
                                   unsigned stride);
/* cumpsgemm::exp_max_ext<T>  (reference: src/exp_stats.cu:534-557) */
unsigned cuMpSGEMM_exp_max_ext_s(cuMpSGEMM_handle_t handle, unsigned m, unsigned n,
                                 const float *ptr, unsigned ld, unsigned batch_size,
                                 unsigned stride);
unsigned cuMpSGEMM_exp_max_ext_c(cuMpSGEMM_handle_t handle, unsigned m, unsigned n,
                                 const cuComplex *ptr, unsigned ld, unsigned batch_size,
                                 unsigned stride);
/* cumpsgemm::get_exp_stats  (reference: src/exp_stats.cu:615-629).  Synchronises. */
void cuMpSGEMM_get_exp_stats(cuMpSGEMM_handle_t handle, unsigned buffer_id,
                             size_t *underflow_count, size_t *total_count);
/* cumpsgemm::get_current_exp_stats_buffer_id / reset_exp_stats_buffer_id */
unsigned cuMpSGEMM_get_current_exp_stats_buffer_id(cuMpSGEMM_handle_t handle);
void cuMpSGEMM_reset_exp_stats_buffer_id(cuMpSGEMM_handle_t handle);
/* cumpsgemm::set_exp_stats_params  (reference: src/exp_stats.cu:631-638) */
void cuMpSGEMM_set_exp_stats_params(cuMpSGEMM_handle_t handle, float ignore_threshold,
                                    float underflow_threshold, float underflow_ratio_tolerance);
/* cumpsgemm::enable_exp_stats / disable_exp_stats */
void cuMpSGEMM_enable_exp_stats(cuMpSGEMM_handle_t handle);
void cuMpSGEMM_disable_exp_stats(cuMpSGEMM_handle_t handle);
/* cumpsgemm::get_max_exp  (reference: src/dynamic_scaling.cu:352-361).  Synchronises. */
float cuMpSGEMM_get_max_exp(cuMpSGEMM_handle_t handle, unsigned buffer_id);
/* cumpsgemm::get_exp_stats_compute_mode_level  (reference: src/exp_stats.cu:675-683) */
int cuMpSGEMM_get_exp_stats_compute_mode_level(cuMpSGEMM_handle_t handle, unsigned buffer_id);

/* ---- dynamic scaling (reference: src/dynamic_scaling.cu:227-350) --------- */
void cuMpSGEMM_scale_A_s(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                         unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                         float *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_scale_A_c(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                         unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                         cuComplex *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_scale_B_s(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                         unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                         float *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_scale_B_c(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                         unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                         cuComplex *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_scale_C_s(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_A_id,
                         unsigned exp_stats_buffer_B_id, unsigned dynamic_launch_flag_buffer_id,
                         unsigned m, unsigned n, float *ptr, unsigned ld, unsigned batch_size,
                         unsigned stride);
void cuMpSGEMM_scale_C_c(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_A_id,
                         unsigned exp_stats_buffer_B_id, unsigned dynamic_launch_flag_buffer_id,
                         unsigned m, unsigned n, cuComplex *ptr, unsigned ld, unsigned batch_size,
                         unsigned stride);
void cuMpSGEMM_reset_scale_A_s(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                               unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                               float *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_reset_scale_A_c(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                               unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                               cuComplex *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_reset_scale_B_s(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                               unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                               float *ptr, unsigned ld, unsigned batch_size, unsigned stride);
void cuMpSGEMM_reset_scale_B_c(cuMpSGEMM_handle_t handle, unsigned exp_stats_buffer_id,
                               unsigned dynamic_launch_flag_buffer_id, unsigned m, unsigned n,
                               cuComplex *ptr, unsigned ld, unsigned batch_size, unsigned stride);

/* ---- dynamic launch (reference: src/dynamic_launch.cu:36-70,
 *      src/cumpsgemm.cu:776-812) ------------------------------------------ */
unsigned cuMpSGEMM_get_current_dynamic_launch_buffer_id(cuMpSGEMM_handle_t handle);
unsigned cuMpSGEMM_get_next_dynamic_launch_buffer_id(cuMpSGEMM_handle_t handle);
int cuMpSGEMM_get_dynamic_launch_gemm_compute_mode(cuMpSGEMM_handle_t handle, unsigned buffer_id);
void cuMpSGEMM_get_dynamic_launch_scaling_mode_AB(cuMpSGEMM_handle_t handle, unsigned buffer_id,
                                                  int *scale_A, int *scale_B);
void cuMpSGEMM_set_dynamic_launch_buffer_by_exp_stats(cuMpSGEMM_handle_t handle,
                                                      unsigned dynamic_launch_buffer_id,
                                                      unsigned A_exp_stats_buffer_id,
                                                      unsigned B_exp_stats_buffer_id);
/* cumpsgemm::dynamic_launch::set_/unset_dynamic_launch_flag_buffer_id
 * (reference: src/dynamic_launch.cu:60-70): selects the flag slot a following
 * gemm(..., CUMPSGEMM_AUTO) call is gated by. */
void cuMpSGEMM_set_dynamic_launch_flag_buffer_id(cuMpSGEMM_handle_t handle, unsigned id);
void cuMpSGEMM_unset_dynamic_launch_flag_buffer_id(cuMpSGEMM_handle_t handle);

/* ---- timers (reference: src/cumpsgemm.cu:814-849) ------------------------ */
void cuMpSGEMM_enable_exp_stats_profiling(cuMpSGEMM_handle_t handle);
void cuMpSGEMM_disable_exp_stats_profiling(cuMpSGEMM_handle_t handle);
void cuMpSGEMM_reset_exp_stats_profiling(cuMpSGEMM_handle_t handle);
void cuMpSGEMM_print_exp_stats_profiling(cuMpSGEMM_handle_t handle, unsigned csv);
/* cumpsgemm::debug::get_exp_stats_profiling_result for one timer name; returns 0 when the
 * timer never ran. */
int cuMpSGEMM_get_exp_stats_profiling_result(cuMpSGEMM_handle_t handle, const char *name,
                                             double *time_sum_s, unsigned long long *n);

/* ---- gemm variants reporting the tile configuration used ----------------- */
/* cumpsgemm::gemm<T> / gemm_stridedBatch<T> with their used_kernel_module_id out-parameter
 * (reference: include/cumpsgemm/cumpsgemm.hpp:18-43). */
cublasStatus_t cuMpSGEMM_sgemm_module(
    cuMpSGEMM_handle_t handle, cublasOperation_t op_A, cublasOperation_t op_B, uint64_t m,
    uint64_t n, uint64_t k, const float *alpha, const float *a, uint64_t lda, const float *b,
    uint64_t ldb, const float *beta, float *c, uint64_t ldc, cuMpSGEMM_compute_mode_t mode,
    unsigned *used_kernel_module_id);

/* ---- kernel status -------------------------------------------------------- */
/* Every wait inside the GEMM kernel is bounded; a wait that gives up records a non-zero
 * code in a device word.  This call synchronises the handle's stream, returns the word and
 * clears it.  0 = no error; 1 = a producer / converter waited for a free stage, 2 = the MMA
 * issuer for operands, 3 / 7 = the MMA issuer for the drain of an accumulator, 4 / 5 = the
 * epilogue for an accumulator, 6 = bad launch, 8 = a role of the grouped products for its next tile.
 * The results of a call in which a wait gave up are not valid, nor are those of products of rows grouped by
 * expert that follow it on the handle before this call has cleared the word (they count with words that such
 * a kernel leaves behind, and that are set right here). */
int cuMpSGEMM_get_kernel_status(cuMpSGEMM_handle_t handle);
/* Which kernels the handle's last GEMM call launched, and in *cut_along_k (nullable) whether any of
 * its tiles was cut along K; host state only, nothing is synchronised.  CUMPSGEMM_ROUTE_NONE: no call
 * yet, or the last one was refused or failed. */
enum {
  CUMPSGEMM_ROUTE_NONE = 0,
  CUMPSGEMM_ROUTE_PRESPLIT_SINGLE = 1, /* split pass, then one CTA per tile */
  CUMPSGEMM_ROUTE_PRESPLIT_PAIR = 2,   /* split pass, then one CTA pair per tile */
  CUMPSGEMM_ROUTE_STREAMING = 3,       /* operands split between TMA and the tensor core; CTA pairs, or
                                        * single CTAs for batches of matrices with few rows */
  CUMPSGEMM_ROUTE_ON_THE_FLY = 4       /* single CTAs that load and split the operands themselves: the
                                        * kernel for small products, or the one that CUMPSGEMM_FUSED=1, or
                                        * a switch that keeps streaming off, selects */
};
int cuMpSGEMM_get_last_route(cuMpSGEMM_handle_t handle, int *cut_along_k);
/* Rows and columns of C (of the real, expanded product) in a tile of that call: 256 rows on CTA pairs, 128
 * on single CTAs; 0 x 0 without a route.  Returns 0, or 1 for a null argument. */
int cuMpSGEMM_get_last_tile(cuMpSGEMM_handle_t handle, int *rows, int *cols);
/* Self-test of the bounded wait: a one-CTA kernel waits, with the same routine the GEMM kernels
 * use, on a barrier that nothing signals; after limit_ms it must give up, record its code and
 * return normally.  Returns the status word (expected: 2, the "waited for operands" code) and
 * the time the wait took.  The context stays usable; nothing faults. */
int cuMpSGEMM_selftest_bounded_wait(cuMpSGEMM_handle_t handle, unsigned limit_ms,
                                    double *waited_ms);
/* Self-test of what follows a wait that gave up: the words that the products of rows grouped by expert
 * count tiles and slices with are zero between calls, and a kernel that gave up may leave them otherwise.
 * Returns how many of them are not zero; then, unless byte is 0, sets every byte of them to it and the
 * status word to 8, as such a kernel would.  No kernel runs; synchronises the handle's stream.
 * cuMpSGEMM_get_kernel_status has to bring them back to zero.  Negative: a CUDA error. */
int cuMpSGEMM_selftest_grouped_counters(cuMpSGEMM_handle_t handle, unsigned char byte);
/* The device the handle was created on; -1 without a handle. */
int cuMpSGEMM_get_device(cuMpSGEMM_handle_t handle);
/* Cap (bytes) for the workspace a call may use at once: the panels of a strided batch beyond it are
 * (with the sums of K slices, where the pre-split route cuts K) are processed in chunks of at least
 * one matrix, and sums of K pieces that would take a call beyond a limit it otherwise keeps are left
 * out (the tiles stay whole then).
 * 0 restores the default (8 GiB). */
void cuMpSGEMM_set_workspace_limit(cuMpSGEMM_handle_t handle, size_t bytes);
/* Compatibility switch for the exponent statistics (off by default; also set by the
 * environment variable CUMPSGEMM_COUNT_TAIL_PADDING=1 at handle creation).  The reference's
 * counting kernels walk a matrix four elements at a time and, when m*n is not a multiple of
 * 4, append zeros to the last group and count them like data
 * (reference: src/exp_stats.cu:101-116 and :222-238).  With the switch on, exp_stats_ext
 * adds the same (4 - m*n % 4) % 4 zero elements per matrix to `total` (and to `underflow`
 * when 0 is below the stage's threshold), so counts and decisions equal the reference's for
 * such shapes too; with it off only real matrix elements are counted. */
void cuMpSGEMM_set_count_tail_padding(cuMpSGEMM_handle_t handle, int enable);
/* A handle reads the tuning variables (CUMPSGEMM_TILE_N, CUMPSGEMM_PAIR, CUMPSGEMM_DRAIN_CHUNK,
 * CUMPSGEMM_FIRST_CHUNK, CUMPSGEMM_PACE, CUMPSGEMM_FUSED, CUMPSGEMM_SPLIT_K,
 * CUMPSGEMM_TAIL_SPLIT, CUMPSGEMM_STREAM) once, when it is created, so that a GEMM call does not
 * query the environment; this reads them again. */
void cuMpSGEMM_reload_tuning_env(cuMpSGEMM_handle_t handle);
/* Host-only query (no GPU needed): the K slices of the CTA-pair kernel's last, partly filled wave,
 * for `total_tiles` tiles of 256 x 256 with a K loop of k_pad values (a multiple of 64; tf32 != 0
 * for the TF32 kinds) on `clusters` CTA pairs.  Tiles [0, *split_begin) are not sliced; each later
 * tile is cut into *slices K slices of *slice_k values, *work_items work items in all.
 * *slices == 1: no tile is cut into slices of its own.  That includes a last wave that is more
 * than half full and is shared by all pairs in pieces of equal length, which this query cannot
 * express: cuMpSGEMM_plan_pair reports the whole plan.  Returns 0, or 1 for invalid arguments.  No
 * counterpart in the reference (its atomic split-K kernel, src/cumpsgemm.cu:272-304, is the nearest
 * relative). */
int cuMpSGEMM_plan_pair_tail(unsigned total_tiles, unsigned clusters, unsigned k_pad, int tf32,
                             unsigned *split_begin, unsigned *slices, unsigned *slice_k,
                             unsigned *work_items);
/* Host-only query (no GPU needed): how the CTA-pair kernel deals the same tiles.  *units is the K
 * loop in units of 64 values; tiles [0, *whole_tiles) run whole; the K loops of the others, laid end
 * to end (u units in all), are shared by *piece_clusters pairs (0: every tile is whole).
 * *slice_units > 0: every such tile is cut into *slices slices of that many units (the last may be
 * shorter), one pair each; *slice_units == 0: pair c takes units [c * u / p, (c + 1) * u / p) for
 * p = *piece_clusters.  A second kernel adds the pieces.  Returns 0, or 1 for invalid arguments. */
int cuMpSGEMM_plan_pair(unsigned total_tiles, unsigned clusters, unsigned k_pad, int tf32,
                        unsigned *units, unsigned *whole_tiles, unsigned *piece_clusters,
                        unsigned *slices, unsigned *slice_units);
/* Host-only query (no GPU needed): how the kernel that splits its operands between TMA and the
 * tensor core would deal an m x n x k x batch problem (sizes of the real, expanded problem) in
 * 256 x tile_n pair tiles (tile_n 256 or 128) to `clusters` CTA pairs.  *units is the K loop in
 * units of 64 values; tiles [0, *whole_tiles) of *total_tiles run whole; the k range of the
 * others, laid end to end, is shared by *piece_clusters pairs, pair c taking units
 * [c * u / p, (c + 1) * u / p) of the u units; *slices > 1: every tile is cut into that many and
 * a second kernel adds them.  Returns 0, or 1 for invalid arguments. */
int cuMpSGEMM_plan_stream(uint64_t m, uint64_t n, uint64_t k, uint64_t batch, int tile_n,
                          unsigned clusters, unsigned *total_tiles, unsigned *units,
                          unsigned *whole_tiles, unsigned *piece_clusters, unsigned *slices);
/* Per-launch device timing with CUDA events on the handle's stream (off by default).  While
 * enabled every split + GEMM launch group records three events; get_kernel_timing
 * synchronises the stream, returns the number of launch groups since the last query and the
 * summed durations of the split passes and of the GEMM kernels, and clears the record.
 * In AUTO mode both gated kinds are recorded, the deselected one with near-zero time. */
/* Optional stall breakdown of the GEMM kernels: eight 64-bit words in device memory that the
 * kernels add to (cycles the MMA issuer waited for operands [0] and for the accumulator drain
 * [1], the TMA producer for a free stage [2], one drain warp for a finished chunk [3], MMA
 * loop cycles [4], contributing CTAs [5]).  NULL (default) disables it. */
void cuMpSGEMM_set_debug_buffer(cuMpSGEMM_handle_t handle, unsigned long long *dev_words8);
void cuMpSGEMM_set_kernel_timing(cuMpSGEMM_handle_t handle, int enable);
unsigned long long cuMpSGEMM_get_kernel_timing(cuMpSGEMM_handle_t handle, double *split_ms,
                                               double *gemm_ms);

/* ---- interception-layer control (cumpsgemm::hijack_control, reference:
 *      src/cumpsgemm_cublas.cu:1189-1271) ---------------------------------- */
cuMpSGEMM_handle_t cuMpSGEMM_hijack_get_internal_global_handle(void);
/* returns 0, or 1 if the mode is rejected (CUMPSGEMM_FP32_SIMT; the C++ function throws) */
int cuMpSGEMM_hijack_set_compute_mode(int mode);
void cuMpSGEMM_hijack_unset_compute_mode(void);
void cuMpSGEMM_hijack_reset_exp_stats_buffer_id(void);
void cuMpSGEMM_hijack_set_exp_stats_params(float ignore_threshold, float underflow_threshold,
                                           float underflow_tolerance_rate);
void cuMpSGEMM_hijack_enable_restoring_AB_after_scaling(void);
void cuMpSGEMM_hijack_disable_restoring_AB_after_scaling(void);
/* copies at most size-1 characters and NUL-terminates; returns the full length */
size_t cuMpSGEMM_hijack_get_last_called_function_str(char *buf, size_t size);
void cuMpSGEMM_hijack_set_last_called_function_str(const char *str);
void cuMpSGEMM_hijack_clear_last_called_function_str(void);
void cuMpSGEMM_hijack_enable_custom_gemm_Mx2x2(void);
void cuMpSGEMM_hijack_disable_custom_gemm_Mx2x2(void);
int cuMpSGEMM_hijack_is_library_loaded(void);
/* C callback form of hijack_control::set_control_function; NULL unsets. */
typedef int (*cuMpSGEMM_control_function_c_t)(int op_A, int op_B, unsigned m, unsigned n,
                                              unsigned k);
void cuMpSGEMM_hijack_set_control_function(cuMpSGEMM_control_function_c_t fn);
/* The mode the rule chain would pick for a call (control function, then
 * libcumpsgemm_rule.so, then the built-in default).  Reference:
 * cuMpSGEMM_get_compute_mode_internal, src/cumpsgemm_cublas.cu:198-220. */
cuMpSGEMM_compute_mode_t cuMpSGEMM_get_compute_mode_internal(
    const char *const func_name, cublasHandle_t const cublas_handle,
    const cublasOperation_t op_A, const cublasOperation_t op_B, const unsigned m,
    const unsigned n, const unsigned k);

/* ---- multi-GPU support: staged statistics and a GEMM that takes decided
 *      statistics slots.  No counterpart in the reference. ------------------ */
/* Take the next statistics slot and zero it. */
unsigned cuMpSGEMM_exp_stats_begin(cuMpSGEMM_handle_t handle);
/* stage: 1 = max exponent + absolute-threshold counts, 2 = relative-threshold recount
 * (runs on the device only if decision 1 left the slot undecided),
 * 3 = max exponent only. */
void cuMpSGEMM_exp_stats_stage_s(cuMpSGEMM_handle_t handle, int stage, unsigned id, unsigned m,
                                 unsigned n, const float *ptr, unsigned ld, unsigned batch_size,
                                 unsigned stride);
void cuMpSGEMM_exp_stats_stage_c(cuMpSGEMM_handle_t handle, int stage, unsigned id, unsigned m,
                                 unsigned n, const cuComplex *ptr, unsigned ld,
                                 unsigned batch_size, unsigned stride);
/* decision: 1 or 2 (reference: src/exp_stats.cu:169-184, :277-293). */
void cuMpSGEMM_exp_stats_decide(cuMpSGEMM_handle_t handle, int decision, unsigned id);
/* Copy a slot to / from four 64-bit words in device memory:
 * {max exponent bits, total, underflow, mode}.  Ranks all-reduce words 0 (max) and
 * 1..2 (sum) between a stage and its decision. */
void cuMpSGEMM_exp_stats_export(cuMpSGEMM_handle_t handle, unsigned id,
                                unsigned long long *dev_words4);
void cuMpSGEMM_exp_stats_import(cuMpSGEMM_handle_t handle, unsigned id,
                                const unsigned long long *dev_words4);
/* Strided-batch GEMM whose scaling / kind selection comes from statistics slots that were
 * already decided (by the calls above).  mode is CUMPSGEMM_AUTO (flag slot derived from the
 * two statistics slots) or CUMPSGEMM_FP16TCEC_SCALING (both operands scaled). */
cublasStatus_t cuMpSGEMM_sgemm_strided_batch_with_stats(
    cuMpSGEMM_handle_t handle, cublasOperation_t op_A, cublasOperation_t op_B, uint64_t m,
    uint64_t n, uint64_t k, const float *alpha, const float *a, uint64_t lda, uint64_t stridea,
    const float *b, uint64_t ldb, uint64_t strideb, const float *beta, float *c, uint64_t ldc,
    uint64_t stridec, uint64_t batch_count, cuMpSGEMM_compute_mode_t mode, unsigned stats_id_a,
    unsigned stats_id_b);
cublasStatus_t cuMpSGEMM_cgemm_strided_batch_with_stats(
    cuMpSGEMM_handle_t handle, cublasOperation_t op_A, cublasOperation_t op_B, uint64_t m,
    uint64_t n, uint64_t k, const cuComplex *alpha, const cuComplex *a, uint64_t lda,
    uint64_t stridea, const cuComplex *b, uint64_t ldb, uint64_t strideb, const cuComplex *beta,
    cuComplex *c, uint64_t ldc, uint64_t stridec, uint64_t batch_count,
    cuMpSGEMM_compute_mode_t mode, unsigned stats_id_a, unsigned stats_id_b);

/* ---- two-by-two inner problems ------------------------------------------- */
/* C = alpha op(A) op(B) + beta C in plain FP32 for the shapes the reference hands to the
 * third-party cuGEMM-Mx2x2 kernels (src/cumpsgemm_cublas.cu:269-338, :647-725):
 *   *_Mx2x2: op(A) is m x 2, op(B) is 2 x 2, C is m x 2;
 *   *_2xNx2: op(A) is 2 x 2, op(B) is 2 x n, C is 2 x n;
 * m resp. n a power of two (anything else returns CUBLAS_STATUS_INVALID_VALUE).  Column-major
 * device pointers, host alpha / beta, leading dimensions and batch strides in elements;
 * batch_count == 1 with any strides is the single GEMM.  The interception layer takes this
 * route for such shapes when CUMPSGEMM_CUSTOM_GEMM_MX2X2=1 or after
 * hijack_control::enable_custom_gemm_Mx2x2(), whatever the compute mode, as the reference
 * does. */
cublasStatus_t cuMpSGEMM_sgemm_Mx2x2(cuMpSGEMM_handle_t handle, cublasOperation_t op_A,
                                     cublasOperation_t op_B, uint64_t m, const float *alpha,
                                     const float *a, uint64_t lda, uint64_t stridea,
                                     const float *b, uint64_t ldb, uint64_t strideb,
                                     const float *beta, float *c, uint64_t ldc, uint64_t stridec,
                                     uint64_t batch_count);
cublasStatus_t cuMpSGEMM_cgemm_Mx2x2(cuMpSGEMM_handle_t handle, cublasOperation_t op_A,
                                     cublasOperation_t op_B, uint64_t m, const cuComplex *alpha,
                                     const cuComplex *a, uint64_t lda, uint64_t stridea,
                                     const cuComplex *b, uint64_t ldb, uint64_t strideb,
                                     const cuComplex *beta, cuComplex *c, uint64_t ldc,
                                     uint64_t stridec, uint64_t batch_count);
cublasStatus_t cuMpSGEMM_sgemm_2xNx2(cuMpSGEMM_handle_t handle, cublasOperation_t op_A,
                                     cublasOperation_t op_B, uint64_t n, const float *alpha,
                                     const float *a, uint64_t lda, uint64_t stridea,
                                     const float *b, uint64_t ldb, uint64_t strideb,
                                     const float *beta, float *c, uint64_t ldc, uint64_t stridec,
                                     uint64_t batch_count);
cublasStatus_t cuMpSGEMM_cgemm_2xNx2(cuMpSGEMM_handle_t handle, cublasOperation_t op_A,
                                     cublasOperation_t op_B, uint64_t n, const cuComplex *alpha,
                                     const cuComplex *a, uint64_t lda, uint64_t stridea,
                                     const cuComplex *b, uint64_t ldb, uint64_t strideb,
                                     const cuComplex *beta, cuComplex *c, uint64_t ldc,
                                     uint64_t stridec, uint64_t batch_count);

/* ---- allocation-free FP32 GEMM ------------------------------------------- */
/* No counterpart in the reference.  For callers that may not allocate device memory (a
 * process whose memory budget is fixed at start-up, a loop that cannot take the device
 * synchronisation cudaMalloc / cudaFree imply, code without a handle): same arithmetic as
 * cuMpSGEMM_sgemm in FP16TCEC or TF32TCEC mode, but the split operand panels live in a 32 MiB
 * array built into the library instead of a workspace obtained with cudaMalloc, and no handle
 * is needed.  The call issues kernel launches on `stream` and nothing else.
 *   - Problems whose panels exceed 32 MiB return CUBLAS_STATUS_INVALID_VALUE with an error
 *     line and launch nothing.  FP16TCEC panels take 4*(round_up(m,tile_m)+round_up(n,tile_n))*
 *     round_up(k,64) bytes, TF32TCEC twice that, where tile_m x tile_n is the tile the library
 *     picks for the shape (256 x 256 with the CTA-pair kernel, else 128 x 256/128/64), or a
 *     narrower one where that does not fit: whatever has
 *     4*(round_up(m,128)+round_up(n,64))*round_up(k,64) <= 32 MiB is computed (FP16TCEC;
 *     m=n=k=2048 fits exactly).  A tile forced with CUMPSGEMM_TILE_N / CUMPSGEMM_PAIR is kept.
 *   - The first call on a device resolves the array's device address and configures the
 *     kernels; issue it before any stream capture on that device.
 *   - The array is shared by all calls on a GPU: calls that overlap in time on one GPU race.
 *     Each call rewrites all of the region it reads, so no clearing is needed between calls.
 *   - alpha / beta are host pointers; op C is rejected; no status word is kept (waits inside
 *     the kernel remain bounded). */
cublasStatus_t cuMpSGEMM_sgemm_static_scratch(
    cudaStream_t stream, cublasOperation_t op_A, cublasOperation_t op_B, uint64_t m, uint64_t n,
    uint64_t k, const float *alpha, const float *a, uint64_t lda, const float *b, uint64_t ldb,
    const float *beta, float *c, uint64_t ldc, cuMpSGEMM_compute_mode_t compute_mode);

/* ---- products of rows grouped by expert ---------------------------------- */
/* No counterpart in the reference.  The products of a mixture-of-experts layer: rows (tokens) sorted
 * by the group (expert) they belong to, and a weight matrix for each group.  Unlike the rest of this
 * interface, all matrices are ROW-MAJOR, as the frameworks that train and serve such models hold them;
 * ld* is the distance of rows and stride* of matrices, in elements.
 *   group_ends[num_groups], in device memory: the running total of rows after each group, so group e
 *     has the rows [group_ends[e - 1], group_ends[e]) of x, from 0 for the first.  It is read on the
 *     device: nothing waits for the sizes of the groups.  Groups may be empty.  A total below the one in
 *     front of it or above `rows` is taken as that.  NULL, with one group: all rows are of that group.
 *     Rows behind the last total belong to no group; what stands in them never counts.
 *   num_groups <= 1024; rows, n, k < 2^31.  rows may be 0.
 *   type: CUDA_R_16F or CUDA_R_16BF, summed in FP32 and rounded once, or CUDA_R_32F, which `mode`
 *     multiplies with error correction as the other calls do: CUMPSGEMM_FP16TCEC, or
 *     CUMPSGEMM_FP16TCEC_SCALING, which first brings the largest finite magnitude of each operand (of its
 *     rows in groups) to 2^14.  Other modes return CUBLAS_STATUS_NOT_SUPPORTED; 16-bit types do not look
 *     at it.  cuMpSGEMM_grouped_gemm multiplies FP32 operands with at most 6 rows for each group on average
 *     in plain FP32 arithmetic, which passes over a group's weights once for every 8 of its rows.
 *   Any leading dimension, stride and alignment.  FP32 operands, and 8- and 16-bit ones whose address,
 *     leading dimension or stride is not a multiple of 16 bytes, go through the handle's workspace
 *     (CUBLAS_STATUS_ALLOC_FAILED where it cannot hold them).
 *   Results are the same from run to run while the same calls have the same workspace: a call of few
 *     tiles adds up in slices of K where it can have memory for their sums, which is another order of FP32
 *     additions than without (under a workspace limit, or first made while the stream is being captured).
 *   Outputs must not overlap inputs. */

/* y[r, :] = alpha * x[r, :] op(w_e) + beta * y[r, :] for the rows r of each group e; rows of no group:
 * beta * y.  x is rows x k, y rows x n; w_e is stored k x n (op_W = CUBLAS_OP_N) or n x k (CUBLAS_OP_T).
 * The gradient of x is the same call with y's gradient as x, n and k exchanged and the other op_W.
 * beta == 0 does not read y. */
cublasStatus_t cuMpSGEMM_grouped_gemm(cuMpSGEMM_handle_t handle, cublasOperation_t op_W, uint64_t rows,
                                      uint64_t n, uint64_t k, uint32_t num_groups,
                                      const int32_t *group_ends, const float *alpha, const void *x,
                                      uint64_t ldx, const void *w, uint64_t ldw, uint64_t stridew,
                                      const float *beta, void *y, uint64_t ldy, cudaDataType_t type,
                                      cuMpSGEMM_compute_mode_t mode);
/* The gradient of the weights: dw_e = alpha * x_e^T dy_e + beta * dw_e over the rows of group e, stored
 * k x n (CUBLAS_OP_N) or n x k (CUBLAS_OP_T, the transpose).  Groups without rows: beta * dw_e. */
cublasStatus_t cuMpSGEMM_grouped_gemm_wgrad(cuMpSGEMM_handle_t handle, cublasOperation_t op_W,
                                            uint64_t rows, uint64_t n, uint64_t k, uint32_t num_groups,
                                            const int32_t *group_ends, const float *alpha, const void *x,
                                            uint64_t ldx, const void *dy, uint64_t lddy,
                                            const float *beta, void *dw, uint64_t lddw,
                                            uint64_t stridedw, cudaDataType_t type,
                                            cuMpSGEMM_compute_mode_t mode);
/* Product of 8-bit integers with a scale for each row of x (token) and each column of y (channel):
 *   y[r, c] = x_scale[r] * w_scale[e * n + c] * sum_i xq[r, i] wq_e[c, i] (+ bias[e * n + c])
 * for the rows r of each group e; rows of no group: 0.  wq_e is stored n x k.  The sums are exact
 * (k <= 131071), the scales are applied in FP32 and the result is rounded once to y_type (any of the
 * three).  bias may be NULL.  One group with group_ends = NULL is a plain quantised linear layer. */
cublasStatus_t cuMpSGEMM_i8_grouped_gemm(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t n, uint64_t k,
                                         uint32_t num_groups, const int32_t *group_ends,
                                         const int8_t *xq, uint64_t ldx, const float *x_scale,
                                         const int8_t *wq, uint64_t ldw, uint64_t stridew,
                                         const float *w_scale, const float *bias, void *y, uint64_t ldy,
                                         cudaDataType_t y_type);
/* Rows to 8 bits: with top the largest magnitude of a row, scale = top / 127 and
 * q[i] = rint(x[i] * (127 / top)), each step rounded to FP32, ties to even; a row of zeros, or
 * so small that its scale is 0 in FP32, has scale 0 and q = 0, a row with an infinity or NaN scale NaN and
 * q = 0 (its products are NaN).  Row r is taken from row row_index[r] of x (NULL: r); an index outside
 * [0, src_rows) gives a row of zeros.  type: that of x, any of the three. */
cublasStatus_t cuMpSGEMM_quantize_rows_i8(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t k,
                                          const void *x, uint64_t ldx, cudaDataType_t type,
                                          const int32_t *row_index, uint64_t src_rows, int8_t *q,
                                          uint64_t ldq, float *scale);

/* Gated feed-forward blocks: h = act(gate) * up, where gate and up are the halves of pre = x w^T; w_e is stored
 * 2 hidden x k, the rows of the gate first.  Sums, the activation and its derivative are FP32, and each result is
 * rounded once.  gelu is x (1 + erf(x / sqrt 2)) / 2, gelu_tanh its usual approximation by tanh. */
typedef enum {
  CUMPSGEMM_ACTIVATION_NONE = -1,
  CUMPSGEMM_ACTIVATION_SILU = 0,
  CUMPSGEMM_ACTIVATION_GELU = 1,
  CUMPSGEMM_ACTIVATION_GELU_TANH = 2,
  CUMPSGEMM_ACTIVATION_RELU = 3
} cuMpSGEMM_activation_t;
/* y[r, :] = act(x[r] gate_e^T) * (x[r] up_e^T) for the rows r of each group e; rows of no group: 0.  x is rows x k,
 * y rows x hidden; pre (rows x 2 hidden), if not NULL, receives the rounded products, which the backward pass
 * needs.  FP32 needs it in any case.  y comes of unrounded products. */
cublasStatus_t cuMpSGEMM_grouped_gemm_gated(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t hidden,
                                            uint64_t k, uint32_t num_groups, const int32_t *group_ends,
                                            const void *x, uint64_t ldx, const void *w, uint64_t ldw,
                                            uint64_t stridew, cuMpSGEMM_activation_t activation, void *y,
                                            uint64_t ldy, void *pre, uint64_t ldpre, cudaDataType_t type,
                                            cuMpSGEMM_compute_mode_t mode);
/* Backwards through the product behind it as well: with dh = dy op(w_e) (dy rows x k, w_e stored k x hidden,
 * CUBLAS_OP_N, or hidden x k, CUBLAS_OP_T), dpre = [dh * up * act'(gate), dh * act(gate)].  pre: as the call above
 * left it.  Rows of no group: 0.  An infinity in a float16 pre stands for a sum past 65504: times a dh or a slope of 0,
 * or in a gate far below 0, it counts for nothing. */
cublasStatus_t cuMpSGEMM_grouped_gemm_gated_grad(cuMpSGEMM_handle_t handle, cublasOperation_t op_W,
                                                 uint64_t rows, uint64_t hidden, uint64_t k,
                                                 uint32_t num_groups, const int32_t *group_ends,
                                                 const void *dy, uint64_t lddy, const void *w, uint64_t ldw,
                                                 uint64_t stridew, cuMpSGEMM_activation_t activation,
                                                 const void *pre, uint64_t ldpre, void *dpre, uint64_t lddpre,
                                                 cudaDataType_t type, cuMpSGEMM_compute_mode_t mode);
/* The elementwise passes by themselves: out = act(gate) * up (rows x hidden), or where dh (rows x hidden) is not
 * NULL, out = dpre (rows x 2 hidden) as above. */
cublasStatus_t cuMpSGEMM_gated_rows(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t hidden,
                                    const void *pre, uint64_t ldpre, const void *dh, uint64_t lddh,
                                    cuMpSGEMM_activation_t activation, void *out, uint64_t ldo,
                                    cudaDataType_t type);

/* 8-bit floating point (CUDA_R_8F_E4M3, CUDA_R_8F_E5M2) with a scale for each block of 128 columns of a row, or of
 * 128 x 128 of a matrix; the last blocks may be smaller.  With top the largest magnitude in a block and M the type's
 * largest value (448, 57344), scale = top / M and q[i] is the value nearest to x[i] M / top (product and quotient
 * rounded to FP32).  A block of zeros, or so small that its scale is 0 in FP32, has scale 0 and q = 0, one with an
 * infinity or NaN scale NaN and q = 0 (its products are NaN).
 *   Scales of rows lie at scale[row * scale_row + block * scale_block], those of weights one behind the other:
 *   [matrix][block of n][block of k]. */
/* Row r is taken from row row_index[r] of x (NULL: r); an index outside [0, src_rows) gives a row of zeros.  With an
 * activation, x has rows of 2 k, and act(gate) * up of their halves, in FP32, is what is brought to 8 bits. */
cublasStatus_t cuMpSGEMM_quantize_rows_f8(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t k, const void *x,
                                          uint64_t ldx, cudaDataType_t type, const int32_t *row_index,
                                          uint64_t src_rows, int activation, void *q, uint64_t ldq,
                                          cudaDataType_t q_type, float *scale, uint64_t scale_row,
                                          uint64_t scale_block);
cublasStatus_t cuMpSGEMM_quantize_blocks_f8(cuMpSGEMM_handle_t handle, uint32_t matrices, uint64_t n, uint64_t k,
                                            const void *w, uint64_t ldw, uint64_t stridew, cudaDataType_t type,
                                            void *q, uint64_t ldq, uint64_t strideq, cudaDataType_t q_type,
                                            float *scale);
/* y[r, c] = sum over blocks b of k of x_scale[r, b] w_scale[e, c / 128, b] sum_{i in b} xq[r, i] wq_e[c, i]
 * (+ bias[e * n + c]) for the rows r of each group e; rows of no group: 0.  wq_e is stored n x k; bias may be NULL.
 * The products of a block are added in FP32 by the tensor core, the blocks in FP32, and the result is rounded once to y_type.
 * The two scales of a block are multiplied first, in FP32, whose range their product has to keep. */
cublasStatus_t cuMpSGEMM_f8_grouped_gemm(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t n, uint64_t k,
                                         uint32_t num_groups, const int32_t *group_ends, const void *xq,
                                         uint64_t ldx, cudaDataType_t x_type, const float *x_scale,
                                         uint64_t x_scale_row, uint64_t x_scale_block, const void *wq,
                                         uint64_t ldw, uint64_t stridew, cudaDataType_t w_type,
                                         const float *w_scale, const float *bias, void *y, uint64_t ldy,
                                         cudaDataType_t y_type);
/* The gated product with such operands, act(x gate_e^T) * (x up_e^T) of unrounded FP32 products, brought to 8 bits
 * again: q (rows x hidden) and its scales.  wq_e is stored 2 hidden x k; hidden is a multiple of 128.  For few rows
 * (those of 32 for each group, or some more) the FP32 products go by way of the handle's workspace where it can have
 * them, and cuMpSGEMM_quantize_rows_f8's rule brings them to 8 bits.  Otherwise each value is multiplied by M / top, rounded to
 * FP32: q may be the 8-bit value next to the nearest one where a value lies near the middle between the two.  So the two
 * ways, one of which depends on the workspace, may differ by one step of the 8-bit type, and as the order of FP32 sums does. */
cublasStatus_t cuMpSGEMM_f8_grouped_gemm_gated(cuMpSGEMM_handle_t handle, uint64_t rows, uint64_t hidden,
                                               uint64_t k, uint32_t num_groups, const int32_t *group_ends,
                                               const void *xq, uint64_t ldx, cudaDataType_t x_type,
                                               const float *x_scale, uint64_t x_scale_row,
                                               uint64_t x_scale_block, const void *wq, uint64_t ldw,
                                               uint64_t stridew, cudaDataType_t w_type, const float *w_scale,
                                               cuMpSGEMM_activation_t activation, void *q, uint64_t ldq,
                                               cudaDataType_t q_type, float *scale, uint64_t scale_row,
                                               uint64_t scale_block);

#ifdef __cplusplus
}
#endif
#endif
