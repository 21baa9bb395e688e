/*
 * mmaemu_b200 -- C ABI of the B200 (sm_100a) backend for the mmaemu.scaled_mm hot path.
 *
 * Every function is a host function of libmmaemu_b200.so. Pointers named *_dev are device pointers owned by the
 * caller; nothing is allocated internally unless a function says so. All launches are asynchronous on the given
 * cudaStream_t (passed as void*; NULL = the legacy default stream). Functions return MMB200_OK (0) or a negative
 * status, never throw and never abort. Mutable state of the library: per-device function attributes that are set once;
 * the per-device memory pool, internal streams and events of mmb200_scaled_mm_host; the fixed scratch array of mmb200_scaled_mm_static with its
 * cached per-device address; the launch counter; the process-wide test hooks of mmb200_test_hooks; the per-device status
 * words of the int8 kernels (mmb200_int8_status).
 *
 * Operands are FP8 code bytes: A is [M, K] row-major with leading dimension lda (bytes), B is [N, K] row-major with
 * leading dimension ldb -- that is mat2.t() of torch._scaled_mm's column-major [K, N] operand.
 *
 * What each entry point replaces in the reference (astding/mmaemu, paths relative to its root):
 *   mmb200_chain       the kernel ABI v1 entry points mmaemu_{h4,h1,v4,v1}_e4m3e4m3 (mmaemu/backends/cuda/spec.py:3-16)
 *                      together with their launch wrapper chain_fn_for (mmaemu/backends/cuda/kernels.py:85-134);
 *   mmb200_scaled_mm   the compute lines of _scaled_mm_impl (mmaemu/api.py:342-346): execute_plan
 *                      (mmaemu/model/plan.py:169-208: sanitise, per-chunk gathers and launches, slow-accumulation and
 *                      split-K combination, non-finite patch) and epilogue.apply (mmaemu/model/epilogue.py:65-78),
 *                      fused into one launch;
 *   mmb200_accumulate  execute_plan alone, as mmaemu.accumulate uses it (mmaemu/api.py:382-421);
 *   mmb200_scaled_mm_host   the same call for callers that hold host memory (no reference counterpart below the
 *                      Python level: the reference moves tensors with torch).
 */
#ifndef MMAEMU_B200_H
#define MMAEMU_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MMB200_ABI_VERSION 6

/* status codes */
#define MMB200_OK 0
#define MMB200_ERR_BAD_ARG (-1)       /* NULL pointer, negative size, unknown enum, ld < K, misaligned operand */
#define MMB200_ERR_UNSUPPORTED (-2)   /* valid request this build has no kernel for */
#define MMB200_ERR_ARCH (-3)          /* the current device is not sm_100 (the fatbin holds sm_100a code only) */
#define MMB200_ERR_LAUNCH (-4)        /* the CUDA runtime refused the launch or a copy (see mmb200_last_cuda_error) */
#define MMB200_ERR_TOO_LARGE (-5)     /* a size is beyond a documented limit */
#define MMB200_ERR_TIMEOUT (-6)       /* a bounded wait inside a kernel ran out; the output was not written */

/* FP8 operand formats (mmaemu/formats.py:14-19) */
#define MMB200_FMT_E4M3 0
#define MMB200_FMT_E5M2 1

/* output dtypes, numbered like the reference's split-K tables (mmaemu/platform/splitk_table.py OUT_CODES) */
#define MMB200_OUT_F32 0
#define MMB200_OUT_BF16 1
#define MMB200_OUT_F16 2
#define MMB200_OUT_E4M3 3
#define MMB200_OUT_E5M2 4

/* split-K reduction schemes (mmaemu/model/plan.py:46) */
#define MMB200_SCHEME_NONE 0
#define MMB200_SCHEME_SERIAL 1
#define MMB200_SCHEME_PAIRWISE 2
#define MMB200_SCHEME_CONTIGUOUS 3

/* kernel families */
#define MMB200_KERNEL_AUTO 0     /* the fastest kernel that serves the request */
#define MMB200_KERNEL_INTEGER 1  /* pure-integer block model: every format pair and plan */
#define MMB200_KERNEL_FAST 2     /* tensor-core kernels with scratch memory, fp32 round-toward-zero FMA chain without */

/* The `nfma` argument of every entry point names the instruction preset (mmaemu/model/presets.py:68-85): 16 = ada and
 * 32 = hopper are the products per block of the two early-accumulator presets (13 fraction bits, every plan); 288 is
 * b200_mma_sync, 32 products per block aligned on the largest product exponent with 25 fraction bits, the block sum
 * cut to 24 significant bits and added to the accumulator in fp32. The reference characterises no GEMM level for it
 * (plan.py:98-102), so it is served for unsplit fast accumulation only (fast != 0, S == 1; MMB200_ERR_UNSUPPORTED
 * otherwise) and by the integer kernel only. */
#define MMB200_PRESET_ADA 16
#define MMB200_PRESET_HOPPER 32
#define MMB200_PRESET_B200_MMA_SYNC 288

#define MMB200_MAX_SPLITS 64
#define MMB200_MAX_PEERS 15      /* other GPUs that can receive a copy of the output (mmb200_scaled_mm_peers) */

int mmb200_abi_version(void);
const char *mmb200_status_string(int status);
/* Text of the last CUDA runtime error seen by this thread inside the library ("" if none). */
const char *mmb200_last_cuda_error(void);
/* MMB200_OK if `device` can run the kernels, MMB200_ERR_ARCH otherwise. Does not change the current device. */
int mmb200_device_supported(int device);

/* C[m][n] = chain over k = 0..K-1 of A[m][k] * B[n][k] from +0 under the preset with `nfma` products per block
 * (16 = ada, 32 = hopper, 288 = b200_mma_sync); fp32 result, ldc in floats. Non-finite codes count as +0 (the caller sanitises, as
 * execute_plan does). K need not be a multiple of nfma (the tail is zero padded). */
int mmb200_chain(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b, float *C_dev,
                 int64_t ldc, int M, int N, int K, int nfma, int kernel, void *stream);

/* fp32 accumulator before alpha under the plan (nfma, fast, S, scheme), with the IEEE non-finite patch and canonical
 * NaN. S = 1 ignores the scheme. */
int mmb200_accumulate(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b,
                      float *C_dev, int64_t ldc, int M, int N, int K, int nfma, int fast, int S, int scheme,
                      int kernel, void *stream);

/* The whole call: plan, combination, non-finite patch, then alpha = RN32(scale_a * scale_b),
 * y = RN32(fma(acc, alpha, +0)), conversion to out_dtype (fp8 outputs: optional scale_result multiply, saturation),
 * canonical NaN. D is [M, N] row-major of out_dtype with leading dimension ldd (elements). The three scales are
 * device pointers to one fp32 each (scale_result_dev may be NULL); they are read by the kernel, never by the host. */
int mmb200_scaled_mm(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b, void *D_dev,
                     int64_t ldd, int out_dtype, int M, int N, int K, int nfma, int fast, int S, int scheme,
                     const float *scale_a_dev, const float *scale_b_dev, const float *scale_result_dev, int kernel,
                     void *stream);

/* Same computation for HOST operands and a HOST result: copies A and B to the current device, runs the kernel, copies
 * D back and waits for it. Device staging memory, including the scratch memory of the staged kernels, comes from a
 * stream-ordered memory pool of the library (cudaMallocFromPoolAsync; the pool keeps freed memory for the next call) and
 * is returned to it before the call returns. Host buffers should be pinned for full copy speed but need not be.
 * Calls that move 8 MiB or more and have at least two slabs of about 128 output tiles are pipelined: B is copied and
 * decoded once, the rows of A are cut into at most 8 slabs (multiples of 128 rows), each on an internal stream of its
 * own (copy of its rows, its kernels, copy-back of its outputs), so that the copies of some slabs overlap the kernels
 * of others; the caller's stream waits for all of it. Rows are independent of one another
 * and the plan is that of the whole call, so the result is the same bits. One pipelined call at a time per device
 * (others wait on a mutex); MMAEMU_B200_HOST_PIPELINE=0 in the environment turns the slabs off. When a bounded wait
 * inside a kernel runs out the call returns MMB200_ERR_TIMEOUT; D is then not written by an unpipelined call and
 * unspecified after a pipelined one (finished slabs have been copied back). */
int mmb200_scaled_mm_host(const void *A_host, int64_t lda, int fmt_a, const void *B_host, int64_t ldb, int fmt_b,
                          void *D_host, int64_t ldd, int out_dtype, int M, int N, int K, int nfma, int fast, int S,
                          int scheme, float scale_a, float scale_b, const float *scale_result /* host, nullable */,
                          int kernel, void *stream);

/* Scratch memory. The fastest path decodes both operands once into device scratch memory (4 bytes per element, rounded up
 * to 128 x 32 tiles; 10 per element of A and 8 of B while $MMAEMU_B200_TC_EPASS is 0) and streams the decoded tiles into shared memory with bulk
 * asynchronous copies. mmb200_workspace_bytes gives the size for a shape; the *_ws entry points take the memory from
 * the caller (128-byte aligned, at least that size, used only until the call's work on the stream has finished) and
 * are otherwise identical to mmb200_scaled_mm / mmb200_accumulate. 0 means that no scratch-memory kernel takes the shape
 * (an empty one, or more than 65,535 tiles of 128 rows or columns). With workspace_dev == NULL, a workspace that is too
 * small, or a request the fast kernels do not serve, they behave exactly like the entry points without workspace.
 * The reference has no counterpart: its kernels decode inside the main loop (mmaemu/backends/cuda/csrc/h4.cu:190-211). */
size_t mmb200_workspace_bytes(int M, int N, int K);
/* The same for a split-K plan with S splits (S = 1: as above). With that much scratch the staged fast kernels also walk
 * split plans: they consume the k-tiles in the plan's order and keep the running total and the pair slot of the split
 * reduction in the scratch memory (8 more bytes per output, rounded up to 128 x 128 tiles, plus the tile order). With
 * less, split plans run on the integer kernel as they do without workspace. For shapes with few 128 x 128 output tiles the
 * size also covers the chain results of K-sliced execution (plans with several chains are spread over the SMs along K and
 * summed in the plan's order by a second kernel; up to 4 GiB, not used when the workspace is smaller or when
 * $MMAEMU_B200_SLICES is 0). Calls with at most 16 rows, and calls whose 128 x 128 output tiles and chains would leave
 * most SMs without a CTA, run on kernels that work on 16 rows per CTA and decode both operands themselves (no
 * pre-decode launches; $MMAEMU_B200_ROW_GROUPS=0 keeps them to calls of at most 16 rows). Same results bit for bit
 * either way. */
size_t mmb200_workspace_bytes_split(int M, int N, int K, int S);
int mmb200_scaled_mm_ws(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b,
                        void *D_dev, int64_t ldd, int out_dtype, int M, int N, int K, int nfma, int fast, int S,
                        int scheme, const float *scale_a_dev, const float *scale_b_dev, const float *scale_result_dev,
                        int kernel, void *workspace_dev, size_t workspace_bytes, void *stream);
int mmb200_accumulate_ws(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b,
                         float *C_dev, int64_t ldc, int M, int N, int K, int nfma, int fast, int S, int scheme,
                         int kernel, void *workspace_dev, size_t workspace_bytes, void *stream);

/* Multi-GPU assembly fused into the kernel. Large calls are split by output rows (or by any output rectangle: pass the
 * operand and output pointers of the rectangle's first element with the full leading dimensions) across the GPUs of one
 * machine, K is never split across GPUs, and every GPU needs the whole result. Instead of an all-gather after the
 * kernel, mmb200_scaled_mm_peers stores every output element of this GPU's rectangle into D_dev and, at the same
 * index, into each of the n_peers buffers peer_D[i]: device pointers, valid in this process, to the same rectangle of
 * the other GPUs' result buffers (peer-mapped memory, e.g. symmetric memory or CUDA IPC; plain stores over NVLink, no
 * multicast, no loads from peer memory). The caller orders the kernels on all GPUs against the readers with its own
 * barrier after the call (and before it, if the buffers are being reused). n_peers = 0 is mmb200_scaled_mm_ws.
 * `peer_D` is a HOST array of n_peers device pointers (read during the call). The reference has no multi-GPU path
 * (docs/limitations.md:100 of astding/mmaemu). */
int mmb200_scaled_mm_peers(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b,
                           void *D_dev, int64_t ldd, int out_dtype, int M, int N, int K, int nfma, int fast, int S,
                           int scheme, const float *scale_a_dev, const float *scale_b_dev,
                           const float *scale_result_dev, int kernel, void *workspace_dev, size_t workspace_bytes,
                           void *const *peer_D, int n_peers, void *stream);

/* Bounded waits and their status word. The scratch-memory kernels wait for their bulk copies on mbarriers with a bound
 * (about four seconds); a wait that runs out makes the kernel record 1 in a status word inside the scratch memory, skip
 * the output (D keeps its previous contents) and return, instead of spinning forever. Launches are asynchronous, so the
 * word is read after the stream has drained: mmb200_workspace_status synchronises `stream`, reads the word of the call
 * that last used `workspace_dev` with this shape and split count, and returns MMB200_OK or MMB200_ERR_TIMEOUT;
 * mmb200_workspace_status_offset gives the byte offset of the int32 word for callers that read it themselves
 * (mmb200_scaled_mm_host checks it before copying D back and returns MMB200_ERR_TIMEOUT). The reference has no
 * counterpart: its kernels hold no waits (mmaemu/backends/cuda/csrc/h4.cu:289-303 synchronises with barriers only). */
size_t mmb200_workspace_status_offset(int M, int N, int K, int S);
int mmb200_workspace_status(const void *workspace_dev, int M, int N, int K, int S, void *stream);
/* The same for the fixed scratch array of mmb200_scaled_mm_static on the current device. */
int mmb200_scaled_mm_static_status(int M, int N, int K, void *stream);
/* Test hook, process-wide: every later scratch-memory launch bounds its waits by `wait_polls` polls (<= 0: the
 * default) and announces `announce_extra_bytes` more bytes per stage to the mbarrier than it copies (<= 0: none), so
 * that the wait runs out without anything faulting. For the tests of the status word only. */
void mmb200_test_hooks(int wait_polls, int announce_extra_bytes);

/* Quantise prologue fused into the staged path: the activations X [M, K] (MMB200_HP_F32 or MMB200_HP_BF16, row stride
 * ldx elements, 16-byte aligned rows) are multiplied by *quant_scale_dev, clamped to +-448 and rounded to E4M3 (nearest
 * even; for bf16 activations the scale and the product are first rounded to bf16, as torch's type promotion has it) -- bit for bit torch's
 * (x * scale).clamp(-448, 448).to(torch.float8_e4m3fn) on a CUDA device (NaN gives 0x7F) -- inside the pass that
 * decodes operand A, so the codes are never read back from memory before the GEMM. The codes are also written to
 * A_codes_dev [M, K] (row stride lda, a multiple of 16; 16-byte aligned) for the caller to keep. Everything after that
 * is mmb200_scaled_mm_ws with fmt_a = E4M3. Needs the scratch memory (mmb200_workspace_bytes_split) and K a positive
 * multiple of 16: otherwise MMB200_ERR_UNSUPPORTED and nothing is written. With M or N zero nothing is written either.
 * Replaces the separate quantisation pass of the reference's FP8 examples (examples/evo2_offload.py:124-129), which
 * runs as torch operations before mmaemu.scaled_mm; the reference has no fused counterpart. */
#define MMB200_HP_F32 1
#define MMB200_HP_BF16 2
#define MMB200_HP_F16 3          /* the int8 entry points only */
int mmb200_quantize_scaled_mm_ws(const void *X_dev, int64_t ldx, int x_dtype, const float *quant_scale_dev,
                                 void *A_codes_dev, int64_t lda, const void *B_dev, int64_t ldb, int fmt_b,
                                 void *D_dev, int64_t ldd, int out_dtype, int M, int N, int K, int nfma, int fast, int S,
                                 int scheme, const float *scale_a_dev, const float *scale_b_dev,
                                 const float *scale_result_dev, void *workspace_dev, size_t workspace_bytes,
                                 void *stream);

/* The scratch-memory path for callers that cannot allocate device memory and have none to lend: the scratch is a
 * fixed array inside the library's device image, so the call performs no allocation of any kind. It serves what
 * mmb200_scaled_mm_ws serves with its fast kernel (unsplit plan, K a multiple of 16, 16-byte aligned operands and
 * leading dimensions; anything else returns MMB200_ERR_UNSUPPORTED) for shapes whose mmb200_workspace_bytes is at most
 * MMB200_STATIC_SCRATCH_BYTES (larger ones return MMB200_ERR_TOO_LARGE). All calls on a device share the array: calls
 * that overlap on the GPU race. The first call on a device looks up the array's address and should come before any
 * stream capture. It has no counterpart in the reference, which allocates its outputs with torch. */
#define MMB200_STATIC_SCRATCH_BYTES (64u << 20)
int mmb200_scaled_mm_static(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb, int fmt_b,
                            void *D_dev, int64_t ldd, int out_dtype, int M, int N, int K, int nfma, int fast,
                            const float *scale_a_dev, const float *scale_b_dev, const float *scale_result_dev,
                            void *stream);

/* Which kernel family a request with these operands and this plan runs on WITHOUT scratch memory when `kernel` is
 * MMB200_KERNEL_AUTO: MMB200_KERNEL_FAST (16-byte aligned operands, leading dimensions and K that are multiples of 16, an
 * unsplit plan) or MMB200_KERNEL_INTEGER. With scratch memory of mmb200_workspace_bytes_split the *_ws entry points run every
 * plan and any operands on the fast kernels too, except split plans of such other operands that leave a split without k-tiles;
 * a request for MMB200_KERNEL_FAST by name, the quantise prologue, mmb200_scaled_mm_static and mmb200_scaled_mm_host keep
 * to 16-byte operands (the last to K a multiple of 16). Pure host logic: no CUDA call, nothing is dereferenced. It has no
 * counterpart in the reference, whose kernels each serve one format pair and one preset (mmaemu/backends/registry.py). */
int mmb200_kernel_for(const void *A_dev, int64_t lda, const void *B_dev, int64_t ldb, int K, int nfma, int S);

/* ---- Ragged groups: rows [m_0 + .. + m_{e-1}, + m_e) of A are multiplied with the weights of group e.
 *
 * mmb200_grouped_scaled_mm is mmb200_scaled_mm_ws for every group: group e has m_splits[e] rows of A and D, the operand
 * B + e * group_stride_b, the scales scale_a_dev[e * sa_stride] and scale_b_dev[e * sb_stride] (stride 0: one scale for all
 * groups) and the split decision splits[e], schemes[e] (NULL: no group is split). The result has the bits of a loop of
 * mmb200_scaled_mm_ws calls, whatever kernel runs. m_splits, splits and schemes are HOST arrays of E entries, read during
 * the call (the split decision of the emulated platform depends on a group's rows). With scratch memory the unsplit groups
 * run in one pass of launches (up to 8 GiB of decoded operands), the others one after the other. Scratch memory as there:
 * mmb200_grouped_workspace_bytes, or, where that much is not to be had, mmb200_grouped_workspace_bytes_one_by_one, with which
 * every group runs by itself on the scratch-memory kernels. mmb200_grouped_status synchronises `stream` and reports whether a
 * bounded wait of the call that last used the memory ran out (outputs of the groups whose waits ran out then keep their
 * previous contents, all others are written). The reference has no grouped call. */
#define MMB200_MAX_GROUPS 4096
size_t mmb200_grouped_workspace_bytes(const int *m_splits, const int *splits, int E, int N, int K, int fmt_a, int fmt_b,
                                      int nfma, int fast);
size_t mmb200_grouped_workspace_bytes_one_by_one(const int *m_splits, const int *splits, int E, int N, int K);
int mmb200_grouped_scaled_mm(const void *A_dev, int64_t lda, int fmt_a, const void *B_dev, int64_t ldb,
                             int64_t group_stride_b, int fmt_b, void *D_dev, int64_t ldd, int out_dtype,
                             const int *m_splits, const int *splits, const int *schemes, int E, int N, int K, int nfma,
                             int fast, const float *scale_a_dev, int64_t sa_stride, const float *scale_b_dev,
                             int64_t sb_stride, const float *scale_result_dev, int kernel, void *workspace_dev, size_t workspace_bytes,
                             void *stream);
int mmb200_grouped_status(const void *workspace_dev, void *stream);

/* ---- int8. Integer tensor-core sums are exact on every GPU, so these calls emulate no platform.
 *
 * mmb200_quantize_int8: per row of X [rows, K] (x_dtype MMB200_HP_*, row stride ldx elements) scale = RN32(amax / 127) and
 * the codes [rows, K] (row stride ldc): the integer nearest to 127 x / amax, ties to even, decided exactly. A zero row has
 * scale 0; a row with a NaN or an infinity has scale NaN and codes 0. */
int mmb200_quantize_int8(const void *X_dev, int64_t ldx, int x_dtype, int8_t *codes_dev, int64_t ldc, float *scale_dev,
                         int64_t rows, int K, void *stream);

/* D[r][n] = out(fma(RN32(acc), RN32(sa sb), bias)), acc = sum_k A[r][k] W[g][n][k] (exact; K <= MMB200_INT8_MAX_K,
 * T <= MMB200_INT8_MAX_ROWS, N <= MMB200_INT8_MAX_N), rounded
 * to fp32 and then to out_dtype (F32, BF16 or F16; canonical NaN). A is [T, K] int8 with row stride lda, W [E, N, K] with row
 * stride ldw and group stride group_stride_w. sa = scale_a_dev[r * sa_stride], sb = scale_b_dev[g * sb_group_stride +
 * n * sb_stride], bias = bias_dev[g * bias_group_stride + n] of bias_dtype (MMB200_HP_*; bias_dev NULL: none).
 * offs_dev NULL: one group (E = 1) of all T rows. Else offs_dev[g] (device, int32) is the end of group g's rows; ends are
 * taken as a running maximum and clamped to [0, T], so no value leads out of the operands. Rows behind the last group are
 * set to zero (zero_rest != 0) or left as they are. Operands whose rows do not start on 16 bytes are copied into scratch
 * memory of mmb200_int8_workspace_bytes first (16-byte aligned; 0 bytes: none needed). */
#define MMB200_INT8_MAX_K 131071
#define MMB200_INT8_MAX_ROWS (1 << 23)
#define MMB200_INT8_MAX_N (1 << 30)
size_t mmb200_int8_workspace_bytes(const int8_t *A_dev, int64_t lda, const int8_t *W_dev, int64_t ldw,
                                   int64_t group_stride_w, int T, int N, int K, int E);
/* (25 fields of 64 bits, so that a binding can pack them in one go) */
typedef struct mmb200_int8_args {
  const int8_t *A_dev;
  int64_t lda;
  const int8_t *W_dev;
  int64_t ldw, group_stride_w;
  void *D_dev;
  int64_t ldd, out_dtype, T, N, K, E;
  const int *offs_dev;
  const float *scale_a_dev;
  int64_t sa_stride;
  const float *scale_b_dev;
  int64_t sb_group_stride, sb_stride;
  const void *bias_dev;
  int64_t bias_dtype, bias_group_stride, zero_rest;
  void *workspace_dev;
  uint64_t workspace_bytes;
  void *stream;
} mmb200_int8_args;
int mmb200_int8_scaled_mm(const mmb200_int8_args *args);
/* The kernel that a call of this shape runs on: kind << 16 | rows of a tile << 4 | parts of K, kind 0: one tile per CTA (a
 * cluster of `parts` CTAs shares a tile), 1: persistent CTAs, 2: persistent pairs of CTAs. ragged: whether offs_dev is given.
 * Pure host logic (148 SMs are assumed where no device answers). */
int mmb200_int8_kernel_for(int T, int N, int K, int E, int ragged);
/* Synchronises `stream`: MMB200_ERR_TIMEOUT when a bounded wait of an int8 kernel has run out on the current device since the
 * last such call, else MMB200_OK. One word for the calls of all streams and threads: it does not say whose outputs are unspecified.
 * With MMAEMU_B200_CHECK_STATUS=1 in the environment mmb200_int8_scaled_mm counts on a word of its own instead, synchronises its
 * stream and returns MMB200_ERR_TIMEOUT itself (up to 64 such calls at once on a device; the next one waits for one of them). */
int mmb200_int8_status(void *stream);

/* Issue-rate probe for roofline denominators: launches `ctas` blocks of 256 threads in which every thread executes
 * iters x 32 independent instructions of one kind (kind 0: fma.rz.f32; kind 1: three-input integer add and three-input
 * logic operation alternating) and stores one float per thread to sink_dev (ctas * 256 floats). The caller times the
 * launch; lane-instructions = ctas * 256 * iters * 32. Not counted by mmb200_launch_count. The reference measures its
 * kernels' rates with a host script instead (tools/bench_kernels.py:271-350 of astding/mmaemu). */
int mmb200_probe_issue_rate(int kind, int ctas, int iters, float *sink_dev, void *stream);

/* Number of kernel launches the library has issued in this process (all threads), for launch accounting. */
int64_t mmb200_launch_count(void);

#ifdef __cplusplus
}
#endif
#endif /* MMAEMU_B200_H */
