// Launch parameters of the int8 operators (kernel_quantise.cu, kernel_int8.cu) and their launchers; no part of common.cuh,
// which the emulated kernels share.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mmb {

#if defined(__CUDACC__)
// Programmatic dependent launch: these kernels start while the previous one of the stream is still running, set up barriers and
// TMEM, and wait here, before their first access to memory, until it has completed. Every thread waits, so a kernel is never
// complete before its predecessors are. The next kernel may start as soon as every CTA of this one has.
__device__ __forceinline__ void wait_for_predecessor() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// Launch with that attribute; `cluster`: CTAs per cluster (0: the kernel's own).
template <class... P, class... A>
cudaError_t launch_dependent(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}
#endif

struct QuantiseParams {
  const void* x;          // [rows, K], row stride ldx elements
  int8_t* codes;          // [rows, K], row stride ldc
  float* scale;           // [rows]
  long long ldx, ldc, rows;
  int K;
  bool vec_in, vec_out;   // every row of x starts on 16 bytes; every row of codes on 8 (4 for fp32 x)
};
cudaError_t launch_quantise(const QuantiseParams& p, int dtype, cudaStream_t st);

// y[r][n] = out(RN32(fma(RN32(sum_k a[r][k] w[g][n][k]), RN32(scale_a[r] scale_b[g][n]), bias[g][n]))) for the rows r of
// group g.
struct Int8Params {
  const int8_t* a;        // [T, K], row stride lda
  const int8_t* w;        // [E, N, K], row stride ldw, group stride gsw
  void* d;                // [T, N], row stride ldd
  const float* scale_a;   // [T] or one (sa_stride 0)
  const float* scale_b;   // [E, N] (sb_group, sb_stride), [N] or one
  const void* bias;       // null, or [E, N] (group stride bias_group)
  const int* offs;        // ends of the groups [E]; null: one group of all T rows
  int* status;            // device word: 1 when a bounded wait ran out
  long long lda, ldw, gsw, ldd, sb_group, bias_group;
  int T, N, K, E;
  int sa_stride, sb_stride;
  int bias_dtype, out_dtype;
  int zero_rest;          // rows behind the last group are set to zero
  int k_blocks, tiles_n, tiles_t;       // set by the launcher
  int wait_polls, announce_extra;
};
// Scratch memory for operands that TMA cannot read in place (0: none needed).
size_t int8_workspace_bytes(const Int8Params& p);
cudaError_t launch_int8(const Int8Params& p, void* workspace, cudaStream_t st, int* launches);
int int8_kernel_for(const Int8Params& p);       // mmb200_int8_kernel_for
// The device's status word (zero until a bounded wait of an int8 kernel runs out).
cudaError_t int8_status_word(int** word);

}  // namespace mmb
