// Launch parameters of the int8 operators (kernel_quantise.cu, kernel_int8.cu) and their launchers; no part of common.cuh,
// which the emulated kernels share.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mmb {

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
  int* status;            // device word that bounded waits count up when they run out; null: the device's common one
  long long lda, ldw, gsw, ldd, sa_stride, sb_stride, sb_group, bias_group;
  int T, N, K, E;
  int bias_dtype, out_dtype;
  int zero_rest;          // rows behind the last group are set to zero
  int k_blocks, tiles_n;  // set by the launcher
  int wait_polls, announce_extra;
};
// Scratch memory for operands that TMA cannot read in place (0: none needed).
size_t int8_workspace_bytes(const Int8Params& p);
cudaError_t launch_int8(const Int8Params& p, void* workspace, cudaStream_t st, int* launches);
int int8_kernel_for(const Int8Params& p);       // mmb200_int8_kernel_for
// The current device's status words, which bounded waits of the int8 kernels count up when they run out (and nobody clears): the
// common one, then those of the calls that check their own waits.
constexpr int INT8_STATUS_WORDS = 65;
cudaError_t int8_status_words(int** words);

}  // namespace mmb
