// Symmetric int8 quantisation with one scale per row: the operands of the int8 products (kernel_int8.cu).
//
// Per row: amax = max |x|, scale = RN32(amax / 127), code = the integer nearest to the real number 127 x / amax, ties to
// even. The codes are decided exactly, so they do not depend on how a division or a reciprocal rounds: t = RN(x * RN(127 /
// amax)) is off by less than 127 * 2^-22.9 = 1.7e-5, so its nearest integer is the answer unless t lies within 2e-5 of a
// half; there 254 |x| and (2 q + 1) amax are compared, both exact in fp64 (31 bits). A zero row has scale 0 and codes 0; a
// row with a NaN or an infinity has scale NaN and codes 0, so every product with it is NaN.
//
// What bounds it: one read of x and one write of the codes. A row is read once into registers (16-byte loads) by as many
// threads as hold it, the maximum is taken across them, and the codes leave from the registers.
#include "common.cuh"
#include "int8.h"

#include <cuda_fp16.h>

namespace mmb {
namespace {

constexpr float SMALL = 7.8886090522101181e-31f;      // 2^-100: below it 127 / amax may overflow

template <int T>
struct Elem;
template <>
struct Elem<MMB200_HP_F32> {
  static constexpr int SIZE = 4, PER16 = 4;
  static __device__ __forceinline__ float get(const void* p, long long i) { return __ldg(static_cast<const float*>(p) + i); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <>
struct Elem<MMB200_HP_BF16> {
  static constexpr int SIZE = 2, PER16 = 8;
  static __device__ __forceinline__ float get(const void* p, long long i) {
    return __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t*>(p) + i) << 16);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[2 * q] = __uint_as_float(w[q] << 16);
      f[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
    }
  }
};
template <>
struct Elem<MMB200_HP_F16> {
  static constexpr int SIZE = 2, PER16 = 8;
  static __device__ __forceinline__ float get(const void* p, long long i) { return __half2float(__ldg(static_cast<const __half*>(p) + i)); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[q]));
      f[2 * q] = g.x;
      f[2 * q + 1] = g.y;
    }
  }
};

// What a row's codes are computed with.
struct RowScale {
  float amax, inv;
  bool zero, exact;      // no codes but 0; decide every code in fp64
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.amax = amax;
  r.zero = !(amax > 0.0f) || !(amax < __int_as_float(0x7F800000));
  r.exact = amax < SMALL;
  r.inv = r.zero || r.exact ? 0.0f : __fdiv_rn(127.0f, amax);
  return r;
}
__device__ __forceinline__ float scale_of(float amax) {
  return amax < __int_as_float(0x7F800000) ? __fdiv_rn(amax, 127.0f) : __uint_as_float(CANON_NAN32);
}
// Nearest integer of 127 x / amax by exact comparison: 254 |x| against (2 q + 1) amax for q = the floor.
__device__ __noinline__ int code_exact(float x, float amax) {
  const double twice = 254.0 * (double)fabsf(x), a = (double)amax;
  double q = floor(twice / (2.0 * a));                 // at most one off; put right below
  if (2.0 * q * a > twice) q -= 1.0;
  else if (2.0 * (q + 1.0) * a <= twice) q += 1.0;
  const double mid = (2.0 * q + 1.0) * a;
  int c = (int)q;
  if (twice > mid || (twice == mid && (c & 1))) ++c;
  return x < 0.0f ? -c : c;
}
__device__ __forceinline__ int code_of(float x, const RowScale& r) {
  const float t = __fmul_rn(x, r.inv), q = rintf(t);
  int c = (int)q;
  if (r.exact || fabsf(t - q) > 0.49998f) c = code_exact(x, r.amax);
  return c;
}
// max(a, |b|) with NaN kept as +infinity's successor: non-negative floats order like their bit patterns, NaN above infinity.
__device__ __forceinline__ uint32_t abs_max(uint32_t a, float b) { return max(a, __float_as_uint(b) & 0x7FFFFFFFu); }

// THREADS threads per row (a warp, or the whole block), up to VPT 16-byte vectors each. The last vector of a row may be
// partial. Rows longer than THREADS * VPT vectors are read twice.
template <int T, int BLOCK, bool WARP_ROW, int VPT>
__global__ void __launch_bounds__(BLOCK) quantise_kernel(const __grid_constant__ QuantiseParams p) {
  using E = Elem<T>;
  constexpr int PER = E::PER16, GROUP = WARP_ROW ? 32 : BLOCK;
  const int tid = WARP_ROW ? threadIdx.x % 32 : threadIdx.x;
  const long long row = WARP_ROW ? (long long)blockIdx.x * (BLOCK / 32) + threadIdx.x / 32 : (long long)blockIdx.x;
  if (WARP_ROW && row >= p.rows) return;               // whole warps; no block barrier in this form
  const char* x = static_cast<const char*>(p.x) + row * p.ldx * E::SIZE;
  int8_t* out = p.codes + row * p.ldc;
  const int vecs = (p.K + PER - 1) / PER;
  const bool vec_in = p.vec_in, vec_out = p.vec_out;
  auto load = [&](int v, float* f) {
    if (vec_in && (v + 1) * PER <= p.K) {
      E::unpack(__ldg(reinterpret_cast<const uint4*>(x) + v), f);
    } else {
#pragma unroll
      for (int q = 0; q < PER; ++q) f[q] = v * PER + q < p.K ? E::get(x, v * PER + q) : 0.0f;
    }
  };
  auto store = [&](int v, const float* f, const RowScale& r) {
    uint32_t w[PER / 4];
#pragma unroll
    for (int q = 0; q < PER / 4; ++q) {
      w[q] = 0;
      if (!r.zero) {
#pragma unroll
        for (int b = 0; b < 4; ++b) w[q] |= (uint32_t)(code_of(f[4 * q + b], r) & 0xFF) << (8 * b);
      }
    }
    if (vec_out && (v + 1) * PER <= p.K) {
      if (PER == 8) *reinterpret_cast<uint2*>(out + v * PER) = make_uint2(w[0], w[PER / 4 - 1]);
      else *reinterpret_cast<uint32_t*>(out + v * PER) = w[0];
    } else {
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (v * PER + q < p.K) out[v * PER + q] = (int8_t)(w[q / 4] >> (8 * (q % 4)));
    }
  };
  float f[VPT][PER];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * GROUP + tid;
    if (v < vecs) load(v, f[i]);
    else
#pragma unroll
      for (int q = 0; q < PER; ++q) f[i][q] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int q = 0; q < PER; ++q) top = abs_max(top, f[i][q]);
  for (int v = VPT * GROUP + tid; v < vecs; v += GROUP) {
    float g[PER];
    load(v, g);
#pragma unroll
    for (int q = 0; q < PER; ++q) top = abs_max(top, g[q]);
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if constexpr (!WARP_ROW) {
    __shared__ uint32_t part[BLOCK / 32];
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = top;
    __syncthreads();
    top = part[threadIdx.x % (BLOCK / 32)];
    top = __reduce_max_sync(0xFFFFFFFFu, top);
  }
  const float amax = __uint_as_float(top);
  const RowScale r = row_scale(amax);
  if (tid == 0) p.scale[row] = scale_of(amax);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * GROUP + tid;
    if (v < vecs) store(v, f[i], r);
  }
  for (int v = VPT * GROUP + tid; v < vecs; v += GROUP) {
    float g[PER];
    load(v, g);
    store(v, g, r);
  }
}

template <int T>
cudaError_t launch(const QuantiseParams& p, cudaStream_t st) {
  const int vecs = (p.K + Elem<T>::PER16 - 1) / Elem<T>::PER16;
  if (vecs <= 64) quantise_kernel<T, 128, true, 2><<<(unsigned)((p.rows + 3) / 4), 128, 0, st>>>(p);
  else if (vecs <= 256) quantise_kernel<T, 128, false, 2><<<(unsigned)p.rows, 128, 0, st>>>(p);
  else if (vecs <= 1024) quantise_kernel<T, 256, false, 4><<<(unsigned)p.rows, 256, 0, st>>>(p);
  else quantise_kernel<T, 512, false, 4><<<(unsigned)p.rows, 512, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantise(const QuantiseParams& p, int dtype, cudaStream_t st) {
  switch (dtype) {
    case MMB200_HP_F32: return launch<MMB200_HP_F32>(p, st);
    case MMB200_HP_BF16: return launch<MMB200_HP_BF16>(p, st);
    default: return launch<MMB200_HP_F16>(p, st);
  }
}

}  // namespace mmb
