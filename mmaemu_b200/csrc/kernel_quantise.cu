// Symmetric int8 quantisation with one scale per row: the operands of the int8 products (kernel_int8.cu).
//
// Per row: amax = max |x|, scale = RN32(amax / 127), code = the integer nearest to the real number 127 x / amax, ties to
// even. The codes are decided exactly, so they do not depend on how a division or a reciprocal rounds: x * RN(127 / amax) is
// off by less than 127 * 2^-24 = 7.6e-6, so its nearest integer is the answer unless it lies within 2e-5 of a half; there
// 254 |x| and (2 q + 1) amax are compared, both exact in fp64 (31 bits). A zero row has scale 0 and codes 0; a
// row with a NaN or an infinity has scale NaN and codes 0, so every product with it is NaN.
//
// What bounds it: one read of x and one write of the codes. A row is read once into registers (16-byte loads) by as many
// threads as hold it, the maximum is taken across them, and the codes leave from the registers. 8192 x 8192 bf16 takes 36.8 us,
// 5.5 TB/s or 83 % of the measured copy rate, fp32 58 us, 5.8 TB/s; for 16-bit values the issue slots are in use three quarters of the
// time (9 instructions per value and 4 more of a thread's fixed work), so instructions count: conversions on the quarter-rate pipe
// took 80 us, single FMAs 40. 1536 threads per SM leave 40 registers for each (the kernels take 32 to 39); blocks that keep a row
// ahead in registers took 49 us, 128 threads with twice the vectors 39. Of rows beyond 8192 fp32 or 16384 16-bit values, which no
// block holds, the rest is read a second time: 4096 x 16384 fp32 73 us, 4096 x 28672 bf16 82 us (4.6 and 4.3 TB/s of what has to
// move).
#include "common.cuh"
#include "int8.h"

#include <cuda_fp16.h>

namespace mmb {
namespace {

constexpr float SMALL = 7.8886090522101181e-31f;      // 2^-100: below it 127 / amax may overflow
constexpr float RAISE = 1.2676506002282294e+30f;      // 2^100

// A 16-byte vector of a type: how many values, their largest magnitude, their values in fp32. The magnitudes are kept as
// bit patterns, which order like the numbers, NaN above infinity; 16-bit ones in pairs.
template <int T>
struct Elem {
  static constexpr int SIZE = T == MMB200_HP_F32 ? 4 : 2, PER16 = 16 / SIZE;
  static __device__ __forceinline__ uint32_t top_of(uint32_t top, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) top = SIZE == 4 ? max(top, w[q] & 0x7FFFFFFFu) : __vmaxu2(top, w[q] & 0x7FFF7FFFu);
    return top;
  }
  static __device__ __forceinline__ float amax_of(uint32_t top) {     // of a maximum over all threads
    if (SIZE == 4) return __uint_as_float(top);
    const uint16_t h = (uint16_t)max(top & 0xFFFFu, top >> 16);
    return T == MMB200_HP_BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[PER16]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (SIZE == 4) {
        f[q] = __uint_as_float(w[q]);
      } else if constexpr (T == MMB200_HP_BF16) {
        f[2 * q] = __uint_as_float(w[q] << 16);
        f[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
      } else {
        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[q]));
        f[2 * q] = g.x;
        f[2 * q + 1] = g.y;
      }
    }
  }
};

// What a row's codes are computed with. Rows of tiny values are raised by 2^100 first (exact).
struct RowScale {
  float amax, inv;
  bool zero, tiny;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.zero = !(amax > 0.0f) || !(amax < __int_as_float(0x7F800000));
  r.tiny = amax < SMALL;
  r.amax = r.tiny ? __fmul_rn(amax, RAISE) : amax;
  r.inv = r.zero ? 0.0f : __fdiv_rn(127.0f, r.amax);
  return r;
}
__device__ __forceinline__ float scale_of(float amax) {
  return amax < __int_as_float(0x7F800000) ? __fdiv_rn(amax, 127.0f) : __uint_as_float(CANON_NAN32);
}
// Nearest integer of 127 x / amax where it is near a half: 254 |x| against (2 q + 1) amax, q the floor.
__device__ __forceinline__ uint32_t code_at_border(float x, const RowScale& r) {
  const int q = (int)floorf(__fmul_rn(fabsf(x), r.inv));
  const double twice = 254.0 * (double)fabsf(x), mid = (double)(2 * q + 1) * (double)r.amax;
  const int c = q + (twice > mid || (twice == mid && (q & 1)) ? 1 : 0);
  return (uint32_t)(x < 0.0f ? -c : c);
}
// Two fp32 FMAs in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long x, y, z, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
// The codes of N values, packed. In [2^23, 2^24) one ulp is 1, so RN(x inv + 1.5 * 2^23) holds the nearest integer in its
// low bits (ties to even, two's complement): two and a half instructions per value, none on the quarter-rate conversion pipe.
// `off` collects the largest distance from the integer, so that borders cost one test per vector.
template <int N>
__device__ __forceinline__ void codes_of(float (&x)[N], const RowScale& r, uint32_t (&w)[N / 4]) {
  constexpr float MAGIC = 12582912.0f, NEAR = 0.49998f;
  uint32_t b[N];
  float off = 0.0f;
  if (r.tiny) {
#pragma unroll
    for (int q = 0; q < N; ++q) x[q] = __fmul_rn(x[q], RAISE);
  }
  const float2 inv = make_float2(r.inv, r.inv), magic = make_float2(MAGIC, MAGIC), minus = make_float2(-1.0f, -1.0f);
#pragma unroll
  for (int q = 0; q < N; q += 2) {
    const float2 v = make_float2(x[q], x[q + 1]), m = fma2(v, inv, magic);
    const float2 d = fma2(v, inv, fma2(m, minus, magic));          // x inv - (m - MAGIC); the difference is exact
    off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
    b[q] = __float_as_uint(m.x);
    b[q + 1] = __float_as_uint(m.y);
  }
  if (off > NEAR) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (fabsf(__fmaf_rn(x[q], r.inv, -__fsub_rn(__uint_as_float(b[q]), MAGIC))) > NEAR) b[q] = code_at_border(x[q], r);
  }
#pragma unroll
  for (int q = 0; q < N / 4; ++q)
    w[q] = r.zero ? 0u : __byte_perm(__byte_perm(b[4 * q], b[4 * q + 1], 0x0040), __byte_perm(b[4 * q + 2], b[4 * q + 3], 0x0040), 0x5410);
}

// The row's threads (a warp, or the whole block) hold VPT 16-byte vectors each. The last vector of a row may be partial.
// What a row has beyond that is read twice.
template <int T, int BLOCK, bool WARP_ROW, int VPT>
__global__ void __launch_bounds__(BLOCK, 1536 / BLOCK) quantise_kernel(const __grid_constant__ QuantiseParams p) {
  using E = Elem<T>;
  dependent_launch_wait();
  dependent_launch_next();
  constexpr int PER = E::PER16, GROUP = WARP_ROW ? 32 : BLOCK;
  const int tid = WARP_ROW ? threadIdx.x % 32 : threadIdx.x;
  const long long row = WARP_ROW ? (long long)blockIdx.x * (BLOCK / 32) + threadIdx.x / 32 : (long long)blockIdx.x;
  if (WARP_ROW && row >= p.rows) return;               // whole warps; no block barrier in this form
  const char* x = static_cast<const char*>(p.x) + row * p.ldx * E::SIZE;
  int8_t* out = p.codes + row * p.ldc;
  const int vecs = (p.K + PER - 1) / PER;
  const bool vec_in = p.vec_in, vec_out = p.vec_out;
  auto load = [&](int v) -> uint4 {
    if (vec_in && (v + 1) * PER <= p.K) return __ldg(reinterpret_cast<const uint4*>(x) + v);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (v * PER + q >= p.K) break;
      if constexpr (E::SIZE == 4) w[q] = __ldg(reinterpret_cast<const uint32_t*>(x) + v * PER + q);
      else w[q / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(x) + v * PER + q) << (16 * (q % 2));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  auto store = [&](int v, const uint4& raw, const RowScale& r) {
    float f[PER];
    uint32_t w[PER / 4];
    E::unpack(raw, f);
    codes_of<PER>(f, r, w);
    if (vec_out && (v + 1) * PER <= p.K) {
      if (PER == 8) *reinterpret_cast<uint2*>(out + v * PER) = make_uint2(w[0], w[PER / 4 - 1]);
      else *reinterpret_cast<uint32_t*>(out + v * PER) = w[0];
    } else {
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (v * PER + q < p.K) out[v * PER + q] = (int8_t)(w[q / 4] >> (8 * (q % 4)));
    }
  };
  uint4 raw[VPT];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) raw[i] = i * GROUP + tid < vecs ? load(i * GROUP + tid) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int i = 0; i < VPT; ++i) top = E::top_of(top, raw[i]);
  for (int v = VPT * GROUP + tid; v < vecs; v += GROUP) top = E::top_of(top, load(v));
  if (E::SIZE == 2) top = max(top & 0xFFFFu, top >> 16);
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if constexpr (!WARP_ROW) {
    __shared__ uint32_t part[BLOCK / 32];
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = top;
    __syncthreads();
    top = part[threadIdx.x % (BLOCK / 32)];
    top = __reduce_max_sync(0xFFFFFFFFu, top);
  }
  const float amax = E::amax_of(top);
  const RowScale r = row_scale(amax);
  if (tid == 0) p.scale[row] = scale_of(amax);
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (i * GROUP + tid < vecs) store(i * GROUP + tid, raw[i], r);
  for (int v = VPT * GROUP + tid; v < vecs; v += GROUP) store(v, load(v), r);
}

template <int T>
cudaError_t launch(const QuantiseParams& p, cudaStream_t st) {
  const int vecs = (p.K + Elem<T>::PER16 - 1) / Elem<T>::PER16;
  if (vecs <= 64) return launch_dependent(quantise_kernel<T, 128, true, 2>, dim3((unsigned)((p.rows + 3) / 4)), 128, 0, st, p);
  if (vecs <= 256) return launch_dependent(quantise_kernel<T, 128, false, 2>, dim3((unsigned)p.rows), 128, 0, st, p);
  if (vecs <= 1024) return launch_dependent(quantise_kernel<T, 256, false, 4>, dim3((unsigned)p.rows), 256, 0, st, p);
  return launch_dependent(quantise_kernel<T, 512, false, 4>, dim3((unsigned)p.rows), 512, 0, st, p);
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
