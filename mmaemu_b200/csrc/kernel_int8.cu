// Products of int8 matrices with a scale for each row and column: y = out(fma(RN32(acc), RN32(sa sb), bias)), acc the exact
// int32 sum over k (K <= 131071, so |acc| <= 2^14 K < 2^31). Dense, or for ragged groups of rows with a weight matrix each.
//
// tcgen05.mma kind::i8 (int8 x int8 into int32 in TMEM). The weights' output channels are the 128 lanes of the accumulator
// and the rows (tokens) its columns, so few rows make a narrow tile instead of an empty one, the channel's scale and bias are
// one register per thread, and the stores of a warp cover 32 consecutive outputs of a row.
//
// int8_tile_kernel: few rows. One tile of 128 channels x 16, 32 or 64 rows per cluster; the CTAs of a cluster each take a part of
// K and add their int32 sums through distributed shared memory. Integer sums are exact in any order, so the split changes no
// bit. Bound by reading the weights: 16 x 8192 x 28672 in 40 us, 5.8 TB/s; 16 x 4096 x 8192 in 10.5 us (8.2 where the 33.5 MB of
// weights are still in L2), of which 3.5 are launch, first copies and the cluster's sum (64 rows, 512 channels, K = 512 in 3.3 us;
// 13 while a thread read the sums one by one). Times of this file: replayed from a graph over operands that do not stay in L2.
//
// int8_single_kernel, int8_pair_kernel: more rows. Persistent; TMEM holds two accumulators, so the output of a tile leaves while
// the next one is multiplied. A CTA works on 128 channels x 64, 128 or 256 rows, a pair of CTAs on neighbouring SMs
// (cta_group::2) on 256 x 256, each holding half of both operands, so that a byte of shared memory feeds twice the products.
// Large products are bound by power: 8192 x 24576 x 8192 takes 1.15 ms, 2.87 POP/s (a call among others 1.19 ms, 2.77); the 8192-cube
// 2.9 POP/s, with operands of zeros 4.0. 4096 rows in 64 groups on 1536 x 2048 weights: 45 us for 201 MB of weights (one-tile
// CTAs: 55 us).
//
// An MMA of 128 channels takes about 120 cycles up to 128 rows, so a CTA needs 0.25 us per 128 bytes of K however few rows it
// has. The output loop must not wait: with a scale loaded per row instead of handed round by shuffles it took 27 us per tile of
// 256 x 256, now 4.5 us, which still bounds products with K of 1024 and less (8192 x 8192 x 1024: 64 to 72 us, of which the MMAs
// would take 37).
#include <cuda.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstring>

#include "int8.h"
#include "staging.cuh"

namespace mmb {
namespace {

__device__ int g_int8_status[INT8_STATUS_WORDS];

constexpr int CH = 128;                    // output channels of a tile
constexpr int KB = 128;                    // bytes of K per stage: one 128-byte swizzle atom
constexpr int TILE_THREADS = 192;          // warp 0: copies, warp 1: MMAs, warps 2 to 5: output

// ---- device helpers
__device__ __forceinline__ uint64_t desc_sw128(const void* ptr) {      // K-major, 128-byte swizzle, 8-row groups 1024 bytes apart
  return ((uint64_t)(smem_addr(ptr) >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void commit(unsigned long long* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Copies of a box of rows (channels) for a kernel of CTAS CTAs per worker; `bar`: shared address of the barrier they count on.
template <int CTAS>
__device__ __forceinline__ void load_rows(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CTAS == 1)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_channels(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CTAS == 1)
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int4 remote_int4(uint32_t addr, int rank) {        // of a CTA of the cluster
  uint32_t there;
  int4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(there));
  return v;
}
template <int N>
__device__ __forceinline__ void tmem_load(int (&r)[N], uint32_t addr) {
  static_assert(N == 16 || N == 32, "columns of a load");
#pragma unroll
  for (int h = 0; h < N; h += 16)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
                 "[%16];"
                 : "=r"(r[h]), "=r"(r[h + 1]), "=r"(r[h + 2]), "=r"(r[h + 3]), "=r"(r[h + 4]), "=r"(r[h + 5]), "=r"(r[h + 6]),
                   "=r"(r[h + 7]), "=r"(r[h + 8]), "=r"(r[h + 9]), "=r"(r[h + 10]), "=r"(r[h + 11]), "=r"(r[h + 12]),
                   "=r"(r[h + 13]), "=r"(r[h + 14]), "=r"(r[h + 15])
                 : "r"(addr + h) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int q = 0; q < N; ++q) asm volatile("" : "+r"(r[q])::"memory");
}

// ---- the output of one thread: channel n of group g
template <int OUT> struct OutType;
template <> struct OutType<MMB200_OUT_F32> { using type = uint32_t; };
template <> struct OutType<MMB200_OUT_BF16> { using type = uint16_t; };
template <> struct OutType<MMB200_OUT_F16> { using type = uint16_t; };

__device__ __forceinline__ float bias_at(const Int8Params& p, long long i) {
  if (!p.bias) return 0.0f;
  if (p.bias_dtype == MMB200_HP_F32) return __ldg(static_cast<const float*>(p.bias) + i);
  if (p.bias_dtype == MMB200_HP_F16) return __half2float(__ldg(static_cast<const __half*>(p.bias) + i));
  return __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t*>(p.bias) + i) << 16);
}
// (FMA and the conversions return the framework's NaN: 0x7FFFFFFF, 0x7FFF)
template <int OUT>
__device__ __forceinline__ typename OutType<OUT>::type out_bits(float y) {
  if constexpr (OUT == MMB200_OUT_F32) return __float_as_uint(y);
  uint16_t h;
  if constexpr (OUT == MMB200_OUT_BF16) asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(h) : "f"(y));
  else asm("cvt.rn.f16.f32 %0, %1;" : "=h"(h) : "f"(y));
  return h;
}
// Scale of row `lane` of a chunk of CHUNK rows, `left` of which exist.
template <int CHUNK>
__device__ __forceinline__ float row_scales(const Int8Params& p, long long row, int left) {
  const int lane = threadIdx.x % 32;
  return lane < CHUNK && lane < left ? __ldg(p.scale_a + (row + lane) * p.sa_stride) : 0.0f;
}
// The output of a warp: its 32 channels (one per lane; `real`: inside N) of the rows [row0, row0 + rows), whose sums are the
// columns of the accumulator at `acc`, or zero without products. The scale of a row is held by one lane and handed round;
// `scale` comes in for the first chunk, so that its load runs before the accumulator is complete.
template <int OUT, int BT>
__device__ __forceinline__ void write_rows(const Int8Params& p, uint32_t acc, bool products, long long row0, int rows, int n, bool real, float sb,
                                           float bias, float scale) {
  constexpr int CHUNK = BT < 32 ? BT : 32;
  using O = typename OutType<OUT>::type;
  O* out = static_cast<O*>(p.d) + row0 * p.ldd + n;
  auto value = [&](int sum, float s, int q) {
    return out_bits<OUT>(__fmaf_rn(__int2float_rn(sum), __fmul_rn(__shfl_sync(0xFFFFFFFFu, s, q), sb), bias));
  };
#pragma unroll 1
  for (int c = 0; c < rows; c += CHUNK) {
    int r[CHUNK];
    if (products) {
      tmem_load<CHUNK>(r, acc + c);
    } else {
#pragma unroll
      for (int q = 0; q < CHUNK; ++q) r[q] = 0;
    }
    const float s = scale;
    scale = row_scales<CHUNK>(p, row0 + c + CHUNK, rows - c - CHUNK);
    const int left = rows - c;
    if (left >= CHUNK && __all_sync(0xFFFFFFFFu, real)) {
#pragma unroll
      for (int q = 0; q < CHUNK; q += 8) {
        O y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = value(r[q + j], s, q + j);
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j * p.ldd] = y[j];
        out += 8 * p.ldd;
      }
    } else {
#pragma unroll
      for (int q = 0; q < CHUNK; ++q) {
        const O y = value(r[q], s, q);
        if (real && q < left) *out = y;
        out += p.ldd;
      }
    }
  }
}

// The same for the sums of a cluster, [row][channel] in the shared memory of each of its CTAs: CTA `rank` writes the rows
// rank, rank + parts, ..., a warp a row, a lane four channels. All the loads of a row are in flight at once.
template <int OUT>
__device__ __forceinline__ void write_sums(const Int8Params& p, const int* part, int parts, int rank, long long row0, int rows, int n0, int g) {
  using O = typename OutType<OUT>::type;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32 - 2, n = n0 + 4 * lane;
  float sb[4], bias[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    sb[q] = n + q < p.N ? __ldg(p.scale_b + (long long)g * p.sb_group + (long long)(n + q) * p.sb_stride) : 0.0f;
    bias[q] = n + q < p.N ? bias_at(p, (long long)g * p.bias_group + n + q) : 0.0f;
  }
  for (int c = rank + parts * warp; c < rows; c += 4 * parts) {
    const uint32_t addr = smem_addr(part + c * CH + 4 * lane);
    int4 v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < parts) v[q] = remote_int4(addr, q);
    const float sa = __ldg(p.scale_a + (row0 + c) * p.sa_stride);
    int sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q < parts) { sum[0] += v[q].x; sum[1] += v[q].y; sum[2] += v[q].z; sum[3] += v[q].w; }
    O* out = static_cast<O*>(p.d) + (row0 + c) * p.ldd + n;
    O y[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) y[q] = out_bits<OUT>(__fmaf_rn(__int2float_rn(sum[q]), __fmul_rn(sa, sb[q]), bias[q]));
    if (n + 4 <= p.N && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(O)) == 0) {
      if constexpr (sizeof(O) == 4) *reinterpret_cast<uint4*>(out) = make_uint4(y[0], y[1], y[2], y[3]);
      else *reinterpret_cast<uint2*>(out) = make_uint2(y[0] | ((uint32_t)y[1] << 16), y[2] | ((uint32_t)y[3] << 16));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (n + q < p.N) out[q] = y[q];
    }
  }
}

// ---- groups. Ends are taken as a running maximum, clamped to [0, T], so that no content of offs leads out of the operands.
struct Group { int g, start, end, tile, last; };       // g < 0: no such tile; last: the end of the last group
// 32 groups at a time, one per lane of a warp: rows [start, end) and the tiles of BT rows up to the group's last. `last`: the end
// of the groups before the chunk; `tiles`: their tiles.
template <int BT>
struct GroupChunk {
  int start, end, upto;
  __device__ __forceinline__ void load(const Int8Params& p, int base, int last, int tiles) {
    const int lane = threadIdx.x % 32;
    end = !p.offs ? p.T : base + lane < p.E ? min(max(__ldg(p.offs + base + lane), 0), p.T) : 0;
    end = max(end, last);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xFFFFFFFFu, end, d);
      if (lane >= d) end = max(end, other);
    }
    start = __shfl_up_sync(0xFFFFFFFFu, end, 1);
    if (lane == 0) start = last;
    upto = (end - start + BT - 1) / BT + (lane == 0 ? tiles : 0);
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xFFFFFFFFu, upto, d);
      if (lane >= d) upto += other;
    }
  }
};
// The group of tile `slot` of BT rows, found by one warp (every lane returns it).
template <int BT>
__device__ __forceinline__ Group find_group(const Int8Params& p, int slot) {
  if (!p.offs) return Group{0, 0, p.T, slot, p.T};
  int tiles = 0, last = 0, base = 0;
  Group r{-1, 0, 0, 0, 0};
  GroupChunk<BT> c;
  for (; base < p.E && r.g < 0; base += 32) {
    c.load(p, base, last, tiles);
    const unsigned after = __ballot_sync(0xFFFFFFFFu, c.upto > slot);
    if (after) {
      const int l = __ffs(after) - 1;
      r.g = base + l;
      r.start = __shfl_sync(0xFFFFFFFFu, c.start, l);
      r.end = __shfl_sync(0xFFFFFFFFu, c.end, l);
      r.tile = slot - __shfl_sync(0xFFFFFFFFu, c.upto - (c.end - c.start + BT - 1) / BT, l);
    }
    tiles = __shfl_sync(0xFFFFFFFFu, c.upto, 31);
    last = __shfl_sync(0xFFFFFFFFu, c.end, 31);
  }
  if (p.zero_rest) {                         // the end of the last group
    for (int e = base + threadIdx.x % 32; e < p.E; e += 32) last = max(last, min(max(__ldg(p.offs + e), 0), p.T));
    last = __reduce_max_sync(0xFFFFFFFFu, last);
  }
  r.last = last;
  return r;
}
// Zeros in the rows behind the last group: the channels [n0, n1), rows first, first + step, ... by `threads` threads.
template <int OUT>
__device__ __forceinline__ void zero_rows(const Int8Params& p, int first, int step, int n0, int n1, int thread, int threads) {
  if (!p.zero_rest) return;
  for (long long row = first; row < p.T; row += step)
    for (int n = n0 + thread; n < n1; n += threads) static_cast<typename OutType<OUT>::type*>(p.d)[row * p.ldd + n] = 0;
}

template <int BT>
constexpr int tile_stages() { return BT <= 16 ? 6 : (BT <= 32 ? 5 : 4); }
template <int BT>
struct SmemTile {
  static constexpr int STAGES = tile_stages<BT>();
  struct Stage { unsigned char w[CH * KB], a[BT * KB]; } stage[STAGES];
  unsigned long long full[STAGES], empty[STAGES], done;
  uint32_t tmem;
  Group group;
};

template <int BT, int OUT>
__global__ void __launch_bounds__(TILE_THREADS) int8_tile_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                 const __grid_constant__ CUtensorMap map_a,
                                                                 const __grid_constant__ Int8Params p) {
  using Smem = SmemTile<BT>;
  constexpr int STAGES = Smem::STAGES, COLS = BT < 32 ? 32 : BT;
  static_assert(STAGES * sizeof(typename Smem::Stage) >= (size_t)BT * CH * 4, "partial sums reuse the stages");
  extern __shared__ unsigned char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int rank, parts;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
  const int n0 = (int)(blockIdx.x / (unsigned)parts) * CH;
  const int kb0 = (int)((long long)p.k_blocks * rank / parts), nk = (int)((long long)p.k_blocks * (rank + 1) / parts) - kb0;
  if (threadIdx.x == 0) {
    for (int q = 0; q < STAGES; ++q) { mbar_init(&sm.full[q], 1); mbar_init(&sm.empty[q], 1); }
    mbar_init(&sm.done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  dependent_launch_wait();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem)), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (warp == 2) {
    const Group found = find_group<BT>(p, (int)blockIdx.y);
    if (lane == 0) sm.group = found;
  }
  fence_before();
  __syncthreads();
  fence_after();
  dependent_launch_next();
  const uint32_t tmem = sm.tmem;
  const Group g = sm.group;
  const int row0 = g.start + g.tile * BT;
  const bool work = g.g >= 0 && row0 < g.end;     // the same for every CTA of the cluster
  if (warp >= 2 && rank == 0) zero_rows<OUT>(p, g.last + (int)blockIdx.y, (int)gridDim.y, n0, min(n0 + CH, p.N), threadIdx.x - 64, 128);
  bool ok = true;
  if (work && nk > 0) {
    if (warp == 0) {
      if (lane == 0) {
        int issued = 0;
        for (int t = 0; t < nk; ++t) {
          const int s = t % STAGES;
          if (t >= STAGES && !mbar_wait(&sm.empty[s], ((t / STAGES) - 1) & 1, p.wait_polls)) { ok = false; break; }
          mbar_expect_tx(&sm.full[s], (uint32_t)sizeof(typename Smem::Stage) + (uint32_t)p.announce_extra);
          load_channels<1>(sm.stage[s].w, &map_w, (kb0 + t) * KB, n0, g.g, smem_addr(&sm.full[s]));
          load_rows<1>(sm.stage[s].a, &map_a, (kb0 + t) * KB, row0, smem_addr(&sm.full[s]));
          issued = t + 1;
        }
        // the CTA must not end while a copy may be in flight: wait for the last copy into every stage (bounded)
        for (int t = issued > STAGES ? issued - STAGES : 0; t < issued; ++t)
          if (!mbar_wait(&sm.full[t % STAGES], (t / STAGES) & 1, p.wait_polls)) ok = false;
      }
      __syncwarp();
    } else if (warp == 1) {
      if (lane == 0) {
        // int32 accumulator, signed 8-bit operands, both K-major
        constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BT >> 3) << 17) | ((uint32_t)(CH >> 4) << 24);
        for (int t = 0; t < nk; ++t) {
          const int s = t % STAGES;
          if (!mbar_wait(&sm.full[s], (t / STAGES) & 1, p.wait_polls)) { ok = false; break; }
          fence_after();
          const uint64_t dw = desc_sw128(sm.stage[s].w), da = desc_sw128(sm.stage[s].a);
#pragma unroll
          for (int k = 0; k < KB / 32; ++k)         // 32 k per instruction: 32 bytes further inside the swizzle atom
            mma_i8(tmem, dw + 2 * k, da + 2 * k, IDESC, t > 0 || k > 0 ? 1u : 0u);
          commit(&sm.empty[s]);
        }
        commit(&sm.done);
      }
      __syncwarp();
    }
    // everyone: the products of this CTA are complete (a failed role still commits, so this ends)
    if (!mbar_wait(&sm.done, 0, p.wait_polls)) ok = false;
    fence_after();
  }
  if (!ok) atomicAdd(p.status, 1);
  const bool bad = __syncthreads_or(ok ? 0 : 1) != 0;
  const int lane_ch = 32 * (warp % 4) + lane, n = n0 + lane_ch;
  const uint32_t mine = tmem + ((uint32_t)(32 * (warp % 4)) << 16);
  int* part = reinterpret_cast<int*>(&sm.stage[0]);                 // [column][channel]
  if (parts > 1) {
    if (warp >= 2 && work) {
#pragma unroll 1
      for (int c = 0; c < BT; c += 16) {
        int r[16];
        if (nk > 0) {
          tmem_load(r, mine + c);
        } else {
#pragma unroll
          for (int q = 0; q < 16; ++q) r[q] = 0;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) part[(c + q) * CH + lane_ch] = r[q];
      }
    }
    cluster_arrive();
    cluster_wait();
  }
  if (work && warp >= 2 && !bad) {
    const bool real = n < p.N;
    const float sb = real ? __ldg(p.scale_b + (long long)g.g * p.sb_group + (long long)n * p.sb_stride) : 0.0f;
    const float bias = real ? bias_at(p, (long long)g.g * p.bias_group + n) : 0.0f;
    const int rows = min(g.end - row0, BT);
    if (parts == 1) write_rows<OUT, BT>(p, mine, nk > 0, row0, rows, n, real, sb, bias, row_scales<(BT < 32 ? BT : 32)>(p, row0, rows));
    else write_sums<OUT>(p, part, parts, rank, row0, rows, n0, g.g);
  }
  if (parts > 1) {                                  // nobody leaves while its sums may be read
    cluster_arrive();
    cluster_wait();
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLS));
  }
}

// ---- persistent workers: one CTA per SM, or a pair of CTAs on neighbouring SMs
// Ragged groups: the end of a group's rows and the tiles of BT rows up to it, in shared memory.
struct GroupTable { int end, upto; };
// A worker's tile is CH * CTAS channels x up to BT rows. In a pair each CTA holds its channels and half of the rows.
template <int CTAS, int BT>
struct Worker {
  static constexpr int ROWS = BT / CTAS;                            // rows that a CTA brings, at most
  static constexpr int BOX = ROWS < 64 ? ROWS : 64;                 // a copy's rows: only the copies that a tile needs are made
  static constexpr int STAGES = 196608 / ((CH + ROWS) * KB);        // 192 KB of stages
  static constexpr int COLS = 2 * BT < 32 ? 32 : 2 * BT;            // two accumulators
  struct Stage { unsigned char w[CH * KB], a[ROWS * KB]; };
  struct Smem {
    Stage stage[STAGES];
    unsigned long long full[STAGES];       // (of the pair's first CTA) the copies of all CTAs have landed
    unsigned long long empty[STAGES];      // the MMAs that read the stage are done
    unsigned long long acc_full[2];        // the accumulator is complete
    unsigned long long acc_empty[2];       // (first CTA) all output warps have read it
    unsigned long long drain;
    uint32_t tmem;
    GroupTable groups[1];                  // as many as the launch has groups
  };
  static size_t bytes(const Int8Params& p) { return sizeof(Smem) + 1024 + (p.offs ? sizeof(GroupTable) * (size_t)p.E : 0); }
};
constexpr int WORKER_THREADS = 320;        // warp 0: copies, warp 1: MMAs, warps 2 to 9: output (a quarter of the channels, half of the rows)
constexpr int BAND_ROWS = 2048;            // rows that share a pass over the channels (16 MB of them at K = 8192 stay in L2)

template <int CTAS>
__device__ __forceinline__ uint32_t first_cta(const void* ptr) {
  if constexpr (CTAS == 1) return smem_addr(ptr);
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(ptr)));
  return a;
}
template <int CTAS>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  if constexpr (CTAS == 1)
    mma_i8(d, a, b, idesc, add);
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void commit_all(unsigned long long* bar) {        // arrives at the barrier of every CTA of the worker
  if constexpr (CTAS == 1)
    commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
}

// Written by one warp.
template <int BT>
__device__ __forceinline__ void write_groups(const Int8Params& p, GroupTable* table) {
  const int lane = threadIdx.x % 32;
  int tiles = 0, last = 0;
  GroupChunk<BT> c;
  for (int base = 0; base < p.E; base += 32) {
    c.load(p, base, last, tiles);
    if (base + lane < p.E) table[base + lane] = GroupTable{c.end, c.upto};
    tiles = __shfl_sync(0xFFFFFFFFu, c.upto, 31);
    last = __shfl_sync(0xFFFFFFFFu, c.end, 31);
  }
}
// The tiles of a launch in order: group by group, inside a group bands of BAND_ROWS rows, inside a band channel tile by
// channel tile. A worker walks an increasing sequence of indices; every role of a CTA has a walker of its own.
template <int BT>
struct Walker {
  int g = 0, end = 0;
  __device__ __forceinline__ bool find(const Int8Params& p, const GroupTable* table, int tiles_n, long long t, int& row0, int& n_tile) {
    constexpr int BAND = BAND_ROWS / BT;
    int start = 0, before = 0, upto;
    if (p.offs) {
      if ((long long)table[g].upto * tiles_n <= t) {       // the first group behind with more tiles up to it
        int lo = g + 1, hi = p.E;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if ((long long)table[mid].upto * tiles_n > t) hi = mid;
          else lo = mid + 1;
        }
        if (lo >= p.E) return false;
        g = lo;
      }
      if (g > 0) {
        start = table[g - 1].end;
        before = table[g - 1].upto;
      }
      end = table[g].end;
      upto = table[g].upto;
    } else {
      end = p.T;
      upto = (p.T + BT - 1) / BT;
      if ((long long)upto * tiles_n <= t) return false;
    }
    const int tiles_t = upto - before;
    const long long i = t - (long long)before * tiles_n, per_band = (long long)BAND * tiles_n;
    const int band = (int)(i / per_band), j = (int)(i - band * per_band), width = min(BAND, tiles_t - band * BAND);
    n_tile = j / width;
    row0 = start + (band * BAND + j % width) * BT;
    return true;
  }
  // Columns of the tile's accumulator: its rows, rounded up to what the MMA takes (16, a pair 32).
  template <int CTAS>
  __device__ __forceinline__ int columns(int row0) const {
    constexpr int STEP = 16 * CTAS;
    return min(BT, (end - row0 + STEP - 1) / STEP * STEP);
  }
};

template <int CTAS, int BT, int OUT>
__device__ __forceinline__ void int8_worker(const CUtensorMap& map_w, const CUtensorMap& map_a, const Int8Params& p) {
  using W = Worker<CTAS, BT>;
  constexpr int STAGES = W::STAGES;
  extern __shared__ unsigned char smem_raw[];
  typename W::Smem& sm = *reinterpret_cast<typename W::Smem*>(smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int rank = 0;
  if (CTAS == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int tiles_n = (p.N + CTAS * CH - 1) / (CTAS * CH), nk = p.k_blocks;
  const long long first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
  if (threadIdx.x == 0) {
    for (int q = 0; q < STAGES; ++q) { mbar_init(&sm.full[q], 1); mbar_init(&sm.empty[q], 1); }
    for (int q = 0; q < 2; ++q) { mbar_init(&sm.acc_full[q], 1); mbar_init(&sm.acc_empty[q], 8 * CTAS); }
    mbar_init(&sm.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  dependent_launch_wait();
  if (warp == 2 && p.offs) write_groups<BT>(p, sm.groups);
  if (warp == 1) {
    if constexpr (CTAS == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem)), "n"(W::COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sm.tmem)), "n"(W::COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) {                        // the other CTA's barriers and TMEM are ready too
    cluster_arrive();
    cluster_wait();
  }
  fence_after();
  dependent_launch_next();
  const uint32_t tmem = sm.tmem;
  bool ok = true;
  Walker<BT> walk;
  int row0, n_tile;
  if (warp == 0) {
    if (lane == 0) {
      unsigned it = 0;
      for (long long t = first; ok && walk.find(p, sm.groups, tiles_n, t, row0, n_tile); t += step) {
        const int mine = walk.template columns<CTAS>(row0) / CTAS, my_row = row0 + mine * rank, boxes = (mine + W::BOX - 1) / W::BOX;
        const uint32_t bytes = CTAS * (uint32_t)(sizeof(sm.stage[0].w) + boxes * W::BOX * KB);
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const unsigned s = it % STAGES, round = it / STAGES;
          if (round && !mbar_wait(&sm.empty[s], (round - 1) & 1, p.wait_polls)) { ok = false; break; }
          if (rank == 0) mbar_expect_tx(&sm.full[s], bytes + (uint32_t)p.announce_extra);
          const uint32_t bar = first_cta<CTAS>(&sm.full[s]);
          load_channels<CTAS>(sm.stage[s].w, &map_w, kb * KB, (CTAS * n_tile + rank) * CH, walk.g, bar);
          for (int q = 0; q < boxes; ++q) load_rows<CTAS>(sm.stage[s].a + q * W::BOX * KB, &map_a, kb * KB, my_row + q * W::BOX, bar);
        }
      }
      // no CTA ends while a copy may be in flight: the worker's first CTA waits for the last copies into every stage (bounded)
      if (rank == 0)
        for (unsigned q = it > (unsigned)STAGES ? it - STAGES : 0; q < it; ++q)
          if (!mbar_wait(&sm.full[q % STAGES], (q / STAGES) & 1, p.wait_polls)) ok = false;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t SHAPE = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(CTAS * CH >> 4) << 24);
      unsigned it = 0, i = 0;
      for (long long t = first; ok && walk.find(p, sm.groups, tiles_n, t, row0, n_tile); t += step, ++i) {
        const uint32_t acc = tmem + (i & 1) * BT, idesc = SHAPE | ((uint32_t)(walk.template columns<CTAS>(row0) >> 3) << 17);
        if (i >= 2 && !mbar_wait(&sm.acc_empty[i & 1], ((i >> 1) - 1) & 1, p.wait_polls)) { ok = false; break; }
        fence_after();
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const unsigned s = it % STAGES;
          if (!mbar_wait(&sm.full[s], (it / STAGES) & 1, p.wait_polls)) { ok = false; break; }
          fence_after();
          const uint64_t dw = desc_sw128(sm.stage[s].w), da = desc_sw128(sm.stage[s].a);
#pragma unroll
          for (int k = 0; k < KB / 32; ++k) multiply<CTAS>(acc, dw + 2 * k, da + 2 * k, idesc, kb > 0 || k > 0 ? 1u : 0u);
          commit_all<CTAS>(&sm.empty[s]);
        }
        if (ok) commit_all<CTAS>(&sm.acc_full[i & 1]);
      }
      // nothing in flight when the TMEM is given back
      if constexpr (CTAS == 1) commit(&sm.drain);
      else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(&sm.drain)) : "memory");
      if (!mbar_wait(&sm.drain, 0, WAIT_POLLS)) ok = false;
    }
    __syncwarp();
  } else {
    const int half = warp < 6 ? 0 : BT / 2;
    const uint32_t mine = tmem + ((uint32_t)(32 * (warp % 4)) << 16) + half;
    unsigned i = 0;
    for (long long t = first; walk.find(p, sm.groups, tiles_n, t, row0, n_tile); t += step, ++i) {
      const int n = (CTAS * n_tile + rank) * CH + 32 * (warp % 4) + lane, rows = min(walk.end - row0 - half, BT / 2);
      const bool real = n < p.N;
      const float sb = real ? __ldg(p.scale_b + (long long)walk.g * p.sb_group + (long long)n * p.sb_stride) : 0.0f;
      const float bias = real ? bias_at(p, (long long)walk.g * p.bias_group + n) : 0.0f;
      const float scale = row_scales<(BT < 64 ? BT / 2 : 32)>(p, row0 + half, rows);
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.acc_full[i & 1], (i >> 1) & 1, p.wait_polls));
      if (!ok) break;
      fence_after();
      write_rows<OUT, BT / 2>(p, mine + (i & 1) * BT, nk > 0, row0 + half, rows, n, real, sb, bias, scale);
      fence_before();
      __syncwarp();
      // (relaxed: the accumulator's values are in registers; a release would wait for the tile's stores to reach memory)
      if (lane == 0) {
        if constexpr (CTAS == 1)
          asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&sm.acc_empty[i & 1])) : "memory");
        else
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(first_cta<CTAS>(&sm.acc_empty[i & 1])) : "memory");
      }
    }
    if (ok && p.zero_rest)
      zero_rows<OUT>(p, sm.groups[p.E - 1].end + (int)blockIdx.x, (int)gridDim.x, 0, p.N, threadIdx.x - 64, WORKER_THREADS - 64);
  }
  if (!ok) atomicAdd(p.status, 1);
  fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) {
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    fence_after();
    if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(W::COLS));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(W::COLS));
  }
}
template <int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(WORKER_THREADS, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Int8Params p) {
  int8_worker<2, 256, OUT>(map_w, map_a, p);
}
template <int BT, int OUT>
__global__ void __launch_bounds__(WORKER_THREADS, 1)
    int8_single_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Int8Params p) {
  int8_worker<1, BT, OUT>(map_w, map_a, p);
}

// Rows of any alignment -> rows of `pitch` bytes (a multiple of 16) that TMA can read. The bytes behind K are not read.
struct Repack {
  const int8_t* src;
  int8_t* dst;
  long long ld, group_stride, rows_per_group, rows;
};
__global__ void __launch_bounds__(256) repack_kernel(const __grid_constant__ Repack r0, const __grid_constant__ Repack r1, int K, long long pitch) {
  dependent_launch_wait();
  dependent_launch_next();
  for (long long i = blockIdx.x; i < r0.rows + r1.rows; i += gridDim.x) {
    const bool second = i >= r0.rows;
    const Repack& r = second ? r1 : r0;
    const long long row = second ? i - r0.rows : i;
    const int8_t* s = r.src + row / r.rows_per_group * r.group_stride + row % r.rows_per_group * r.ld;
    int8_t* d = r.dst + row * pitch;
    // 16 bytes a thread: the five aligned words around them, shifted (the first and last word of a row byte by byte, so that
    // nothing outside the row is read)
    const unsigned shift = 8 * (unsigned)(reinterpret_cast<uintptr_t>(s) & 3);
    for (int k = threadIdx.x * 16; k < K; k += 4096) {
      uint32_t v[4];
      if (k >= 4 && k + 20 <= K) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(s + k - (shift >> 3));
        uint32_t a[5];
#pragma unroll
        for (int q = 0; q < 5; ++q) a[q] = q < 4 || shift ? __ldg(w + q) : 0u;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = __funnelshift_r(a[q], a[q + 1], shift);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (k + 4 * q + b < K) v[q] |= (uint32_t)(uint8_t)__ldg(s + k + 4 * q + b) << (8 * b);
        }
      }
      *reinterpret_cast<uint4*>(d + k) = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

// ---- host
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static std::atomic<EncodeFn> cached{nullptr};
  EncodeFn fn = cached.load(std::memory_order_acquire);
  if (fn) return fn;
  void* entry = nullptr;
  cudaDriverEntryPointQueryResult found;
  if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &found) != cudaSuccess ||
      found != cudaDriverEntryPointSuccess || !entry)
    return nullptr;
  fn = reinterpret_cast<EncodeFn>(entry);
  cached.store(fn, std::memory_order_release);
  return fn;
}
// A map of bytes [groups][rows][K] with boxes of box_rows rows and 128 bytes, 128-byte swizzle, zeros outside.
cudaError_t byte_map(CUtensorMap* map, const void* base, int K, long long rows, long long ld, int groups, long long group_stride,
                     int box_rows, bool three) {
  const EncodeFn fn = encoder();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)group_stride};
  const cuuint32_t box[3] = {KB, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, three ? 3 : 2, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
// TMA reads rows in place when every row starts on 16 bytes and the strides are below 2^40.
bool in_place(const void* base, long long ld, long long rows, long long group_stride, int groups) {
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  if (rows > 1 && ((ld & 15) || ld >= (1ll << 40))) return false;
  return groups <= 1 || (group_stride > 0 && !(group_stride & 15) && group_stride < (1ll << 40));
}
long long pitch_of(int K) { return ((long long)K + 127) / 128 * 128; }

int sms() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Shared memory of a kernel beyond the default, asked for once per device (1 us of every call otherwise).
struct SmemLimit {
  std::atomic<unsigned long long> done{0};
  cudaError_t set(const void* kern, size_t bytes) {
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return err;
  }
};

struct Maps { CUtensorMap w, a; };

template <int BT, int OUT>
cudaError_t launch_tile(const Int8Params& p, const Maps& m, int parts, unsigned tiles_t, cudaStream_t st) {
  auto kern = int8_tile_kernel<BT, OUT>;
  constexpr size_t SMEM = sizeof(SmemTile<BT>) + 1024;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static SmemLimit limit;
  const cudaError_t err = limit.set(reinterpret_cast<const void*>(kern), SMEM);
  if (err != cudaSuccess) return err;
  return launch_dependent_cluster(kern, dim3((unsigned)(p.tiles_n * parts), tiles_t), TILE_THREADS, SMEM, (unsigned)parts, st, m.w, m.a, p);
}
// Persistent workers on `tiles` tiles (at most).
template <int CTAS, int BT, int OUT>
cudaError_t launch_worker(const Int8Params& p, const Maps& m, long long tiles, cudaStream_t st) {
  void (*kern)(CUtensorMap, CUtensorMap, Int8Params);
  if constexpr (CTAS == 2) kern = int8_pair_kernel<OUT>;
  else kern = int8_single_kernel<BT, OUT>;
  constexpr size_t MOST = sizeof(typename Worker<CTAS, BT>::Smem) + 1024 + sizeof(GroupTable) * MMB200_MAX_GROUPS;
  static_assert(MOST <= 232448, "shared memory of a CTA");
  static SmemLimit limit;
  const cudaError_t err = limit.set(reinterpret_cast<const void*>(kern), MOST);
  if (err != cudaSuccess) return err;
  const long long workers = sms() / CTAS;
  return launch_dependent(kern, dim3((unsigned)(CTAS * (tiles < workers ? tiles : workers))), WORKER_THREADS,
                          Worker<CTAS, BT>::bytes(p), st, m.w, m.a, p);
}
template <int CTAS, int BT>
cudaError_t launch_worker_out(const Int8Params& p, const Maps& m, long long tiles, cudaStream_t st) {
  switch (p.out_dtype) {
    case MMB200_OUT_F32: return launch_worker<CTAS, BT, MMB200_OUT_F32>(p, m, tiles, st);
    case MMB200_OUT_BF16: return launch_worker<CTAS, BT, MMB200_OUT_BF16>(p, m, tiles, st);
    default: return launch_worker<CTAS, BT, MMB200_OUT_F16>(p, m, tiles, st);
  }
}
template <int BT>
cudaError_t launch_out(const Int8Params& p, const Maps& m, int parts, unsigned tiles_t, cudaStream_t st) {
  switch (p.out_dtype) {
    case MMB200_OUT_F32: return launch_tile<BT, MMB200_OUT_F32>(p, m, parts, tiles_t, st);
    case MMB200_OUT_BF16: return launch_tile<BT, MMB200_OUT_BF16>(p, m, parts, tiles_t, st);
    default: return launch_tile<BT, MMB200_OUT_F16>(p, m, parts, tiles_t, st);
  }
}

// Kernel, rows of a tile and parts of K by estimated time, in microseconds. A CTA takes TAU per 128 bytes of K and tile (MMAs of
// 128 channels take about 120 cycles up to 128 rows); all of them together get L2_RATE out of the caches and HBM_RATE out of
// memory; the slowest of the three counts, and a part of the first (REST), as they overlap only in part. START and the output of
// the last tile (OUT per row) come on top, the cluster's sum (SUM, and PART and SUM_ROW each) and every further wave of one-tile
// CTAs (WAVE). Two one-tile CTAs on an SM take SHARE times as long as one; memory is up to SPARE slower with few CTAs. Measured
// on whole calls, replayed from a graph on three sets of operands in turn (so weights below about 40 MB came from L2): 117 shapes of 1
// to 2048 rows, 512 to 24576 channels, K from 512 to 28672; the choice was within 5 % of the best of all of them for 102, within
// 15 % for all.
enum Kind { TILE, SINGLE, PAIR };
struct Choice { Kind kind; int rows, parts; };
long long most_row_tiles(const Int8Params& p, int rows) {               // of all groups: every one may end in a partial tile
  return p.offs ? (long long)p.T / rows + (p.E < p.T ? p.E : p.T) : ((long long)p.T + rows - 1) / rows;
}
Choice choose(const Int8Params& p) {
  constexpr double L2_RATE = 14e6, HBM_RATE = 6.1e6, OUT = 0.011, SUM = 1.8, PART = 0.1, SUM_ROW = 0.02;
  constexpr double WAVE = 2.0, REST = 0.15, SHARE = 1.6, SPARE = 0.1;
  const long long n_sm = sms(), used = p.E < p.T ? p.E : p.T;             // groups with rows, at most
  const double hbm = ((double)used * p.N + p.T) * p.K / HBM_RATE;
  Choice best{TILE, 16, 1};
  double least = 1e30;
  auto consider = [&](Kind kind, int rows, int parts, double start, double tau) {
    if (kind == TILE && most_row_tiles(p, rows) > 65535) return;          // grid y
    const int ctas_per_tile = kind == PAIR ? 2 : 1, occupancy = kind == TILE ? 2 : 1;
    const long long tiles_n = ((long long)p.N + CH * ctas_per_tile - 1) / (CH * ctas_per_tile);
    // every group has a tile, and ends in one that is half full on average
    const double ragged = (double)p.T / rows + 0.5 * used;
    const double tiles_t = !p.offs ? (double)(((long long)p.T + rows - 1) / rows) : ragged > used ? ragged : (double)used;
    const double tiles = tiles_t * tiles_n, workers = (double)(n_sm / ctas_per_tile);
    auto waves = [](double n, double at_once) { return n <= at_once ? 1.0 : (double)(long long)(n / at_once + 0.999); };
    // rows that a tile copies: its own, a one-tile CTA all
    const double copied = kind == TILE ? rows : (double)p.T / tiles_t + (p.T > 64 ? 32 : 0);
    const double l2 = tiles * p.k_blocks * KB * (CH * ctas_per_tile + copied) / L2_RATE;
    const double ctas = tiles * parts;
    double turns = waves(ctas, workers);                                 // of an SM's tensor pipe
    if (kind == TILE) {                                                  // two CTAs on an SM overlap
      const double rounds = waves(ctas, 2.0 * n_sm), rest = ctas - (rounds - 1.0) * 2.0 * n_sm;
      turns = (rounds - 1.0) * SHARE + (rest <= n_sm ? 1.0 : SHARE);
    }
    const double mma = tau * p.k_blocks / parts * turns;
    double t = mma > l2 ? mma : l2;
    const double memory = hbm * (ctas < 2.0 * n_sm ? 1.0 + SPARE * (1.0 - ctas / (2.0 * n_sm)) : 1.0);
    t = t > memory ? t : memory;
    t += REST * mma + start + OUT * rows + (parts > 1 ? SUM + PART * parts + SUM_ROW * rows : 0.0);
    if (kind == TILE) t += WAVE * (waves(tiles * parts, workers * occupancy) - 1.0);
    if (parts > 1 && tiles * parts > 2.0 * n_sm) return;                 // clusters that wait for room cost more than they save
    if (t < least) {
      least = t;
      best = Choice{kind, rows, parts};
    }
  };
  for (int parts = 1; parts <= 8 && parts <= (p.k_blocks > 1 ? p.k_blocks : 1); parts *= 2) {
    consider(TILE, 16, parts, 1.4, 0.25);
    consider(TILE, 32, parts, 1.4, 0.25);
    consider(TILE, 64, parts, 1.4, 0.26);
  }
  consider(SINGLE, 64, 1, 2.6, 0.27);
  consider(SINGLE, 128, 1, 2.6, 0.28);
  consider(SINGLE, 256, 1, 2.6, 0.40);
  consider(PAIR, 256, 1, 3.2, 0.34);
  return best;
}

}  // namespace

cudaError_t int8_status_words(int** words) {
  static std::atomic<int*> cached[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev >= 0 && dev < 64 && (*words = cached[dev].load(std::memory_order_acquire)) != nullptr) return cudaSuccess;
  err = cudaGetSymbolAddress(reinterpret_cast<void**>(words), g_int8_status);
  if (err == cudaSuccess && dev >= 0 && dev < 64) cached[dev].store(*words, std::memory_order_release);
  return err;
}

size_t int8_workspace_bytes(const Int8Params& p) {
  size_t n = 0;
  if (p.K <= 0) return 0;
  if (!in_place(p.a, p.lda, p.T, 0, 1)) n += (size_t)p.T * pitch_of(p.K);
  if (!in_place(p.w, p.ldw, p.N, p.gsw, p.E)) n += (size_t)p.E * p.N * pitch_of(p.K);
  return n;
}

int int8_kernel_for(const Int8Params& p_in) {
  Int8Params p = p_in;
  p.k_blocks = (p.K + KB - 1) / KB;
  const Choice c = choose(p);
  return c.kind << 16 | c.rows << 4 | c.parts;
}

cudaError_t launch_int8(const Int8Params& p_in, void* workspace, cudaStream_t st, int* launches) {
  Int8Params p = p_in;
  staged_wait_limits(&p.wait_polls, &p.announce_extra);
  cudaError_t err = p.status ? cudaSuccess : int8_status_words(&p.status);
  if (err != cudaSuccess) return err;
  int8_t* ws = static_cast<int8_t*>(workspace);
  if (p.K > 0) {
    const long long pitch = pitch_of(p.K);
    Repack r[2];
    std::memset(r, 0, sizeof(r));
    r[0].rows_per_group = r[1].rows_per_group = 1;
    if (!in_place(p.a, p.lda, p.T, 0, 1)) {
      r[0] = Repack{p.a, ws, p.lda, 0, p.T, p.T};
      p.a = ws;
      p.lda = pitch;
      ws += (size_t)p.T * pitch;
    }
    if (!in_place(p.w, p.ldw, p.N, p.gsw, p.E)) {
      r[1] = Repack{p.w, ws, p.ldw, p.gsw, p.N, (long long)p.E * p.N};
      p.w = ws;
      p.ldw = pitch;
      p.gsw = pitch * p.N;
    }
    const long long rows = r[0].rows + r[1].rows, most = 16ll * sms();
    if (rows) {
      err = launch_dependent(repack_kernel, dim3((unsigned)(rows < most ? rows : most)), 256, 0, st, r[0], r[1], p.K, pitch);
      if (err != cudaSuccess) return err;
      *launches += 1;
    }
  }
  p.k_blocks = (p.K + KB - 1) / KB;
  p.tiles_n = (p.N + CH - 1) / CH;
  const Choice best = choose(p);
  const int bt = best.rows;
  const long long tiles_t = most_row_tiles(p, bt);
  Maps m;
  std::memset(&m, 0, sizeof(m));
  if (p.K > 0) {
    // (a single row's stride is never used, but the map wants a multiple of 16)
    const long long ldw = p.N > 1 ? p.ldw : pitch_of(p.K), lda = p.T > 1 ? p.lda : pitch_of(p.K);
    err = byte_map(&m.w, p.w, p.K, p.N, ldw, p.E, p.E > 1 ? p.gsw : pitch_of(p.K), CH, true);
    if (err == cudaSuccess) err = byte_map(&m.a, p.a, p.K, p.T, lda, 1, 0, bt < 64 ? bt : 64, false);
    if (err != cudaSuccess) return err;
  }
  const long long tiles = tiles_t * p.tiles_n;
  if (best.kind == PAIR) {
    err = launch_worker_out<2, 256>(p, m, tiles_t * ((p.N + 2 * CH - 1) / (2 * CH)), st);
  } else if (best.kind == SINGLE) {
    if (bt == 64) err = launch_worker_out<1, 64>(p, m, tiles, st);
    else if (bt == 128) err = launch_worker_out<1, 128>(p, m, tiles, st);
    else err = launch_worker_out<1, 256>(p, m, tiles, st);
  } else {
    if (bt == 16) err = launch_out<16>(p, m, best.parts, (unsigned)tiles_t, st);
    else if (bt == 32) err = launch_out<32>(p, m, best.parts, (unsigned)tiles_t, st);
    else err = launch_out<64>(p, m, best.parts, (unsigned)tiles_t, st);
  }
  if (err != cudaSuccess) return err;
  *launches += 1;
  return cudaSuccess;
}

}  // namespace mmb
