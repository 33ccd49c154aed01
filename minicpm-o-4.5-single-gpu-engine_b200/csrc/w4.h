// What the kernels of the products with 4-bit weights share: how a weight lies in memory and how codes become 16-bit
// operands.
//
// A weight is W[n][k] = (code - zero) * scale: code 0 .. 15, zero 8 unless each group has its own (0 .. 15), one scale
// (bf16 or fp16) for each row and `group` (32, 64 or 128) consecutive k.
//
// Sums are taken over the whole numbers (code - zero), which 16-bit operands hold exactly, and a group's sum is multiplied by
// its scale in fp32 after it: no weight is ever rounded, and the scale costs a multiplication for each group and output
// instead of one for each weight.
//
// Layout: a header of 128 bytes (int32 status, the rest zero), then tiles of 64 rows x 128 k, [row block][k tile], each
// one contiguous piece that one bulk copy brings:
//   codes   [4 strips of 16 rows][2 blocks of 64 k][32 lanes][4 words]: a word is a lane's A fragment of an m16n8k16 product
//           of 16 k, j of the block.  Lane (g, t) = (lane / 4, lane % 4) has rows g and g + 8 of the strip and k = 16 j + 4 t + 0 .. 3:
//           nibbles i and i + 4 are register i, rows g, g + 8, g, g + 8; k + 0, 1 for i < 2 and k + 2, 3 for the others.  So
//           a lane's part of x is 8 consecutive bytes, widened registers are what tcgen05.st 16x256b takes, and no product reaches
//           over a group.
//   scales  [128 / group][64] 16-bit, then zeros [128 / group][64] bytes where there are any: place g * 8 + strip * 2 + half
//           for row strip * 16 + half * 8 + g, so that a lane finds the eight rows it holds in one piece.
// Rows and k past the weight's are codes that equal their zero, with scale 0.  A gated pair (gate, up) is one weight whose
// rows alternate by eights: rows 0 .. 7 of a strip are eight gate rows, 8 .. 15 the up rows of the same outputs, so
// that one thread of an m16n8 product has both.
#pragma once

#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace t2w {

constexpr int kW4Rows = 64, kW4K = 128, kW4Header = 128, kW4Codes = kW4Rows * kW4K / 2;

__host__ __device__ constexpr int w4_tile_bytes(int group, bool zeros) {
  return kW4Codes + (kW4K / group) * kW4Rows * (zeros ? 3 : 2);
}
// place of row r (0 .. 63) among a tile's scales and zeros
__host__ __device__ constexpr int w4_place(int r) { return (r & 7) * 8 + (r >> 4) * 2 + ((r >> 3) & 1); }
// packed rows of a weight of n rows (gated: n outputs, two rows each)
__host__ __device__ constexpr int64_t w4_rows(int64_t n, bool gated) { return gated ? (n + 7) / 8 * 16 : n; }

// One product with a 4-bit weight, as the launchers take it.
struct W4Dev {
  const uint8_t* tiles;  // behind the header
  int* status;
  const void* x;  // [rows][k], 16 bits
  int64_t x_ld;
  int rows, k, n;  // n: outputs of a row
  int tiles_k;     // k tiles of 128
  int blocks;      // row blocks of 64
  int scale_half;  // scales are fp16
  int act;         // gated: T2W_ACT_*
  const void* bias;
  const void* residual;
  int64_t res_ld;
  void* out;  // [rows][n] contiguous
};
// How many clusters of `split` blocks of a kernel are resident at once: clusters lie within a GPC each, so that it is fewer than the
// blocks without clusters are (of 148 one an SM, 132 in clusters of 4, 120 in clusters of 8).  `cache` keeps the answer for
// each device and split (1, 2, 4, 8); 0 is none yet.
struct ClusterRoom {
  std::atomic<int> at[16][4] = {};
};
template <class K>
int cluster_room(K* kernel, int split, int threads, int smem, ClusterRoom& cache) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::atomic<int>* kept = dev >= 0 && dev < 16 ? &cache.at[dev][split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3] : nullptr;
  if (kept && kept->load(std::memory_order_relaxed) > 0) return kept->load(std::memory_order_relaxed);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();  // (a shape that does not fit is not an error of the call)
    return 0;
  }
  if (kept) kept->store(n, std::memory_order_relaxed);
  return n;
}

// Launchers: one for few rows of x, one for many (each takes any number).
cudaError_t launch_w4_few(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st);
cudaError_t launch_w4_many(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st);

// ---------------------------------------------------------------- waiting
// mbar_wait without its look at %globaltimer, which costs about a microsecond: these kernels hand over every few hundred
// clocks, and most waits are not met at once.  The limit is in SM clocks.
T2W_DEV bool w4_wait(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t at = smem_u32(bar);
  if (mbar_try_wait(at, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(at, parity)) return true;
    if ((i & 63u) == 0 && clock64() - t0 > kWaitLimitCycles) {
      atomicExch(err, T2W_ERR_TIMEOUT);
      return false;
    }
  }
}

// The same by a whole warp, with one answer; `ready` is what a look at the barrier, taken ahead of other work, has said.  (A wait
// for a barrier that is ready costs about 150 clocks, a look whose answer is not needed at once next to none.)
T2W_DEV bool w4_wait_warp(uint64_t* bar, uint32_t parity, int* err, bool ready = false) {
  if (__all_sync(0xffffffffu, ready)) return true;
  return __all_sync(0xffffffffu, w4_wait(bar, parity, err));
}

// ---------------------------------------------------------------- clusters
T2W_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
T2W_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
T2W_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
T2W_DEV uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
T2W_DEV float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
// The sum over the cluster's blocks (1, 2, 4 or 8), in their order, of four values at one place of each; four reads are under
// way at once.
T2W_DEV float4 cluster_sum4(uint32_t addr, int split) {
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int s0 = 0; s0 < split; s0 += 4) {
    float4 v[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) v[s] = s0 + s < split ? ld_cluster4(cluster_addr(addr, s0 + s)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      r.x += v[s].x;
      r.y += v[s].y;
      r.z += v[s].z;
      r.w += v[s].w;
    }
  }
  return r;
}

// ---------------------------------------------------------------- codes to operands
template <bool HALF>
struct W4Num;
template <>
struct W4Num<false> {
  // 128 + code: bf16 numbers from 128 to 256 are whole, so a code's bits become its value by being put into them
  static constexpr uint32_t kMagic = 0x43004300u;
  static T2W_DEV uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static T2W_DEV float to_float(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static T2W_DEV uint16_t from_float(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};
template <>
struct W4Num<true> {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 + code
  static T2W_DEV uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static T2W_DEV float to_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static T2W_DEV uint16_t from_float(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
// What widening takes off for the zeros of rows g and g + 8 (in both halves of a register).
template <bool HALF>
T2W_DEV uint32_t w4_zero(uint32_t z) {
  return W4Num<HALF>::kMagic + z * 0x00010001u;
}
template <bool HALF>
T2W_DEV uint32_t w4_zero_hi(uint32_t z) {
  return HALF ? 0xd400d400u + z * 0x00100010u /* -(64 + zero) */ : w4_zero<HALF>(z);
}
// The four registers of a word: code - zero, with zlo for rows g and zhi (of w4_zero_hi) for rows g + 8.  A code's bits are
// put under an exponent that makes its steps whole (a long-known way to turn few bits into a float without a conversion).
// fp16 has room for two codes side by side: one 16 times too large is brought back by the multiplication-addition that takes
// its zero off (exact: 6 bits and a sign), which saves two of three shifts; bf16 has not.
template <bool HALF>
T2W_DEV void w4_widen(uint32_t w, uint32_t zlo, uint32_t zhi, uint32_t (&a)[4]) {
  if constexpr (HALF) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t u = w >> (4 * i), sixteenth = 0x2c002c00u;
      uint32_t lo, hi;
      asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(lo) : "r"(u), "r"(0x000f000fu), "r"(W4Num<HALF>::kMagic));
      asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(hi) : "r"(u), "r"(0x00f000f0u), "r"(W4Num<HALF>::kMagic));
      a[i] = W4Num<HALF>::sub(lo, zlo);
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(a[i + 1]) : "r"(hi), "r"(sixteenth), "r"(zhi));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t v;
      asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "r"(0x000f000fu), "r"(W4Num<HALF>::kMagic));
      a[i] = W4Num<HALF>::sub(v, (i & 1) ? zhi : zlo);
    }
  }
}

// Four consecutive outputs of a row, as far as there are any: one store where they lie on 8 bytes.
T2W_DEV void w4_store4(uint16_t* out, const uint16_t (&v)[4], int count) {
  if (count >= 4 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
    *reinterpret_cast<uint2*>(out) = make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) out[i] = v[i];
  }
}
T2W_DEV float w4_scale(uint16_t v, int half) { return half ? W4Num<true>::to_float(v) : W4Num<false>::to_float(v); }

// ---------------------------------------------------------------- activations
// y sigmoid(s), from e = e^-|s|, which is at most 1 and so never too large: y / (1 + e), times e where s < 0.  (y / (1 + e^-s)
// is 0 below s = -88.7, where e^-s passes fp32, and y e^s is not yet under bf16's least numbers.)  Relative error (8 + 1.2 |s|)
// 2^-23 (__expf is off by 2 + 1.2 |s| steps); from s = -87.3 down e is subnormal, which adds steps of 2^-149 |y|.  Infinities
// and NaN go as in the formula.
T2W_DEV float w4_sigmoid_mul(float y, float s) {
  const float e = __expf(-fabsf(s));
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return y * (s < 0.f ? e * r : r);
}
T2W_DEV float w4_act(float g, int act) {
  if (act == T2W_ACT_SILU) return w4_sigmoid_mul(g, g);
  // GELU in its tanh form: g (1 + tanh t) / 2 = g sigmoid(2 t), t = sqrt(2 / pi) (g + 0.044715 g^3)
  return w4_sigmoid_mul(g, 1.5957691216057308f * (g + 0.044715f * g * g * g));
}

// Outputs n .. n + 3 of row m from their sums (gated: gate and up), as far as n < p.n.
template <bool HALF, bool GATED>
T2W_DEV void w4_finish4(const W4Dev& p, int m, int64_t n, float4 sum, float4 up) {
  float v[4] = {sum.x, sum.y, sum.z, sum.w};
  const float u[4] = {up.x, up.y, up.z, up.w};
  const int count = (int)min((int64_t)4, p.n - n);
  uint16_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (GATED) {
      v[i] = w4_act(v[i], p.act) * u[i];
    } else if (i < count) {
      if (p.bias) v[i] += W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.bias)[n + i]);
      if (p.residual) v[i] += W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.residual)[(int64_t)m * p.res_ld + n + i]);
    }
    out[i] = W4Num<HALF>::from_float(v[i]);
  }
  w4_store4(static_cast<uint16_t*>(p.out) + (int64_t)m * p.n + n, out, count);
}

}  // namespace t2w
