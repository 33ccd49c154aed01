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
//   codes   [4 strips of 16 rows][2 blocks of 64 k][32 lanes][4 words]: a lane's 16 bytes are what it feeds to four
//           m16n8k16 products.  Lane (g, t) = (lane / 4, lane % 4), word j = 2 q + h: rows g and g + 8 of the strip, k =
//           32 q + 8 t + 4 h + 0 .. 3 of the block.  Nibble i and i + 4 of the word are register i of the A fragment: rows
//           g, g + 8, g, g + 8; k + 0, 1 for i < 2 and k + 2, 3 for the others.  So 8 consecutive k of x are one 16-byte piece of a
//           lane's B fragments, and no product reaches over a group of 32.
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
// Launchers: one for few rows of x, one for many (each takes any number).
cudaError_t launch_w4_few(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st);
cudaError_t launch_w4_many(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st);

// ---------------------------------------------------------------- clusters
T2W_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
T2W_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
T2W_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
T2W_DEV float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
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
// magic + zero in both halves
template <bool HALF>
T2W_DEV uint32_t w4_zero(uint32_t z) {
  return W4Num<HALF>::kMagic + z * 0x00010001u;
}
// the four registers of a word: code - zero, with zlo for rows g and zhi for rows g + 8
template <bool HALF>
T2W_DEV void w4_widen(uint32_t w, uint32_t zlo, uint32_t zhi, uint32_t (&a)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "r"(0x000f000fu), "r"(W4Num<HALF>::kMagic));
    a[i] = W4Num<HALF>::sub(v, (i & 1) ? zhi : zlo);
  }
}
T2W_DEV float w4_scale(uint16_t v, int half) { return half ? W4Num<true>::to_float(v) : W4Num<false>::to_float(v); }

// ---------------------------------------------------------------- activations (fp32, relative error of a few 2^-22)
// y sigmoid(y); the quotient is kept off __fdividef, whose result is 0 for divisors above 2^126: y / (1 + e^-y) is that
// small there that fp32 holds it as a subnormal or 0, and +-inf and NaN go as in the formula
T2W_DEV float w4_sigmoid_mul(float y, float s) { return y / (1.f + __expf(-s)); }
T2W_DEV float w4_act(float g, int act) {
  if (act == T2W_ACT_SILU) return w4_sigmoid_mul(g, g);
  // GELU in its tanh form: g (1 + tanh t) / 2 = g sigmoid(2 t), t = sqrt(2 / pi) (g + 0.044715 g^3)
  return w4_sigmoid_mul(g, 1.5957691216057308f * (g + 0.044715f * g * g * g));
}

}  // namespace t2w
