// Products with 4-bit weights for few rows of x: y[m][n] = sum_k x[m][k] W[n][k] (+ bias, + residual, or a gated pair's
// activation and product), bound by the weights' bytes.
//
// A block of 8 warps has 64 rows of W and a share of k; each of its warps streams every eighth tile (64 x 128, one bulk
// copy into a ring of its own) through m16n8k16 products, with W as the 16-row operand and up to 8 NT rows of x as the
// columns.  Codes widen in registers to whole numbers (w4.h), a group's sum is scaled in fp32.  The first copies are
// issued before the kernel waits for the one before it in the stream: weights do not depend on it, so their way from HBM is
// hidden behind its end.  Sums of the 8 warps are joined through shared memory, those of a cluster's blocks (k split over
// up to 8) through distributed shared memory: no workspace, no atomics, the same order in every call.
#include "common.cuh"
#include "kernels.h"
#include "w4.h"

namespace t2w {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kMaxStages = 3;
constexpr int kPitch = 68;  // of a column of 64 sums: on 16 bytes, and 8 columns apart in the banks

template <bool HALF>
T2W_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int NT>
struct XFrag {
  uint2 v[NT][8];  // [8 rows of x][16 k]: 4 consecutive k each
};

// A lane's pieces of x for a k tile: row m0 + 8 nt + g, k = 128 tile + 16 j + 4 t; zeros past either end (k is a multiple
// of 32, so a piece lies inside or outside).
template <int NT>
T2W_DEV void load_x(XFrag<NT>& f, const W4Dev& p, int m0, int tile, int g, int t) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int m = m0 + 8 * nt + g, k0 = tile * kW4K + 4 * t;
    const uint16_t* row = static_cast<const uint16_t*>(p.x) + (int64_t)m * p.x_ld + k0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f.v[nt][j] = (m < p.rows && k0 + 16 * j < p.k) ? *reinterpret_cast<const uint2*>(row + 16 * j) : make_uint2(0, 0);
  }
}

template <bool HALF, int NT, int G, bool ZEROS, bool GATED>
__global__ void __launch_bounds__(kThreads, 2) k_w4_few(const W4Dev p, int split, int stages) {
  constexpr int kTile = w4_tile_bytes(G, ZEROS), kGroups = kW4K / G, kCols = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);  // [warp][stage]
  float* part = reinterpret_cast<float*>(smem + kWarps * kMaxStages * 8);  // the block's sums [column of x][kPitch]
  constexpr int kPart = (kWarps * kMaxStages * 8 + kCols * kPitch * 4 + 127) / 128 * 128;
  uint8_t* ring = smem + kPart + warp * stages * kTile;
  uint64_t* full = bars + warp * kMaxStages;

  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int rb = blockIdx.x / split, m0 = blockIdx.y * kCols;
  const int k_end = (int)((int64_t)p.tiles_k * (rank + 1) / split);
  const int first = (int)((int64_t)p.tiles_k * rank / split) + warp;
  int tile = first;
  const uint8_t* src = p.tiles + (int64_t)rb * p.tiles_k * kTile;
  if (lane == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    for (int s = 0; s < stages && tile + s * kWarps < k_end; ++s) {
      mbar_expect_tx(&full[s], kTile);
      bulk_load(ring + s * kTile, src + (int64_t)(tile + s * kWarps) * kTile, kTile, &full[s]);
    }
  }
  __syncwarp();
  pdl_wait();
  pdl_launch();

  float acc[4][NT][4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][nt][i] = 0.f;
  XFrag<NT> x;
  if (tile < k_end) load_x<NT>(x, p, m0, tile, g, t);
  int stage = 0;
  uint32_t phase = 0;
  for (; tile < k_end; tile += kWarps) {
    if (!w4_wait_warp(&full[stage], phase, p.status)) {
      // The status tells that the outputs are void.  What else is under way lands (or is given up) before the ring is used.
      for (int i = 1; i < stages && tile + i * kWarps < k_end; ++i) {
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
        w4_wait(&full[stage], phase, p.status);
      }
      break;
    }
    const uint8_t* buf = ring + stage * kTile;
    alignas(16) uint16_t scale[kGroups][8];
    alignas(8) uint8_t zero[kGroups][8];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      *reinterpret_cast<uint4*>(scale[i]) = *reinterpret_cast<const uint4*>(buf + kW4Codes + i * 128 + g * 16);
      if constexpr (ZEROS)
        *reinterpret_cast<uint2*>(zero[i]) = *reinterpret_cast<const uint2*>(buf + kW4Codes + kGroups * 128 + i * 64 + g * 8);
    }
    if (NT > 1 && tile >= first + kWarps) load_x<NT>(x, p, m0, tile, g, t);  // (no registers to read ahead)
    const XFrag<NT> cur = x;
    if (NT == 1 && tile + kWarps < k_end) load_x<NT>(x, p, m0, tile + kWarps, g, t);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      uint4 code[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) code[kb] = reinterpret_cast<const uint4*>(buf)[(r * 2 + kb) * 32 + lane];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        float sum[NT][4] = {};
        const uint32_t zlo = w4_zero<HALF>(ZEROS ? zero[i][2 * r] : 8u), zhi = w4_zero<HALF>(ZEROS ? zero[i][2 * r + 1] : 8u);
#pragma unroll
        for (int s = 0; s < G / 16; ++s) {  // products of 16 k
          const int j = i * (G / 16) + s;
          const uint32_t w = (&code[j >> 2].x)[j & 3];
          uint32_t a[4];
          w4_widen<HALF>(w, zlo, zhi, a);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<HALF>(sum[nt], a, cur.v[nt][j].x, cur.v[nt][j].y);
        }
        const float slo = w4_scale(scale[i][2 * r], p.scale_half), shi = w4_scale(scale[i][2 * r + 1], p.scale_half);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[r][nt][0] = fmaf(slo, sum[nt][0], acc[r][nt][0]);
          acc[r][nt][1] = fmaf(slo, sum[nt][1], acc[r][nt][1]);
          acc[r][nt][2] = fmaf(shi, sum[nt][2], acc[r][nt][2]);
          acc[r][nt][3] = fmaf(shi, sum[nt][3], acc[r][nt][3]);
        }
      }
    }
    __syncwarp();  // the tile has been read: its place may be filled again
    if (lane == 0 && tile + stages * kWarps < k_end) {
      mbar_expect_tx(&full[stage], kTile);
      bulk_load(ring + stage * kTile, src + (int64_t)(tile + stages * kWarps) * kTile, kTile, &full[stage]);
    }
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }

  // The warps' sums [64][kCols] in the rings' place, once all copies are read.
  float* mine = reinterpret_cast<float*>(smem + kPart + warp * kCols * 64 * 4);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      *reinterpret_cast<float2*>(mine + (r * 16 + g) * kCols + nt * 8 + 2 * t) = make_float2(acc[r][nt][0], acc[r][nt][1]);
      *reinterpret_cast<float2*>(mine + (r * 16 + 8 + g) * kCols + nt * 8 + 2 * t) = make_float2(acc[r][nt][2], acc[r][nt][3]);
    }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem + kPart);
#pragma unroll
  for (int e = threadIdx.x; e < 64 * kCols; e += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += all[w * 64 * kCols + e];
    part[(e % kCols) * kPitch + e / kCols] = v;
  }
  if (split > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  // This block's share of the outputs, four along n to a thread.
  constexpr int kQuads = GATED ? 8 : 16;
  const int cols = min(kCols, p.rows - m0);
  const uint32_t base = smem_u32(part);
  for (int e = rank * (kQuads * kCols / split) + threadIdx.x; e < (rank + 1) * (kQuads * kCols / split); e += kThreads) {
    const int m = e / kQuads, o = e % kQuads * 4;
    const int64_t n = (int64_t)rb * (GATED ? 32 : 64) + o;
    if (m >= cols || n >= p.n) continue;
    const int at = m * kPitch + (GATED ? (o >> 3) * 16 + (o & 7) : o);
    float4 v, u = make_float4(0.f, 0.f, 0.f, 0.f);
    if (split > 1) {
      v = cluster_sum4(base + at * 4, split);
      if constexpr (GATED) u = cluster_sum4(base + at * 4 + 32, split);
    } else {
      v = *reinterpret_cast<const float4*>(part + at);
      if constexpr (GATED) u = *reinterpret_cast<const float4*>(part + at + 8);
    }
    w4_finish4<HALF, GATED>(p, m0 + m, n, v, u);
  }
  if (split > 1) {  // no block leaves while another reads its sums
    cluster_arrive();
    cluster_wait();
  }
}

template <bool HALF, int NT, int G, bool ZEROS, bool GATED>
cudaError_t launch(const W4Dev& p, cudaStream_t st) {
  constexpr int kTile = w4_tile_bytes(G, ZEROS), kCols = 8 * NT;
  constexpr int kPart = (kWarps * kMaxStages * 8 + kCols * kPitch * 4 + 127) / 128 * 128;
  const int chunks = (p.rows + kCols - 1) / kCols;
  int split = 1;
  while (split < 8 && (int64_t)p.blocks * chunks * split < num_sms() && p.tiles_k >= 2 * split) split *= 2;
  const int per_warp = ((p.tiles_k + split - 1) / split + kWarps - 1) / kWarps;
  const int stages = per_warp < kMaxStages ? per_warp : kMaxStages;
  int smem = kWarps * stages * kTile;
  if (smem < kWarps * kCols * 64 * 4) smem = kWarps * kCols * 64 * 4;
  smem += kPart;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = smem_attr_once(k_w4_few<HALF, NT, G, ZEROS, GATED>, kWarps * kMaxStages * kTile + kPart, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.blocks * split, chunks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, k_w4_few<HALF, NT, G, ZEROS, GATED>, p, split, stages);
}

template <bool HALF, int NT, int G, bool ZEROS>
cudaError_t pick_gated(const W4Dev& p, bool gated, cudaStream_t st) {
  return gated ? launch<HALF, NT, G, ZEROS, true>(p, st) : launch<HALF, NT, G, ZEROS, false>(p, st);
}
template <bool HALF, int NT, int G>
cudaError_t pick_zeros(const W4Dev& p, bool zeros, bool gated, cudaStream_t st) {
  return zeros ? pick_gated<HALF, NT, G, true>(p, gated, st) : pick_gated<HALF, NT, G, false>(p, gated, st);
}
template <bool HALF, int NT>
cudaError_t pick_group(const W4Dev& p, int group, bool zeros, bool gated, cudaStream_t st) {
  if (group == 32) return pick_zeros<HALF, NT, 32>(p, zeros, gated, st);
  if (group == 64) return pick_zeros<HALF, NT, 64>(p, zeros, gated, st);
  return pick_zeros<HALF, NT, 128>(p, zeros, gated, st);
}
template <bool HALF>
cudaError_t pick_cols(const W4Dev& p, int group, bool zeros, bool gated, cudaStream_t st) {
  return p.rows <= 8 ? pick_group<HALF, 1>(p, group, zeros, gated, st) : pick_group<HALF, 2>(p, group, zeros, gated, st);
}

}  // namespace

cudaError_t launch_w4_few(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st) {
  return half ? pick_cols<true>(p, group, zeros, gated, st) : pick_cols<false>(p, group, zeros, gated, st);
}

}  // namespace t2w
