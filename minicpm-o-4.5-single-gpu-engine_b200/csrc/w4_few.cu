// Products with 4-bit weights for few rows of x: y[m][n] = sum_k x[m][k] W[n][k] (+ bias, + residual, or a gated pair's
// activation and product).  The floor is the weights' bytes.  What bounds it is that 16 warps an SM fill no unit (1 x 4096 x 131072:
// 58 us, 4.7 TB/s, 59% of the issue slots in use; a warp's time is 16% issuing, 22% fixed latencies, 16% waiting for the half-rate
// integer pipe, 17% for its turn, 8% at barriers), and in small calls the ends: the fence before a cluster's barrier takes 22% of
// the warps' time in 1 x 4096 x 11008, gated.
//
// A cluster of 1, 2 or 4 blocks of 8 warps has a number of row blocks (64 rows of W), whose tiles (64 x 128) it shares out evenly,
// in order, to its warps.  A warp streams its tiles (one bulk copy each, into a ring of its own) through m16n8k16 products,
// with W as the 16-row operand and 8 rows of x as the columns: codes widen in registers to whole numbers (w4.h), a group's sum
// is scaled in fp32.  The first copies are issued before the kernel waits for the one before it in the stream: weights do not
// depend on it, so their way from HBM is hidden behind its end.
//
// Warps meet once, at the end: each leaves the sums of the one or two row blocks that its tiles were of, a block adds its warps'
// and sends them to the block of the cluster that finishes the row block (distributed shared memory), which adds those after
// the cluster's one barrier: no workspace, no atomics, the same order in every call.  (A meeting for each row block instead, k
// shared out to the warps: 20 us for 1 x 4096 x 11008, gated, of which 14 without any product; 14.1 now.  Sums read from the other
// blocks, which takes a second barrier before they may end: 4 us of 21.)
#include "common.cuh"
#include "kernels.h"
#include "w4.h"

#include <algorithm>

namespace t2w {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kStages = 2, kCols = 8;
constexpr int kSeg = kCols * 64 * 4;      // a warp's, or a block's, sums of a row block: [64][kCols]
constexpr int kMaxSplit = 4, kRows = 2;    // blocks of a cluster; row blocks of a pass for each of them
constexpr int kSlots = kMaxSplit > 2 * kRows ? kMaxSplit : 2 * kRows;  // parts that a block may be sent (see `slot`)
constexpr int kBars = kWarps * kStages * 8;

constexpr int few_smem(int tile) { return kBars + kWarps * kStages * tile + (kWarps * 2 + kSlots) * kSeg; }

// c = a b + d
template <bool HALF>
T2W_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float d0, float d1, float d2, float d3) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(d0), "f"(d1), "f"(d2), "f"(d3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(d0), "f"(d1), "f"(d2), "f"(d3));
}

struct XFrag {
  uint2 v[8];  // [16 k]: 4 consecutive k each
};

// A lane's pieces of x for a k tile, from the row's place: k = 128 tile + 16 j + 4 t; zeros past the end (k is a multiple of 32,
// so a piece lies inside or outside), where the weights are 0 but x may be anything.
T2W_DEV void load_x(XFrag& f, const uint16_t* row, int k, int tile, int t) {
  const int left = k - tile * kW4K - 4 * t;
  const uint2* from = reinterpret_cast<const uint2*>(row + tile * kW4K);
  if (left > 112) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = from[4 * j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = 16 * j < left ? from[4 * j] : make_uint2(0, 0);
  }
}

T2W_DEV void st_cluster4(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

template <bool HALF, int G, bool ZEROS, bool GATED>
__global__ void __launch_bounds__(kThreads, 2) k_w4_few(const W4Dev p, int log_split, int clusters) {
  constexpr int kTile = w4_tile_bytes(G, ZEROS), kGroups = kW4K / G;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int block_at[kMaxSplit + 1], warp_at[kWarps + 1];  // first tile of the cluster's blocks, of this block's warps
  __shared__ int block_row[kMaxSplit];                          // row block of block_at
  // (what is done once is kept short, with shifts for divisions: it is fetched from far away, a thousand clocks for 60 lines)
  const int split = 1 << log_split;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem) + warp * kStages;
  uint8_t* ring = smem + kBars + warp * kStages * kTile;
  float* segs = reinterpret_cast<float*>(smem + kBars + kWarps * kStages * kTile);  // [warp][2][64][kCols]
  float* parts = segs + kWarps * 2 * kSeg / 4;                                    // [slot][64][kCols]

  const int rank = split > 1 ? (int)cluster_rank() : 0, cluster = blockIdx.x >> log_split, m0 = blockIdx.y * kCols;
  const int T = p.tiles_k, me = rank * kWarps + warp;
  const int rb_begin = (int)((int64_t)p.blocks * cluster / clusters), rb_end = (int)((int64_t)p.blocks * (cluster + 1) / clusters);
  // Passes of up to `most` row blocks: a block's tiles are then of at most kRows + 1 of them, a warp's of two.
  const int most = kRows * split;
  auto first_of = [&](int tiles, int w) { return (int)((uint32_t)(tiles * w) >> (3 + log_split)); };  // (the product is under 2^31)
  // The copies run ahead over the passes: the next tile's place, and how many of this warp's are left in its pass.
  const uint8_t* copy_from = nullptr;
  int copy_left = 0, copy_rb = rb_begin;
  auto copy = [&](int stage) {
    while (copy_left == 0) {
      if (copy_rb >= rb_end) return;
      const int tiles = min(most, rb_end - copy_rb) * T, at = first_of(tiles, me);
      copy_left = first_of(tiles, me + 1) - at;
      copy_from = p.tiles + ((int64_t)copy_rb * T + at) * kTile;
      copy_rb += most;
    }
    mbar_expect_tx(&full[stage], kTile);
    bulk_load(ring + stage * kTile, copy_from, kTile, &full[stage]);
    copy_from += kTile;
    --copy_left;
  };
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    for (int s = 0; s < kStages; ++s) copy(s);
  }
  __syncwarp();
  if (split > 1) cluster_arrive();  // (waited for before another block's memory is written: it has to run by then)
  int count = min(most, rb_end - rb_begin), tiles = count * T, at = first_of(tiles, me), end = first_of(tiles, me + 1), kt = at % T;
  auto write_bounds = [&]() {
    if (threadIdx.x <= kWarps) warp_at[threadIdx.x] = first_of(tiles, rank * kWarps + threadIdx.x);
    if (threadIdx.x >= 32 && threadIdx.x <= 32 + split) {
      const int s = threadIdx.x - 32, first = first_of(tiles, s * kWarps);
      block_at[s] = first;
      if (s < split) block_row[s] = first / T;
    }
  };
  write_bounds();
  pdl_wait();
  // (lanes of columns that there are not read the last row: their sums are not used)
  const uint16_t* row = static_cast<const uint16_t*>(p.x) + (int64_t)min(m0 + g, p.rows - 1) * p.x_ld + 4 * t;
  XFrag x;
  if (at < end) load_x(x, row, p.k, kt, t);
  pdl_launch();

  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int rb0 = rb_begin; rb0 < rb_end;) {
    float acc[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][i] = 0.f;
    float* seg = segs + warp * 2 * (kSeg / 4);
    auto leave = [&]() {  // the sums so far
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        *reinterpret_cast<float2*>(seg + (r * 16 + g) * kCols + 2 * t) = make_float2(acc[r][0], acc[r][1]);
        *reinterpret_cast<float2*>(seg + (r * 16 + 8 + g) * kCols + 2 * t) = make_float2(acc[r][2], acc[r][3]);
      }
    };
    for (int i = at; i < end && ok; ++i) {
      if (!(ok = w4_wait_warp(&full[stage], phase, p.status))) {
        // The status tells that the outputs are void.  What else may be under way lands, or is given up.
        w4_wait(&full[stage ^ 1], stage ? phase ^ 1u : phase, p.status);
        break;
      }
      const uint8_t* buf = ring + stage * kTile;
      alignas(16) uint16_t raw[kGroups][8];
      float scale[kGroups][8];
      alignas(8) uint8_t zero[kGroups][8];
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        *reinterpret_cast<uint4*>(raw[j]) = *reinterpret_cast<const uint4*>(buf + kW4Codes + j * 128 + g * 16);
        if constexpr (ZEROS)
          *reinterpret_cast<uint2*>(zero[j]) = *reinterpret_cast<const uint2*>(buf + kW4Codes + kGroups * 128 + j * 64 + g * 8);
      }
      if (p.scale_half) {
#pragma unroll
        for (int j = 0; j < kGroups * 8; ++j) scale[j / 8][j % 8] = W4Num<true>::to_float(raw[j / 8][j % 8]);
      } else {
#pragma unroll
        for (int j = 0; j < kGroups * 8; ++j) scale[j / 8][j % 8] = W4Num<false>::to_float(raw[j / 8][j % 8]);
      }
      const bool last = kt + 1 == T;  // of its row block
      kt = last ? 0 : kt + 1;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint4 code[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) code[kb] = reinterpret_cast<const uint4*>(buf)[(r * 2 + kb) * 32 + lane];
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          float sum[4];
          const uint32_t zlo = w4_zero<HALF>(ZEROS ? zero[j][2 * r] : 8u), zhi = w4_zero_hi<HALF>(ZEROS ? zero[j][2 * r + 1] : 8u);
#pragma unroll
          for (int s = 0; s < G / 16; ++s) {  // products of 16 k
            const int k = j * (G / 16) + s;
            const uint32_t w = (&code[k >> 2].x)[k & 3];
            uint32_t a[4];
            w4_widen<HALF>(w, zlo, zhi, a);
            if (s == 0) mma16816<HALF>(sum, a, x.v[k].x, x.v[k].y, 0.f, 0.f, 0.f, 0.f);
            else mma16816<HALF>(sum, a, x.v[k].x, x.v[k].y, sum[0], sum[1], sum[2], sum[3]);
          }
          const float slo = scale[j][2 * r], shi = scale[j][2 * r + 1];
          acc[r][0] = fmaf(slo, sum[0], acc[r][0]);
          acc[r][1] = fmaf(slo, sum[1], acc[r][1]);
          acc[r][2] = fmaf(shi, sum[2], acc[r][2]);
          acc[r][3] = fmaf(shi, sum[3], acc[r][3]);
        }
      }
      // (x for the next tile: other warps' products hide its way; a second set of registers for it cost more than it gave)
      if (i + 1 < end) load_x(x, row, p.k, kt, t);
      __syncwarp();  // the tile has been read: its place may be filled again
      if (lane == 0) copy(stage);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (last && i + 1 < end) {
        leave();
        seg += kSeg / 4;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[r][c] = 0.f;
      }
    }
    if (at < end) leave();
    __syncthreads();
    // The block's sums of each of its row blocks, to the block that finishes it: b % split.  There it has the slots of its
    // row block b / split, one for each block that has tiles of it, in their order: 2 where there are at least as many row
    // blocks as blocks (a block has a row block's worth of tiles then, or more), else `split` (and one row block).
    if (split > 1 && rb0 == rb_begin) cluster_wait();
    const int log_per = count >= split ? 1 : log_split;
    const int cols = min(kCols, p.rows - m0);
    int bound[kWarps + 1];
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) bound[w] = warp_at[w];
    const uint32_t base = smem_u32(parts);
    // 64 threads (128 for more than 4 columns) to a row block, four columns to a thread
    const int wide = cols > 4, e = threadIdx.x & ((64 << wide) - 1), in = wide ? e * 4 : e * 8;
    for (int b = block_row[rank] + (threadIdx.x >> (6 + wide)); b * T < block_at[rank + 1]; b += kThreads >> (6 + wide)) {
      const int from = b * T;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (bound[w] < bound[w + 1] && bound[w] < from + T && bound[w + 1] > from) {
          const float4 q = *reinterpret_cast<const float4*>(segs + (w * 2 + (bound[w] < from)) * (kSeg / 4) + in);
          v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
        }
      int first = 0;  // of the blocks that have tiles of b
      while (block_at[first + 1] <= from) ++first;
      const int at_slot = ((b >> log_split) << log_per) + rank - first;
      st_cluster4(cluster_addr(base + at_slot * kSeg + in * 4, b & (split - 1)), v);
    }
    // (what the next pass begins with is under way meanwhile)
    const int this_rb = rb0, this_count = count;
    rb0 += most;
    if (rb0 < rb_end) {
      count = min(most, rb_end - rb0);
      tiles = count * T;
      at = first_of(tiles, me);
      end = first_of(tiles, me + 1);
      kt = at % T;
      if (at < end) load_x(x, row, p.k, kt, t);
    }
    if (split > 1) {
      __syncwarp();  // (the cluster's barrier takes whole warps, here and below)
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
    // The outputs of this block's row blocks, along n in a warp.
    constexpr int kOut = GATED ? 32 : 64;
    const int o = threadIdx.x % kOut;
    const int owned = (this_count - rank + split - 1) >> log_split;
    for (int q = threadIdx.x / kOut; q < owned * cols; q += kThreads / kOut) {
      const int j = q / cols, m = q - j * cols, b = (j << log_split) + rank;
      const int64_t n = (int64_t)(this_rb + b) * kOut + o;
      if (n >= p.n) continue;
      int from = 0, sources = 0;  // the blocks that have tiles of b
      for (int s = 0; s < split; ++s) {
        from += block_at[s + 1] <= b * T;
        sources += block_at[s] < (b + 1) * T;
      }
      sources -= from;
      const float* in = parts + (j << log_per) * (kSeg / 4) + (GATED ? (o >> 3) * 16 + (o & 7) : o) * kCols + m;
      float v = 0.f, u = 0.f;
      for (int s = 0; s < sources; ++s, in += kSeg / 4) {
        v += in[0];
        if constexpr (GATED) u += in[8 * kCols];
      }
      if constexpr (GATED) {
        v = w4_act(v, p.act) * u;
      } else {
        if (p.bias) v += W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.bias)[n]);
        if (p.residual) v += W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.residual)[(m0 + m) * p.res_ld + n]);
      }
      static_cast<uint16_t*>(p.out)[(int64_t)(m0 + m) * p.n + n] = W4Num<HALF>::from_float(v);
    }
    if (rb0 < rb_end) {  // no block is sent new sums before these are read
      if (split > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
      } else {
        __syncthreads();
      }
      write_bounds();
    }
  }
}

template <bool HALF, int G, bool ZEROS, bool GATED>
cudaError_t launch(const W4Dev& p, cudaStream_t st) {
  constexpr int kTile = w4_tile_bytes(G, ZEROS);
  const int chunks = (p.rows + kCols - 1) / kCols;
  // All blocks are resident at once, in the clusters with which the busiest warp has the fewest tiles: 344 row blocks of 32 tiles
  // (1 x 4096 x 11008, gated) on 148 SMs give it 8 with blocks alone, 5 with clusters of 4.
  const int smem = few_smem(kTile);
  static std::atomic<uint64_t> done{0};
  cudaError_t e = smem_attr_once(k_w4_few<HALF, G, ZEROS, GATED>, smem, done);
  if (e != cudaSuccess) return e;
  static ClusterRoom room;
  int split = 1, log_split = 0, clusters = 1;
  int64_t best = INT64_MAX;
  for (int l = 0; (1 << l) <= kMaxSplit && (1 << l) <= p.tiles_k; ++l) {  // (every block has tiles)
    const int s = 1 << l;
    const int c = std::max(1, std::min(p.blocks, cluster_room(k_w4_few<HALF, G, ZEROS, GATED>, s, kThreads, smem, room) / chunks));
    const int64_t cost = ((int64_t)((p.blocks + c - 1) / c) * p.tiles_k + kWarps * s - 1) / (kWarps * s);
    if (cost < best) {
      best = cost;
      split = s;
      log_split = l;
      clusters = c;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * split, chunks);
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
  return cudaLaunchKernelEx(&cfg, k_w4_few<HALF, G, ZEROS, GATED>, p, log_split, clusters);
}

template <bool HALF, int G, bool ZEROS>
cudaError_t pick_gated(const W4Dev& p, bool gated, cudaStream_t st) {
  return gated ? launch<HALF, G, ZEROS, true>(p, st) : launch<HALF, G, ZEROS, false>(p, st);
}
template <bool HALF, int G>
cudaError_t pick_zeros(const W4Dev& p, bool zeros, bool gated, cudaStream_t st) {
  return zeros ? pick_gated<HALF, G, true>(p, gated, st) : pick_gated<HALF, G, false>(p, gated, st);
}
template <bool HALF>
cudaError_t pick_group(const W4Dev& p, int group, bool zeros, bool gated, cudaStream_t st) {
  if (group == 32) return pick_zeros<HALF, 32>(p, zeros, gated, st);
  if (group == 64) return pick_zeros<HALF, 64>(p, zeros, gated, st);
  return pick_zeros<HALF, 128>(p, zeros, gated, st);
}

}  // namespace

cudaError_t launch_w4_few(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st) {
  return half ? pick_group<true>(p, group, zeros, gated, st) : pick_group<false>(p, group, zeros, gated, st);
}

}  // namespace t2w
