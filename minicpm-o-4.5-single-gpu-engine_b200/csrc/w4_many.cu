// Products with 4-bit weights for many rows of x on tcgen05: D[128 rows of W][NX rows of x] = (W - zero) x^T, one
// accumulator for each group of k, scaled and summed in registers.
//
// A persistent block an SM:
//   warp 0       x: TMA, 128-byte swizzle, stages of 64 k (NX = 256) or 128 k
//   warp 1       TMEM, and tcgen05.mma from one lane (M = 128, N = NX, K = 16)
//   warp 2       packed tiles of W (128 rows x 128 k), bulk copies into a ring of their own
//   2 x 4 warps  widen codes to whole 16-bit numbers and write them as a stage's A operand (K-major, 128-byte swizzle); the
//                warpgroups take the stages in turn
//   NA x 4 warps take a group's accumulator out of TMEM (two take turns), each lane one row of W: acc += scale * sum, so the
//                scale is a register and no weight is rounded; at a tile's end they write the outputs
// What a hand-over costs decides the rest: passing an mbarrier that is ready takes about 100 clocks, a commit 80, the
// issue of 4 products 65.  So with groups of 128 one barrier tells the products' warp everything that a tile waits for (x,
// weights, a free accumulator), and one commit tells that its stage is free and its accumulator full.
// With few tiles k is split over a cluster, whose blocks add their sums through distributed shared memory in a fixed order.
// The first tiles of W come before the kernel waits for the one ahead of it in the stream.  No TMA multicast.
#include "common.cuh"
#include "kernels.h"
#include "w4.h"

namespace t2w {
namespace {

constexpr int kM = 128;              // rows of W of a tile
constexpr int kABlock = kM * 64 * 2;  // widened weights of 64 k
constexpr int kMaxCodes = 8;         // packed tile pairs under way
constexpr int kMaxSmem = 232448;
constexpr int kWiden = 8;             // widening warps
constexpr int kChunk = 16;            // columns that the end of a tile takes at a time

template <int NX>
struct Cfg {
  static constexpr int NA = NX == 256 ? 2 : 1;    // accumulating warpgroups
  static constexpr int CA = NX / NA;              // columns of an accumulating warpgroup
  static constexpr int KB = NX == 256 ? 1 : 2;    // blocks of 64 k in a stage
  static constexpr int THREADS = 128 * (3 + NA);
  static constexpr int A_BYTES = KB * kABlock, B_BYTES = KB * NX * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = NX == 256 ? 4 : 3;
  static constexpr int SLOTS = STAGES * KB / 2 + 2;  // tiles whose scales are kept (see the widening warps)
  static constexpr int TMEM = 2 * NX;
  // Registers: CA = 128 sums need more than an even split has, which the other warps give.  The sum of the warpgroups'
  // shares is at most what the kernel is launched with: 96 each of 640 threads, 128 each of 512.
  static constexpr bool SHIFT = CA == 128;
  static constexpr int LAUNCH = NX == 256 ? 96 : 128;
  static constexpr int R_ROLES = 48, R_WIDEN = NX == 256 ? 48 : 104, R_SUM = NX == 256 ? 168 : 184;
  static_assert(R_ROLES + 2 * R_WIDEN + NA * R_SUM <= (3 + NA) * LAUNCH, "registers");
  static constexpr int fixed(int group) {  // shared memory besides the ring of packed tiles
    return STAGES * STAGE + SLOTS * (kW4K / group) * 256 + 8 * (2 * STAGES + 2 * kMaxCodes + 5) + 16;
  }
};
static_assert(Cfg<256>::STAGES % 2 == 0, "a tile's two stages are always the same two kinds");

struct ManyArgs {
  W4Dev p;
  int zeros, gated;
  int tile_bytes;  // of a packed tile
  int tiles_n, tiles;
  int split;
  int code_stages;
};

template <int N>
T2W_DEV void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
T2W_DEV void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
T2W_DEV void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
T2W_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__host__ __device__ constexpr uint32_t idesc_16(int M, int N, bool half) {
  return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

T2W_DEV void tmem_st32(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]),
      "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]),
      "f"(v[31])
      : "memory");
}
T2W_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The two meetings of a cluster's blocks, for warps that have no part in what lies between them.
T2W_DEV void cluster_pass() {
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  cluster_arrive();
  cluster_wait();
}

// Ring position.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  T2W_DEV void next(int n, int by = 1) {
    if ((stage += by) >= n) {
      stage -= n;
      phase ^= 1u;
    }
  }
};

// A block's k tiles: a share of the cluster's.
struct Span {
  int first, end;
};
T2W_DEV Span span_of(int tiles_k, int rank, int split) {
  return {(int)((int64_t)tiles_k * rank / split), (int)((int64_t)tiles_k * (rank + 1) / split)};
}

// After the cluster's blocks have met: a share of a tile's columns, from all blocks' sums [column][row].
template <bool HALF, int NX>
T2W_DEV void finish_cluster(const ManyArgs& a, const uint8_t* smem, int tile, int rank, int thread, int threads) {
  const W4Dev& p = a.p;
  const int64_t packed0 = (int64_t)(tile % a.tiles_n) * kM;
  const int m0 = (tile / a.tiles_n) * NX, per = NX / a.split;
  const int quads = a.gated ? 16 : 32;  // fours of outputs of a column
  const uint32_t base = smem_u32(smem);
#pragma unroll 1
  for (int e = thread; e < per * quads; e += threads) {
    const int c = rank * per + e / quads, o = e % quads * 4, m = m0 + c;
    const int64_t n = a.gated ? packed0 / 2 + o : packed0 + o;
    if (m >= p.rows || n >= p.n) continue;
    if (a.gated) {
      const uint32_t at = base + (c * kM + (o >> 3) * 16 + (o & 7)) * 4;
      w4_finish4<HALF, true>(p, m, n, cluster_sum4(at, a.split), cluster_sum4(at + 32, a.split));
    } else {
      w4_finish4<HALF, false>(p, m, n, cluster_sum4(base + (c * kM + o) * 4, a.split), make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
}

template <bool HALF, int NX, int G>
__global__ void __launch_bounds__(Cfg<NX>::THREADS, 1)
    k_w4_many(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ ManyArgs a) {
  using C = Cfg<NX>;
  const W4Dev& p = a.p;
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int groups = kW4K / G, slot_bytes = groups * 2 * 128;
  // One barrier for all that a tile's products wait for, and one commit for all that wait for them: where a group is a tile.
  constexpr bool kOne = G == kW4K;
  constexpr int kPerTile = 2 / C::KB;  // stages of a tile
  const int code_bytes = 2 * a.tile_bytes;
  uint8_t* scales = smem + C::STAGES * C::STAGE;  // [slot][half][group][64]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + C::SLOTS * slot_bytes);
  uint64_t* empty = full + C::STAGES;  // the stage's products have ended
  uint64_t* cfull = empty + C::STAGES;
  uint64_t* cempty = cfull + kMaxCodes;
  uint64_t* dfull = cempty + kMaxCodes;  // (not kOne)
  uint64_t* dempty = dfull + 2;
  uint64_t* drain = dempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  uint8_t* codes = smem + (C::fixed(G) + 127) / 128 * 128;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.split > 1 ? (int)cluster_rank() : 0;
  const int first_tile = blockIdx.x / a.split, tile_step = gridDim.x / a.split;
  const Span span = span_of(p.tiles_k, rank, a.split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      // x, the four warps that widen it, and with the tile's first stage the warps that take accumulators
      mbar_init(&full[s], 1 + 4 + (kOne && s % kPerTile == 0 ? 4 * C::NA : 0));
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < a.code_stages; ++s) {
      mbar_init(&cfull[s], 1);
      mbar_init(&cempty[s], kWiden / C::KB);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&dfull[s], 1);
      mbar_init(&dempty[s], 4 * C::NA);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
  }
  __syncthreads();

  if (warp < 4) {
    if constexpr (C::SHIFT) regs_dec<C::R_ROLES>();
    if (warp == 0) {
      pdl_wait();
      if (elect_one()) {
        Ring r;
        int issued = 0;
        bool ok = true;
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
          const int m0 = (tile / a.tiles_n) * NX;
          for (int kb = 2 * span.first; kb < 2 * span.end; kb += C::KB) {
            if (!(ok = w4_wait(&empty[r.stage], r.phase ^ 1u, p.status))) break;
            uint8_t* to = smem + r.stage * C::STAGE + C::A_BYTES;
            mbar_expect_tx(&full[r.stage], C::B_BYTES);
#pragma unroll
            for (int b = 0; b < C::KB; ++b) tma_load_2d(to + b * NX * 128, &tmX, (kb + b) * 64, m0, &full[r.stage]);
            ++issued;
            r.next(C::STAGES);
          }
        }
        // The block does not end, nor is its shared memory used for sums, with a copy under way (where a wait gave up).
        if (!ok)
          for (int i = issued > C::STAGES ? issued - C::STAGES : 0; i < issued; ++i)
            w4_wait(&full[i % C::STAGES], (i / C::STAGES) & 1, p.status);
      }
      __syncwarp();
    } else if (warp == 2) {
      if (elect_one()) {
        Ring r;
        int issued = 0;
        bool ok = true;
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
          const int rb = (tile % a.tiles_n) * 2, halves = rb + 1 < p.blocks ? 2 : 1;
          for (int kt = span.first; kt < span.end; ++kt) {
            if (!(ok = w4_wait(&cempty[r.stage], r.phase ^ 1u, p.status))) break;
            mbar_expect_tx(&cfull[r.stage], halves * a.tile_bytes);
            for (int h = 0; h < halves; ++h)
              bulk_load(codes + r.stage * code_bytes + h * a.tile_bytes,
                        p.tiles + ((int64_t)(rb + h) * p.tiles_k + kt) * a.tile_bytes, a.tile_bytes, &cfull[r.stage]);
            ++issued;
            r.next(a.code_stages);
          }
        }
        if (!ok)
          for (int i = issued > a.code_stages ? issued - a.code_stages : 0; i < issued; ++i)
            w4_wait(&cfull[i % a.code_stages], (i / a.code_stages) & 1, p.status);
      }
      __syncwarp();
    } else if (warp == 1) {
      pdl_wait();
      tmem_alloc(tmem_slot, C::TMEM);
      tmem_relinquish();
      pdl_launch();
      tc_fence_before();
      named_sync(1, 32 + 128 * C::NA);
      tc_fence_after();
      const uint32_t tmem = *tmem_slot;
      // The whole warp goes through the loop, so that descriptors and addresses stay in uniform registers; one lane issues.
      constexpr uint32_t idesc = idesc_16(kM, NX, HALF);
      // Operands' descriptors, stage 0: 32 bytes further for each 16 k, a block further for each 64, a stage for each stage.
      const uint64_t adesc = sdesc_sw128(smem_u32(smem), 1024, 16), bdesc = sdesc_sw128(smem_u32(smem) + C::A_BYTES, 1024, 16);
      constexpr int kStageSteps = 4 * C::KB;                                      // products of a stage
      constexpr int kSteps = G / 16 < kStageSteps ? G / 16 : kStageSteps;  // of a group in it
      Ring sr, dr;
      bool ok = true;
      for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step)
        for (int kb = 2 * span.first; kb < 2 * span.end; kb += C::KB) {
          if (!(ok = w4_wait_warp(&full[sr.stage], sr.phase, p.status))) break;
          const uint64_t ad = adesc + sr.stage * (C::STAGE >> 4), bd = bdesc + sr.stage * (C::STAGE >> 4);
#pragma unroll
          for (int j = 0; j < kStageSteps / kSteps; ++j) {
            const bool fresh = C::KB == 2 || G < 128 || (kb & 1) == 0, last = C::KB == 2 || G < 128 || (kb & 1) != 0;
            if (!kOne && !(ok = w4_wait_warp(&dempty[dr.stage], dr.phase ^ 1u, p.status))) break;
            tc_fence_after();
            const uint32_t d = tmem + dr.stage * NX;
            if (elect_one()) {
#pragma unroll
              for (int i = 0; i < kSteps; ++i) {
                const int k = j * kSteps + i;
                umma_f16(d, ad + (k >> 2) * (kABlock >> 4) + (k & 3) * 2, bd + (k >> 2) * (NX * 128 >> 4) + (k & 3) * 2, idesc,
                         i == 0 && fresh ? 0u : 1u);
              }
              if (!kOne) umma_commit(&dfull[dr.stage]);
              if (j == kStageSteps / kSteps - 1) umma_commit(&empty[sr.stage]);
            }
            __syncwarp();
            if (last) dr.next(2);
          }
          if (!ok) break;
          sr.next(C::STAGES);
        }
      if (!ok) {  // TMEM is not given back with a product under way
        if (elect_one()) umma_commit(drain);
        __syncwarp();
        w4_wait_warp(drain, 0, p.status);
      }
    }
    if (a.split > 1) cluster_pass();
    if (warp == 1) {
      named_sync(1, 32 + 128 * C::NA);
      tc_fence_after();
      tmem_dealloc(*tmem_slot, C::TMEM);
    }
  } else if (warp < 4 + kWiden) {
    if constexpr (C::SHIFT) regs_dec<C::R_WIDEN>();
    // The warpgroups take the stages in turn: with stages of 64 k each its half of every tile, else every other tile.
    const int w = (warp - 4) & 3, mine = (warp - 4) >> 2, g = lane >> 2, t = lane & 3, odd = g & 1;
    const int my_codes = (w * 64 + lane) * 16, my_zeros = kW4Codes + groups * 128 + g * 8 + w * 2;
    const int my_row = (w * 16 + g) * 128, chunk0 = ((4 * odd + t) ^ g) << 4, chunk1 = ((4 * (1 - odd) + t) ^ g) << 4;
    Ring cr, sr;
    sr.stage = mine;
    int slot = 0, turn = 0;
    bool ok = true;
    for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
      const int halves = (tile % a.tiles_n) * 2 + 1 < p.blocks ? 2 : 1;
      for (int kt = span.first; kt < span.end; ++kt) {
        if (C::KB == 1 || turn == mine) {
          if (!(ok = w4_wait_warp(&cfull[cr.stage], cr.phase, p.status))) break;
          const uint8_t* in = codes + cr.stage * code_bytes;
          // 16 rows x 64 k at a time; warp w has strip w of both halves.  Odd rows take (and write) their halves of the k in
          // the other order, so that eight lanes' 16 bytes of the operand lie in eight groups of banks.
          uint2 c[C::KB][2][2];
          uint32_t z[C::KB][2][2];
#pragma unroll
          for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h >= halves) break;
              const uint8_t* src = in + h * a.tile_bytes;
              const int kb = C::KB == 1 ? mine : b;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                c[b][h][i] = *reinterpret_cast<const uint2*>(src + my_codes + kb * 512 + (i ^ odd) * 8);
                z[b][h][i] = 0x0808;
                if (a.zeros) {
                  const int group = G == 32 ? kb * 2 + (i ^ odd) : kb * 64 / G;
                  z[b][h][i] = *reinterpret_cast<const uint16_t*>(src + my_zeros + group * 64);
                }
              }
            }
          if (!(ok = w4_wait_warp(&empty[sr.stage], sr.phase ^ 1u, p.status))) break;
          uint8_t* out = smem + sr.stage * C::STAGE + my_row;
          // The scales move to a slot of their own.  The slot's last tile was SLOTS tiles ago, 2 more than the stages hold; the
          // products of the tile that had this stage have ended (`empty`), so an accumulator was free when they began, so
          // the sums of the group 2 before theirs, and of every tile at least 2 before, are taken.
          if (C::KB == 2 || kW4K == G * 2 || mine == 0 || G < 64) {
            // with stages of 64 k each warpgroup moves the groups that begin in its half
            constexpr int kOwn = C::KB == 2 ? groups : (groups + 1) / 2;
            const int from = C::KB == 1 ? mine * kOwn * 8 : 0;
            const int i = w * 32 + lane, h = i / (kOwn * 8), j = i % (kOwn * 8);
            if (h < halves)
              reinterpret_cast<uint4*>(scales + slot * slot_bytes + h * groups * 128)[from + j] =
                  reinterpret_cast<const uint4*>(in + h * a.tile_bytes + kW4Codes)[from + j];
          }
#pragma unroll
          for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h >= halves) break;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t zlo = w4_zero<HALF>(z[b][h][i] & 255), zhi = w4_zero<HALF>(z[b][h][i] >> 8);
                uint32_t x[4], y[4];
                w4_widen<HALF>(c[b][h][i].x, zlo, zhi, x);
                w4_widen<HALF>(c[b][h][i].y, zlo, zhi, y);
                const int chunk = b * kABlock + h * 64 * 128 + (i ? chunk1 : chunk0);
                *reinterpret_cast<uint4*>(out + chunk) = make_uint4(x[0], x[2], y[0], y[2]);
                *reinterpret_cast<uint4*>(out + 8 * 128 + chunk) = make_uint4(x[1], x[3], y[1], y[3]);
              }
            }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&full[sr.stage]);
            mbar_arrive(&cempty[cr.stage]);
          }
          sr.next(C::STAGES, 2);
        }
        turn ^= 1;
        cr.next(a.code_stages);
        if (++slot == C::SLOTS) slot = 0;
      }
    }
    if (a.split > 1) {
      if constexpr (NX == 256) {
        cluster_pass();
      } else {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        finish_cluster<HALF, NX>(a, smem, first_tile, rank, threadIdx.x - 128, 128 * (2 + C::NA));
        __syncwarp();
        cluster_arrive();
        cluster_wait();
      }
    }
  } else {
    if constexpr (C::SHIFT) regs_inc<C::R_SUM>();
    const int w = warp - 4 - kWiden, part = w >> 2, r = (warp & 3) * 32 + lane;  // row of W in the tile
    if (kOne && lane == 0) {  // both accumulators are free
      mbar_arrive(&full[0]);
      mbar_arrive(&full[kPerTile]);
    }
    pdl_wait();
    named_sync(1, 32 + 128 * C::NA);
    tc_fence_after();
    const uint32_t taddr = *tmem_slot + ((uint32_t)((warp & 3) * 32) << 16) + part * C::CA;
    const uint16_t* my_scales = reinterpret_cast<const uint16_t*>(scales + (r >> 6) * groups * 128) + w4_place(r & 63);
    // kOne: a tile's accumulator is full when its last stage's products have ended, and free for the tile 2 later, whose
    // first stage's barrier is told.
    Ring dr, er;
    er.stage = kPerTile - 1;
    int tell = 2 * kPerTile % C::STAGES, slot = 0;
    auto give_back = [&](int d) {  // accumulator d has been taken
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(kOne ? &full[tell] : &dempty[d]);
      if ((tell += kPerTile) >= C::STAGES) tell -= C::STAGES;
    };
    bool ok = true;
    for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
      const int m0 = (tile / a.tiles_n) * NX + part * C::CA;
      const int64_t packed = (int64_t)(tile % a.tiles_n) * kM + r;  // row of the packed weight
      float acc[C::CA];
      int held = 0;  // the last group's accumulator
#pragma unroll
      for (int c = 0; c < C::CA; ++c) acc[c] = 0.f;
      for (int kt = span.first; kt < span.end && ok; ++kt) {
        for (int gr = 0; gr < groups; ++gr) {
          if (kOne) {
            if (!(ok = w4_wait_warp(&empty[er.stage], er.phase, p.status))) break;
            er.next(C::STAGES, kPerTile);
          } else {
            if (!(ok = w4_wait_warp(&dfull[dr.stage], dr.phase, p.status))) break;
          }
          tc_fence_after();
          const float s = w4_scale(my_scales[slot * (slot_bytes / 2) + gr * 64], p.scale_half);
          const float2 s2 = make_float2(s, s);
#pragma unroll
          for (int c = 0; c < C::CA; c += 32) {
            float v[32];
            tmem_ld32(taddr + dr.stage * NX + c, v);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 q = fma2(s2, make_float2(v[i], v[i + 1]), make_float2(acc[c + i], acc[c + i + 1]));
              acc[c + i] = q.x;
              acc[c + i + 1] = q.y;
            }
          }
          held = dr.stage;
          if (kt + 1 < span.end || gr + 1 < groups) give_back(held);
          dr.next(2);
        }
        if (++slot == C::SLOTS) slot = 0;
      }
      if (!ok) break;
      // The sums go into the accumulator taken last and come back a few columns at a time: what follows is a short loop
      // then, where all columns in a row would be ten thousand bytes of code that no instruction cache has in time.
      const uint32_t own = taddr + held * NX;
#pragma unroll
      for (int c = 0; c < C::CA; c += 32) tmem_st32(own + c, acc + c);
      tmem_st_wait();
      const int cols = min(C::CA, p.rows - m0);
      if (a.split > 1) {
        // [column][row] in the stages' place: every product and copy of this block is complete.
        float* sums = reinterpret_cast<float*>(smem) + part * C::CA * kM + r;
#pragma unroll 1
        for (int c0 = 0; c0 < C::CA; c0 += kChunk) {
          float v[kChunk];
          tmem_ld16(own + c0, v);
#pragma unroll
          for (int c = 0; c < kChunk; ++c) sums[(c0 + c) * kM] = v[c];
        }
        break;  // one tile a cluster
      }
      uint16_t* out = static_cast<uint16_t*>(p.out) + (int64_t)m0 * p.n;
      if (!a.gated) {
        const bool in = packed < p.n;
        const float bias = in && p.bias ? W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.bias)[packed]) : 0.f;
        const uint16_t* res = static_cast<const uint16_t*>(p.residual);
        if (!in) res = nullptr;
        if (res) res += (int64_t)m0 * p.res_ld + packed;
        out += packed;
        const int count = in ? cols : 0;
        uint16_t next[kChunk];  // residuals, read a round ahead
#pragma unroll
        for (int c = 0; c < kChunk; ++c) next[c] = res && c < count ? res[(int64_t)c * p.res_ld] : (uint16_t)0;
#pragma unroll 1
        for (int c0 = 0; c0 < C::CA; c0 += kChunk) {
          float v[kChunk];
          tmem_ld16(own + c0, v);
          if (res) {
            res += kChunk * p.res_ld;
#pragma unroll
            for (int c = 0; c < kChunk; ++c) {
              v[c] += W4Num<HALF>::to_float(next[c]);
              if (c0 + kChunk + c < count) next[c] = res[(int64_t)c * p.res_ld];
            }
          }
#pragma unroll
          for (int c = 0; c < kChunk; ++c)
            if (c0 + c < count) out[(int64_t)(c0 + c) * p.n] = W4Num<HALF>::from_float(v[c] + bias);
        }
      } else {
        // Rows 0 .. 7 of 16 are gates, 8 .. 15 the up rows of the same outputs: lanes 8 apart exchange, and each has one
        // of two columns.
        const bool up = (r & 8) != 0;
        const int64_t n = (packed >> 4) * 8 + (r & 7);
        out += n + (up ? p.n : 0);
        const int count = n < p.n ? cols - (up ? 1 : 0) : 0;
#pragma unroll 1
        for (int c0 = 0; c0 < C::CA; c0 += kChunk) {
          float v[kChunk];
          tmem_ld16(own + c0, v);
#pragma unroll
          for (int c = 0; c < kChunk; c += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 8);
            const float y = w4_act(up ? other : v[c], p.act) * (up ? v[c + 1] : other);
            if (c0 + c < count) out[(int64_t)(c0 + c) * p.n] = W4Num<HALF>::from_float(y);
          }
        }
      }
      give_back(held);
    }
    if (a.split > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      constexpr int kThreads = NX == 256 ? 128 * C::NA : 128 * (2 + C::NA);  // the widening warps help where they have registers
      finish_cluster<HALF, NX>(a, smem, first_tile, rank, (int)threadIdx.x - (C::THREADS - kThreads), kThreads);
      __syncwarp();
      cluster_arrive();  // no block leaves while another reads its sums
      cluster_wait();
    }
    tc_fence_before();
    named_sync(1, 32 + 128 * C::NA);
  }
}

template <bool HALF, int NX, int G>
cudaError_t launch(const W4Dev& p, bool zeros, bool gated, int split, cudaStream_t st) {
  using C = Cfg<NX>;
  ManyArgs a = {};
  a.p = p;
  a.zeros = zeros;
  a.gated = gated;
  a.tile_bytes = w4_tile_bytes(G, zeros);
  a.tiles_n = (p.blocks + 1) / 2;
  const int64_t tiles = (int64_t)a.tiles_n * ((p.rows + NX - 1) / NX);
  if (tiles > (1 << 27)) return cudaErrorInvalidValue;
  a.tiles = (int)tiles;
  a.split = split;
  CUtensorMap map;
  if (!make_tmap_2d(&map, p.x, 2, p.rows, p.k, (uint64_t)p.x_ld * 2, NX, 64)) return cudaErrorInvalidValue;
  // as many packed tiles under way as there is room for
  const int fixed = (C::fixed(G) + 127) / 128 * 128, room = (kMaxSmem - fixed) / (2 * a.tile_bytes);
  a.code_stages = room < kMaxCodes ? room : kMaxCodes;
  const int smem = fixed + a.code_stages * 2 * a.tile_bytes;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = smem_attr_once(k_w4_many<HALF, NX, G>, kMaxSmem, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split > 1 ? a.tiles * split : (a.tiles < num_sms() ? a.tiles : num_sms()));
  cfg.blockDim = dim3(C::THREADS);
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
  return cudaLaunchKernelEx(&cfg, k_w4_many<HALF, NX, G>, map, a);
}

template <bool HALF, int NX>
cudaError_t pick_group(const W4Dev& p, int group, bool zeros, bool gated, int split, cudaStream_t st) {
  if (group == 32) return launch<HALF, NX, 32>(p, zeros, gated, split, st);
  if (group == 64) return launch<HALF, NX, 64>(p, zeros, gated, split, st);
  return launch<HALF, NX, 128>(p, zeros, gated, split, st);
}
template <bool HALF>
cudaError_t pick(const W4Dev& p, int group, bool zeros, bool gated, cudaStream_t st) {
  const int nx = p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : p.rows <= 128 ? 128 : 256;
  const int64_t tiles = (int64_t)((p.blocks + 1) / 2) * ((p.rows + nx - 1) / nx);
  int split = 1;
  while (split < 8 && tiles * split * 2 <= num_sms() && p.tiles_k >= 2 * split) split *= 2;
  if (nx == 32) return pick_group<HALF, 32>(p, group, zeros, gated, split, st);
  if (nx == 64) return pick_group<HALF, 64>(p, group, zeros, gated, split, st);
  if (nx == 128) return pick_group<HALF, 128>(p, group, zeros, gated, split, st);
  return pick_group<HALF, 256>(p, group, zeros, gated, split, st);
}

}  // namespace

cudaError_t launch_w4_many(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st) {
  return half ? pick<true>(p, group, zeros, gated, st) : pick<false>(p, group, zeros, gated, st);
}

}  // namespace t2w
