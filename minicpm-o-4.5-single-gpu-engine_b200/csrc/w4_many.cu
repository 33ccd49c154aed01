// Products with 4-bit weights for many rows of x on tcgen05: D[128 rows of W][NX rows of x] = (W - zero) x^T, one
// accumulator for each group of k, scaled and summed in registers.
//
// A persistent block an SM:
//   warp 0       copies: packed tiles of W (bulk) into a ring of their own, x (TMA, 128-byte swizzle) into the stages
//   warp 1       TMEM, and tcgen05.mma from one lane (M = 128, N = NX, K = 16)
//   ND x 4 warps widen codes to whole 16-bit numbers and write them as the stage's A operand (K-major, 128-byte swizzle)
//   NA x 4 warps take a group's accumulator out of TMEM (two take turns), each lane one row of W: acc += scale * sum, so the
//                scale is a register and no weight is rounded; at a tile's end they write the outputs
// Stages hold 128 k.  The accumulating warps' work does not depend on NX per product: 1 multiplication-addition for `group`
// products.  With few tiles k is split over a cluster, whose blocks add their sums through distributed shared memory in a
// fixed order.  W is not read ahead of x by more than the ring, but its first tiles come before the kernel waits for the one
// ahead of it in the stream.  No TMA multicast.
#include "common.cuh"
#include "kernels.h"
#include "w4.h"

namespace t2w {
namespace {

constexpr int kM = 128;                  // rows of W of a tile
constexpr int kABytes = kM * kW4K * 2;   // a stage's widened weights: two blocks of 64 k
constexpr int kCodeStages = 3;
constexpr int kMaxSmem = 232448;

template <int NX>
struct Cfg {
  static constexpr int ND = NX == 256 ? 1 : 2;  // widening warpgroups
  static constexpr int NA = NX == 256 ? 2 : 1;  // accumulating warpgroups
  static constexpr int CA = NX / NA;            // columns of an accumulating warpgroup
  static constexpr int THREADS = 128 * (1 + ND + NA);
  static constexpr int B_BYTES = NX * kW4K * 2;
  static constexpr int STAGE = kABytes + B_BYTES;
  static constexpr int STAGES = NX == 256 ? 2 : NX >= 64 ? 3 : 4;
  static constexpr int SLOTS = STAGES + 2;  // tiles whose scales are kept (see the widening warps)
  static constexpr int TMEM = 2 * NX < 32 ? 32 : 2 * NX;
  // Registers: the kernel is launched with 128 a thread.  CA = 128 sums need more, which the other warps give: 56 + 104 ND +
  // 176 NA is 512 for NX = 256 and 440 for NX = 128, of 128 (1 + ND + NA) = 512.
  static constexpr bool SHIFT = CA == 128;
};
static_assert(56 + 104 * Cfg<256>::ND + 176 * Cfg<256>::NA <= 128 * (1 + Cfg<256>::ND + Cfg<256>::NA), "registers");
static_assert(56 + 104 * Cfg<128>::ND + 176 * Cfg<128>::NA <= 128 * (1 + Cfg<128>::ND + Cfg<128>::NA), "registers");

struct ManyArgs {
  W4Dev p;
  int group, zeros, gated;
  int tile_bytes;  // of a packed tile
  int tiles_n, tiles;
  int split;
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
  T2W_DEV void next(int n) {
    if (++stage == n) {
      stage = 0;
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

// One output (row m of x, output n): what is added, and the store.
template <bool HALF>
T2W_DEV void store_linear(const W4Dev& p, int m, int n, float v, float bias) {
  v += bias;
  if (p.residual) v += W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.residual)[(int64_t)m * p.res_ld + n]);
  static_cast<uint16_t*>(p.out)[(int64_t)m * p.n + n] = W4Num<HALF>::from_float(v);
}

template <bool HALF, int NX>
__global__ void __launch_bounds__(Cfg<NX>::THREADS, 1)
    k_w4_many(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ ManyArgs a) {
  using C = Cfg<NX>;
  const W4Dev& p = a.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int groups = kW4K / a.group, code_bytes = 2 * a.tile_bytes, slot_bytes = groups * 2 * 128;
  uint8_t* codes = smem + C::STAGES * C::STAGE;
  uint8_t* scales = codes + kCodeStages * code_bytes;  // [slot][half][group][64]
  uint64_t* afull = reinterpret_cast<uint64_t*>(scales + C::SLOTS * slot_bytes);
  uint64_t* bfull = afull + C::STAGES;
  uint64_t* empty = bfull + C::STAGES;
  uint64_t* cfull = empty + C::STAGES;
  uint64_t* cempty = cfull + kCodeStages;
  uint64_t* dfull = cempty + kCodeStages;
  uint64_t* dempty = dfull + 2;
  uint64_t* drain = dempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.split > 1 ? (int)cluster_rank() : 0;
  const int first_tile = blockIdx.x / a.split, tile_step = gridDim.x / a.split;
  const Span span = span_of(p.tiles_k, rank, a.split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&afull[s], 4 * C::ND);
      mbar_init(&bfull[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kCodeStages; ++s) {
      mbar_init(&cfull[s], 1);
      mbar_init(&cempty[s], 4 * C::ND);
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
    if constexpr (C::SHIFT) regs_dec<56>();
    if (warp == 0) {
      if (elect_one()) {
        // Codes run ahead of x by their own ring; both advance tile by tile, codes first.
        Ring cr, xr;
        int c_tile = first_tile, c_k = span.first, issued_c = 0, issued_x = 0;
        auto next_codes = [&]() -> bool {  // one packed tile pair
          if (!mbar_wait(&cempty[cr.stage], cr.phase ^ 1u, p.status)) return false;
          const int rb = (c_tile % a.tiles_n) * 2, halves = rb + 1 < p.blocks ? 2 : 1;
          mbar_expect_tx(&cfull[cr.stage], halves * a.tile_bytes);
          for (int h = 0; h < halves; ++h)
            bulk_load(codes + cr.stage * code_bytes + h * a.tile_bytes,
                      p.tiles + ((int64_t)(rb + h) * p.tiles_k + c_k) * a.tile_bytes, a.tile_bytes, &cfull[cr.stage]);
          ++issued_c;
          cr.next(kCodeStages);
          if (++c_k == span.end) {
            c_k = span.first;
            c_tile += tile_step;
          }
          return true;
        };
        bool ok = true;
        for (int i = 0; i < kCodeStages && c_tile < a.tiles && ok; ++i) ok = next_codes();
        pdl_wait();
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
          const int m0 = (tile / a.tiles_n) * NX;
          for (int kt = span.first; kt < span.end && ok; ++kt) {
            if (!(ok = mbar_wait(&empty[xr.stage], xr.phase ^ 1u, p.status))) break;
            uint8_t* b = smem + xr.stage * C::STAGE + kABytes;
            mbar_expect_tx(&bfull[xr.stage], C::B_BYTES);
            tma_load_2d(b, &tmX, kt * kW4K, m0, &bfull[xr.stage]);
            tma_load_2d(b + C::B_BYTES / 2, &tmX, kt * kW4K + 64, m0, &bfull[xr.stage]);
            ++issued_x;
            xr.next(C::STAGES);
            if (c_tile < a.tiles) ok = next_codes();
          }
        }
        // The block does not end, nor is its shared memory used for sums, with a copy under way (where a wait gave up).
        if (!ok) {
          for (int i = issued_c > kCodeStages ? issued_c - kCodeStages : 0; i < issued_c; ++i)
            mbar_wait(&cfull[i % kCodeStages], (i / kCodeStages) & 1, p.status);
          for (int i = issued_x > C::STAGES ? issued_x - C::STAGES : 0; i < issued_x; ++i)
            mbar_wait(&bfull[i % C::STAGES], (i / C::STAGES) & 1, p.status);
        }
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
      if (elect_one()) {
        constexpr uint32_t idesc = idesc_16(kM, NX, HALF);
        const int steps = a.group / 16;
        Ring sr, dr;
        bool ok = true;
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step)
          for (int kt = span.first; kt < span.end && ok; ++kt) {
            if (!(ok = mbar_wait(&bfull[sr.stage], sr.phase, p.status))) break;
            if (!(ok = mbar_wait(&afull[sr.stage], sr.phase, p.status))) break;
            const uint32_t a0 = smem_u32(smem + sr.stage * C::STAGE), b0 = a0 + kABytes;
            for (int gr = 0; gr < groups && ok; ++gr) {
              if (!(ok = mbar_wait(&dempty[dr.stage], dr.phase ^ 1u, p.status))) break;
              tc_fence_after();
              for (int s = 0; s < steps; ++s) {
                const int k = gr * steps + s;  // 16 k each: four to a block of 64
                umma_f16(tmem + dr.stage * NX, sdesc_sw128(a0 + (k >> 2) * (kABytes / 2) + (k & 3) * 32, 1024, 16),
                         sdesc_sw128(b0 + (k >> 2) * (C::B_BYTES / 2) + (k & 3) * 32, 1024, 16), idesc, s != 0);
              }
              umma_commit(&dfull[dr.stage]);
              dr.next(2);
            }
            if (ok) umma_commit(&empty[sr.stage]);
            sr.next(C::STAGES);
          }
        if (!ok) {  // TMEM is not given back with a product under way
          umma_commit(drain);
          mbar_wait(drain, 0, p.status);
        }
      }
      __syncwarp();
    }
    if (a.split > 1) cluster_pass();
    if (warp == 1) {
      named_sync(1, 32 + 128 * C::NA);
      tc_fence_after();
      tmem_dealloc(*tmem_slot, C::TMEM);
    }
  } else if (warp < 4 + 4 * C::ND) {
    if constexpr (C::SHIFT) regs_dec<104>();
    const int w = warp - 4, g = lane >> 2, t = lane & 3;
    Ring cr, sr;
    int slot = 0;
    bool ok = true;
    for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
      const int halves = (tile % a.tiles_n) * 2 + 1 < p.blocks ? 2 : 1;
      for (int kt = span.first; kt < span.end; ++kt) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&cfull[cr.stage], cr.phase, p.status)))) break;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&empty[sr.stage], sr.phase ^ 1u, p.status)))) break;
        const uint8_t* in = codes + cr.stage * code_bytes;
        uint8_t* out = smem + sr.stage * C::STAGE;
        // The scales move to a slot of their own.  The slot's last tile was SLOTS = STAGES + 2 tiles ago; the products of the
        // tile STAGES ago have ended (`empty`), so its last accumulator was free, so the sums of the tile 2 before it are taken.
        for (int i = w * 32 + lane; i < halves * groups * 8; i += 128 * C::ND) {
          const int h = i / (groups * 8), j = i % (groups * 8);
          reinterpret_cast<uint4*>(scales + slot * slot_bytes + h * groups * 128)[j] =
              reinterpret_cast<const uint4*>(in + h * a.tile_bytes + kW4Codes)[j];
        }
#pragma unroll
        for (int i = 0; i < 16 / (4 * C::ND); ++i) {
          const int u = w + i * 4 * C::ND;  // 16 rows x 64 k
          const int h = u >> 3, strip = (u >> 1) & 3, kb = u & 1;
          if (h >= halves) break;
          const uint8_t* src = in + h * a.tile_bytes;
          const uint4 c = reinterpret_cast<const uint4*>(src)[(strip * 2 + kb) * 32 + lane];
          uint8_t* row = out + kb * (kABytes / 2) + (h * 64 + strip * 16 + g) * 128;
          const uint8_t* zero = src + kW4Codes + groups * 128 + g * 8 + strip * 2;
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            // odd rows write their halves in the other order, so that eight lanes' 16 bytes lie in eight banks' groups
            const int q = i2 ^ (g & 1);
            uint32_t zlo = 8, zhi = 8;
            if (a.zeros) {
              const uint16_t z = *reinterpret_cast<const uint16_t*>(zero + ((kb * 64 + q * 32) / a.group) * 64);
              zlo = z & 255;
              zhi = z >> 8;
            }
            zlo = w4_zero<HALF>(zlo);
            zhi = w4_zero<HALF>(zhi);
            uint32_t x[4], y[4];
            w4_widen<HALF>(q ? c.z : c.x, zlo, zhi, x);
            w4_widen<HALF>(q ? c.w : c.y, zlo, zhi, y);
            const int chunk = ((4 * q + t) ^ g) << 4;
            *reinterpret_cast<uint4*>(row + chunk) = make_uint4(x[0], x[2], y[0], y[2]);
            *reinterpret_cast<uint4*>(row + 8 * 128 + chunk) = make_uint4(x[1], x[3], y[1], y[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&cempty[cr.stage]);
          mbar_arrive(&afull[sr.stage]);
        }
        cr.next(kCodeStages);
        sr.next(C::STAGES);
        if (++slot == C::SLOTS) slot = 0;
      }
    }
    if (a.split > 1) cluster_pass();
  } else {
    if constexpr (C::SHIFT) regs_inc<176>();
    const int w = warp - 4 - 4 * C::ND, part = w >> 2, r = (warp & 3) * 32 + lane;  // row of W in the tile
    pdl_wait();
    named_sync(1, 32 + 128 * C::NA);
    tc_fence_after();
    const uint32_t taddr = *tmem_slot + ((uint32_t)((warp & 3) * 32) << 16) + part * C::CA;
    const uint16_t* my_scales = reinterpret_cast<const uint16_t*>(scales + (r >> 6) * groups * 128) + w4_place(r & 63);
    Ring dr;
    int slot = 0;
    bool ok = true;
    for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
      const int m0 = (tile / a.tiles_n) * NX + part * C::CA;
      const int64_t packed = (int64_t)(tile % a.tiles_n) * kM + r;  // row of the packed weight
      float2 acc[C::CA / 2];
#pragma unroll
      for (int c = 0; c < C::CA / 2; ++c) acc[c] = make_float2(0.f, 0.f);
      for (int kt = span.first; kt < span.end && ok; ++kt) {
        for (int gr = 0; gr < groups; ++gr) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(&dfull[dr.stage], dr.phase, p.status)))) break;
          tc_fence_after();
          const float s = w4_scale(my_scales[slot * (slot_bytes / 2) + gr * 64], p.scale_half);
          const float2 s2 = make_float2(s, s);
#pragma unroll
          for (int c = 0; c < C::CA; c += 32) {
            float v[32];
            tmem_ld32(taddr + dr.stage * NX + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c / 2 + i] = fma2(s2, make_float2(v[2 * i], v[2 * i + 1]), acc[c / 2 + i]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&dempty[dr.stage]);
          dr.next(2);
        }
        if (++slot == C::SLOTS) slot = 0;
      }
      if (!ok) break;
      if (a.split > 1) {
        // Sums [column][row] in the stages' place: every product and copy of this block is complete.
        float* sums = reinterpret_cast<float*>(smem) + part * C::CA * kM + r;
#pragma unroll
        for (int c = 0; c < C::CA / 2; ++c) {
          sums[(2 * c) * kM] = acc[c].x;
          sums[(2 * c + 1) * kM] = acc[c].y;
        }
        break;  // one tile a cluster
      }
      const int cols = min(C::CA, p.rows - m0);
      if (!a.gated) {
        const int n = (int)packed;
        const bool in = packed < p.n;
        const float bias = in && p.bias ? W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.bias)[n]) : 0.f;
#pragma unroll
        for (int c = 0; c < C::CA; ++c)
          if (in && c < cols) store_linear<HALF>(p, m0 + c, n, c & 1 ? acc[c / 2].y : acc[c / 2].x, bias);
      } else {
        // Rows 0 .. 7 of 16 are gates, 8 .. 15 the up rows of the same outputs: lanes 8 apart exchange, and each has one
        // of two columns.
        const bool up = (r & 8) != 0;
        const int64_t n = (packed >> 4) * 8 + (r & 7);
#pragma unroll
        for (int c = 0; c < C::CA / 2; ++c) {
          const float other = __shfl_xor_sync(0xffffffffu, up ? acc[c].x : acc[c].y, 8);
          const float v = w4_act(up ? other : acc[c].x, p.act) * (up ? acc[c].y : other);
          const int col = 2 * c + (up ? 1 : 0);
          if (n < p.n && col < cols) static_cast<uint16_t*>(p.out)[(int64_t)(m0 + col) * p.n + n] = W4Num<HALF>::from_float(v);
        }
      }
    }
    if (a.split > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      // A share of the columns, in all of the cluster's blocks' sums.
      const int64_t packed0 = (int64_t)(first_tile % a.tiles_n) * kM;
      const int m0 = (first_tile / a.tiles_n) * NX, per = NX / a.split;
      const int outs = a.gated ? 64 : 128;
      const uint32_t base = smem_u32(smem);
      for (int e = threadIdx.x - 128 * (1 + C::ND); e < per * outs; e += 128 * C::NA) {
        const int c = rank * per + e / outs, o = e % outs, m = m0 + c;
        const int64_t n = a.gated ? packed0 / 2 + o : packed0 + o;
        if (m >= p.rows || n >= p.n) continue;
        const int row = a.gated ? (o >> 3) * 16 + (o & 7) : o;
        float v = 0.f, u = 0.f;
        for (int s = 0; s < a.split; ++s) {
          v += ld_cluster(base + (c * kM + row) * 4, s);
          if (a.gated) u += ld_cluster(base + (c * kM + row + 8) * 4, s);
        }
        if (a.gated)
          static_cast<uint16_t*>(p.out)[(int64_t)m * p.n + n] = W4Num<HALF>::from_float(w4_act(v, p.act) * u);
        else
          store_linear<HALF>(p, m, (int)n, v, p.bias ? W4Num<HALF>::to_float(static_cast<const uint16_t*>(p.bias)[n]) : 0.f);
      }
      __syncwarp();
      cluster_arrive();  // no block leaves while another reads its sums
      cluster_wait();
    }
    tc_fence_before();
    named_sync(1, 32 + 128 * C::NA);
  }
}

template <bool HALF, int NX>
cudaError_t launch(const W4Dev& p, int group, bool zeros, bool gated, int split, cudaStream_t st) {
  using C = Cfg<NX>;
  ManyArgs a = {};
  a.p = p;
  a.group = group;
  a.zeros = zeros;
  a.gated = gated;
  a.tile_bytes = w4_tile_bytes(group, zeros);
  a.tiles_n = (p.blocks + 1) / 2;
  const int64_t tiles = (int64_t)a.tiles_n * ((p.rows + NX - 1) / NX);
  if (tiles > (1 << 27)) return cudaErrorInvalidValue;
  a.tiles = (int)tiles;
  a.split = split;
  CUtensorMap map;
  if (!make_tmap_2d(&map, p.x, 2, p.rows, p.k, (uint64_t)p.x_ld * 2, NX, 64)) return cudaErrorInvalidValue;
  const int smem = 1024 + C::STAGES * C::STAGE + kCodeStages * 2 * a.tile_bytes + C::SLOTS * (kW4K / group) * 256 +
                   8 * (3 * C::STAGES + 2 * kCodeStages + 5) + 16;
  if (smem > kMaxSmem) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = smem_attr_once(k_w4_many<HALF, NX>, kMaxSmem, done);
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
  return cudaLaunchKernelEx(&cfg, k_w4_many<HALF, NX>, map, a);
}

template <bool HALF>
cudaError_t pick(const W4Dev& p, int group, bool zeros, bool gated, cudaStream_t st) {
  const int nx = p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : p.rows <= 128 ? 128 : 256;
  const int64_t tiles = (int64_t)((p.blocks + 1) / 2) * ((p.rows + nx - 1) / nx);
  int split = 1;
  while (split < 8 && tiles * split * 2 <= num_sms() && p.tiles_k >= 2 * split) split *= 2;
  if (nx == 32) return launch<HALF, 32>(p, group, zeros, gated, split, st);
  if (nx == 64) return launch<HALF, 64>(p, group, zeros, gated, split, st);
  if (nx == 128) return launch<HALF, 128>(p, group, zeros, gated, split, st);
  return launch<HALF, 256>(p, group, zeros, gated, split, st);
}

}  // namespace

cudaError_t launch_w4_many(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st) {
  return half ? pick<true>(p, group, zeros, gated, st) : pick<false>(p, group, zeros, gated, st);
}

}  // namespace t2w
