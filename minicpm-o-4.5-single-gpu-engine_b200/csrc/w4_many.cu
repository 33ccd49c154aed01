// Products with 4-bit weights for many rows of x on tcgen05: D[128 rows of W][NX rows of x] = (W - zero) x^T, one
// accumulator for each group of k, scaled and summed in registers.
//
// A persistent block an SM takes tiles of 128 k, each in H halves of U = NX / H rows of x:
//   warps 0, 2   x: TMA, 128-byte swizzle, one stage (128 k x U rows) for each half, in turn (with NX = 256 warp 0 alone)
//   warps 1, 3   TMEM, and tcgen05.mma from one lane (M = 128, N = U, K = 16), A from TMEM
//   2 or 4 x 4   warps widen codes to whole 16-bit numbers and store them in TMEM, where they are the A operand; the
//                warpgroups take the tiles in turn, and the first lane of each copies its packed tiles, 128 rows x 128 k (with
//                NX = 256, where widening has no registers to spare, warp 2 does: 461 us for 505 in the largest case measured)
//   H x 4 warps  take a group's accumulator out of TMEM (a few take turns), each lane one row of W: acc += scale * sum, so the
//                scale is a register and no weight is rounded; at a tile's end they write the outputs
//
// The weights go through TMEM because shared memory is what such a kernel runs out of: 128 bytes a clock, of which 128 k of
// widened weights would take 256 clocks to write and 256 to read, where the products take 4 NX clocks.
// What a hand-over costs decides the rest: passing an mbarrier that is ready takes about 100 clocks, a commit 80, the
// issue of 4 products 65, a round of waiting, expecting and one copy 600 (one thread brings 12.9 GB/s in pieces of 4 KB, 26.5 in
// pieces of 8 KB).  So
// copies and products are issued by several warps in turn, and with groups of 128 one barrier tells the products' warp what a
// half waits for (x and a free accumulator; the weights too where there is one half), and one commit tells that its stage is
// free and its accumulator full.
// With few tiles k is split over a cluster, whose blocks add their sums through distributed shared memory in a fixed order.
// The first tiles of W come before the kernel waits for the one ahead of it in the stream.  No TMA multicast.
#include "common.cuh"
#include "kernels.h"
#include "w4.h"

namespace t2w {
namespace {

constexpr int kM = 128;        // rows of W of a tile
constexpr int kMaxCodes = 12;  // packed tile pairs under way
constexpr int kMaxSmem = 232448;
constexpr int kACols = 64;     // TMEM columns of a tile's widened weights
constexpr int kChunk = 8;      // columns that the end of a tile takes at a time

template <int NX>
struct Cfg {
  static constexpr int H = NX == 256 ? 2 : 1;  // halves of a tile, and accumulating warpgroups
  static constexpr int U = NX / H;             // rows of x of a half
  static constexpr int TURNS = NX == 256 ? 2 : 4;  // widening warpgroups
  static constexpr int WIDEN = 4 * TURNS;          // widening warps
  static constexpr int THREADS = 128 * (1 + TURNS + H);
  static constexpr int B_BYTES = U * kW4K * 2;
  static constexpr int STAGES = NX == 256 ? 5 : NX == 128 ? 4 : 6;  // of x
  static constexpr int A_TILES = NX == 256 ? 2 : STAGES;            // widened tiles
  static constexpr int ACCS = NX == 256 ? 3 : 2;                    // accumulators
  static constexpr int SLOTS = A_TILES + 2;                         // tiles whose scales are kept (see the widening warps)
  static constexpr int A_AT = ACCS * U;                             // TMEM column of the first widened tile
  static constexpr int TMEM = 512;
  static constexpr bool LEADS = NX != 256;  // widening warpgroups copy their packed tiles
  static_assert(A_AT + A_TILES * kACols <= TMEM, "tensor memory");
  static_assert(H == 2 || A_TILES == STAGES, "one barrier for both operands");
  // Registers: the sums need more than an even split has, which the other warps give.  The sum of the warpgroups' shares is at
  // most what the kernel is launched with: 96 each of 640 threads, 80 each of 768.
  static constexpr int LAUNCH = NX == 256 ? 96 : 80;
  static constexpr int R_ROLES = 48, R_WIDEN = NX == 256 ? 48 : NX == 128 ? 64 : 72, R_SUM = NX == 256 ? 168 : NX == 128 ? 176 : 144;
  static_assert(R_ROLES + TURNS * R_WIDEN + H * R_SUM <= (1 + TURNS + H) * LAUNCH, "registers");
  static constexpr int fixed(int group) {  // shared memory besides the ring of packed tiles
    return STAGES * B_BYTES + SLOTS * (kW4K / group) * 256 + 8 * (2 * STAGES + 2 * A_TILES + 2 * kMaxCodes + H * ACCS + 2 * ACCS + 2) + 16;
  }
};

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
// A strip of 16 rows, 64 k: four m16n8k16 A fragments side by side.
T2W_DEV void tmem_st_frags(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// D (+)= A B with A from TMEM (two numbers to a 32-bit column) and B from shared memory.
T2W_DEV void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 64 columns by two loads (one of 64 would need more registers than the kernel begins with); the wait is inside the block, so
// that no use of a register can come before it.
T2W_DEV void tmem_ld32x2(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr), "r"(taddr + 32)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
T2W_DEV void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
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
  // One barrier for what a half's products wait for, and one commit for all that wait for them: where a group is a tile.
  constexpr bool kOne = G == kW4K;
  constexpr int kFree = 2 * C::ACCS;  // barriers that tell of a free accumulator, taken in turn (see the issuing warps)
  const int code_bytes = 2 * a.tile_bytes;
  uint8_t* scales = smem + C::STAGES * C::B_BYTES;  // [slot][half][group][64]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + C::SLOTS * slot_bytes);  // x of a half (and with H = 1 the weights)
  uint64_t* empty = full + C::STAGES;                                          // the half's products have ended
  uint64_t* afull = empty + C::STAGES;                                         // H = 2: the weights
  uint64_t* aempty = afull + C::A_TILES;
  uint64_t* cfull = aempty + C::A_TILES;
  uint64_t* cempty = cfull + kMaxCodes;
  uint64_t* dfull = cempty + kMaxCodes;  // (not kOne) [half][accumulator]: a warpgroup waits for its own phases alone
  uint64_t* dempty = dfull + C::H * C::ACCS;
  uint64_t* drain = dempty + kFree;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  uint8_t* codes = smem + (C::fixed(G) + 127) / 128 * 128;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.split > 1 ? (int)cluster_rank() : 0;
  const int first_tile = blockIdx.x / a.split, tile_step = gridDim.x / a.split;
  const Span span = span_of(p.tiles_k, rank, a.split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      // x, the four warps that give the accumulator back, and with one half the four that widen
      mbar_init(&full[s], 1 + (kOne ? 4 : 0) + (C::H == 1 ? 4 : 0));
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < C::A_TILES; ++s) {
      mbar_init(&afull[s], 4);
      mbar_init(&aempty[s], C::H);  // a commit of each warp that issued its products
    }
    for (int s = 0; s < C::ACCS; ++s) {
      for (int h = 0; h < C::H; ++h) mbar_init(&dfull[h * C::ACCS + s], 1);
      mbar_init(&dempty[s], 4);
      mbar_init(&dempty[C::ACCS + s], 4);
    }
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
  }
  // Packed tiles are copied by a widening warpgroup's first lane for that group, or by one lane for all; as many as there is
  // room for before anything is waited for.
  const int len = span.end - span.first, my_turn = (warp - 4) >> 2;
  auto further = [&](int& tile, int& kt, int n) {  // n k tiles on
    kt += n;
    while (kt >= span.end) {
      kt -= len;
      tile += tile_step;
    }
  };
  auto copy_codes = [&](int tile, int kt, int stage) {
    const int rb = (tile % a.tiles_n) * 2, halves = rb + 1 < p.blocks ? 2 : 1;
    mbar_expect_tx(&cfull[stage], halves * a.tile_bytes);
    for (int h = 0; h < halves; ++h)
      bulk_load(codes + stage * code_bytes + h * a.tile_bytes, p.tiles + ((int64_t)(rb + h) * p.tiles_k + kt) * a.tile_bytes,
                a.tile_bytes, &cfull[stage]);
  };
  const bool leads = C::LEADS && warp >= 4 && warp < 4 + C::WIDEN && (threadIdx.x & 127) == 0;
  constexpr int kCopyStep = C::LEADS ? C::TURNS : 1;
  if (C::LEADS ? leads : threadIdx.x == 64) {
    const int from = C::LEADS ? my_turn : 0;
    for (int s = from; s < a.code_stages; s += kCopyStep) {
      mbar_init(&cfull[s], 1);
      mbar_init(&cempty[s], 4);
    }
    fence_mbar_init();
    int tile = first_tile, kt = span.first;
    further(tile, kt, from);
    for (int s = from; s < a.code_stages && tile < a.tiles; s += kCopyStep) {
      copy_codes(tile, kt, s);
      further(tile, kt, kCopyStep);
    }
  }
  __syncwarp();
  if (warp == 1) {
    pdl_wait();  // (the kernel before may hold tensor memory)
    tmem_alloc(tmem_slot, C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    regs_dec<C::R_ROLES>();
    if (!C::LEADS && warp == 2) {
      if (lane == 0) {  // (which copied the first)
        Ring r;
        int tile = first_tile, kt = span.first, t = tile, k = kt;
        further(t, k, a.code_stages);
        bool ok = true;
        for (; t < a.tiles && (ok = w4_wait(&cempty[r.stage], r.phase, p.status)); r.next(a.code_stages)) {
          copy_codes(t, k, r.stage);
          further(t, k, 1);
        }
        if (!ok)  // the stages from this one on are under way, or long since full
          for (int i = 0; i < a.code_stages; ++i, r.next(a.code_stages)) w4_wait(&cfull[r.stage], r.phase, p.status);
      }
      __syncwarp();
    } else if ((warp & 1) == 0) {
      pdl_wait();
      if (elect_one()) {
        constexpr int kBy = C::LEADS ? 2 : 1;
        const int me = warp >> 1;
        Ring r;
        r.stage = me;
        int issued = 0, unit = me;  // halves of the block's tiles of 128 k
        bool ok = true;
        for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step, unit -= len * C::H) {
          const int m0 = (tile / a.tiles_n) * NX;
          for (; unit < len * C::H; unit += kBy) {
            if (!(ok = w4_wait(&empty[r.stage], r.phase ^ 1u, p.status))) break;
            uint8_t* to = smem + r.stage * C::B_BYTES;
            const int k = (span.first + unit / C::H) * kW4K, m = m0 + unit % C::H * C::U;
            mbar_expect_tx(&full[r.stage], C::B_BYTES);
            tma_load_2d(to, &tmX, k, m, &full[r.stage]);
            tma_load_2d(to + C::B_BYTES / 2, &tmX, k + 64, m, &full[r.stage]);
            ++issued;
            r.next(C::STAGES, kBy);
          }
        }
        // The block does not end, nor is its shared memory used for sums, with a copy under way (where a wait gave up).
        if (!ok)
          for (int i = issued > C::STAGES ? issued - C::STAGES : 0; i < issued; ++i) {
            const int u = me + kBy * i;
            w4_wait(&full[u % C::STAGES], (u / C::STAGES) & 1, p.status);
          }
      }
      __syncwarp();
    } else if (warp == 1 || C::H == 2 || kOne) {
      if (warp == 1) pdl_launch();
      // The whole warp goes through the loop, so that descriptors and addresses stay in uniform registers; one lane issues.
      // Two warps take the halves in turn (with one half and groups of 128 the tiles): one waits while the other's products
      // run.  Groups are numbered in the order (tile, group, half); number v has accumulator v % ACCS, free once v - ACCS has
      // been taken, which barrier v % kFree tells (with kOne the half's own).  A wait cannot take a phase before for its own:
      // the last number this warp issued needed one back that was filled later than what the barrier told before.
      constexpr int kIssuers = C::H == 2 || kOne ? 2 : 1;
      const int me = kIssuers == 2 ? warp >> 1 : 0;
      constexpr uint32_t idesc = idesc_16(kM, C::U, HALF);
      // x's descriptor, stage 0: 32 bytes further for each 16 k, a block further for each 64, a stage for each stage.
      const uint64_t bdesc = sdesc_sw128(smem_u32(smem), 1024, 16);
      constexpr int kSteps = G / 16;  // products of a group
      Ring sr, ar, dr, fr, pr;
      sr.stage = dr.stage = fr.stage = me;
      bool ok = true, x_ready = false, a_ready = false;
      // this warp's first k tile, and how far the next one is
      const int from = C::H == 1 ? me : 0, by = C::H == 1 ? kIssuers : 1;
      const int tiles = (a.tiles - first_tile + tile_step - 1) / tile_step;
      for (int64_t it = from, all = (int64_t)tiles * len; it < all; it += by) {
        if (C::H == 2 && !(ok = w4_wait_warp(&afull[ar.stage], ar.phase, p.status, a_ready))) break;
        if (!(ok = w4_wait_warp(&full[sr.stage], sr.phase, p.status, x_ready))) break;
        {
          Ring then = sr;
          then.next(C::STAGES, kIssuers);
          x_ready = mbar_test(smem_u32(&full[then.stage]), then.phase);
          if (C::H == 2) {
            then = ar;
            then.next(C::A_TILES);
            a_ready = mbar_test(smem_u32(&afull[then.stage]), then.phase);
          }
        }
        const uint64_t bd = bdesc + sr.stage * (C::B_BYTES >> 4);
        const uint32_t ad = tmem + C::A_AT + (C::H == 2 ? ar.stage : sr.stage) * kACols;
#pragma unroll
        for (int j = 0; j < groups; ++j) {
          if (!kOne && !(ok = w4_wait_warp(&dempty[fr.stage], fr.phase, p.status))) break;
          tc_fence_after();
          const uint32_t d = tmem + dr.stage * C::U;
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
              const int k = j * kSteps + i;
              umma_ts(d, ad + k * 8, bd + (k >> 2) * (C::B_BYTES / 2 >> 4) + (k & 3) * 2, idesc, i != 0);
            }
            if (!kOne) umma_commit(&dfull[me * C::ACCS + pr.stage]);
            if (j == groups - 1) {
              umma_commit(&empty[sr.stage]);
              if (C::H == 2) umma_commit(&aempty[ar.stage]);
            }
          }
          __syncwarp();
          dr.next(C::ACCS, kIssuers);
          fr.next(kFree, kIssuers);
          pr.next(C::ACCS);
        }
        if (!ok) break;
        sr.next(C::STAGES, kIssuers);
        if (!ok) break;
        ar.next(C::A_TILES);
      }
      if (!ok) {  // TMEM is not given back with a product under way
        if (elect_one()) umma_commit(&drain[me]);
        __syncwarp();
        w4_wait_warp(&drain[me], 0, p.status);
      }
      if (kIssuers == 2) named_sync(3, 64);
    }
    if (a.split > 1) cluster_pass();
    if (warp == 1) {
      named_sync(1, 32 + 128 * C::H);
      tc_fence_after();
      tmem_dealloc(tmem, C::TMEM);
    }
  } else if (warp < 4 + C::WIDEN) {
    regs_dec<C::R_WIDEN>();
    // The warpgroups take the tiles in turn; warp w has lanes 32 w .. 32 w + 31 of TMEM: strips 2 w and 2 w + 1 of the 128 rows.
    const int w = (warp - 4) & 3, mine = my_turn, g = lane >> 2, half = w >> 1;
    const int my_codes = half * a.tile_bytes + (w & 1) * 2048 + lane * 16;
    const int my_zeros = half * a.tile_bytes + kW4Codes + groups * 128 + g * 8 + (w & 1) * 4;
    const uint32_t to = tmem + C::A_AT + ((uint32_t)(w * 32) << 16);
    uint64_t* free_a = C::H == 2 ? aempty : empty;
    uint64_t* told = C::H == 2 ? afull : full;
    Ring cr, ar;
    int slot = mine % C::SLOTS, tile = first_tile, kt = span.first;
    further(tile, kt, mine);
    for (int i = 0; i < mine; ++i) {
      cr.next(a.code_stages);
      ar.next(C::A_TILES);
    }
    auto next_c = [&](Ring& r) { r.next(a.code_stages, C::TURNS); };
    auto next_a = [&](Ring& r) { r.next(C::A_TILES, C::TURNS); };
    bool ok = true, c_ready = false, a_ready = false;
    for (; tile < a.tiles; further(tile, kt, C::TURNS)) {
      const int halves = (tile % a.tiles_n) * 2 + 1 < p.blocks ? 2 : 1;
      if (!(ok = w4_wait_warp(&cfull[cr.stage], cr.phase, p.status, c_ready))) break;
      const uint8_t* in = codes + cr.stage * code_bytes;
      // Read before it is widened, where there are registers for it: a strip of 16 rows x 64 k is 16 bytes of a lane.
      constexpr bool kAhead = NX != 256;
      uint4 c[2][2];
      uint32_t z[2][groups];
      if (half < halves) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
            if (kAhead) c[s][b] = *reinterpret_cast<const uint4*>(in + my_codes + s * 1024 + b * 512);
#pragma unroll
          for (int i = 0; i < groups; ++i)
            z[s][i] = a.zeros ? *reinterpret_cast<const uint16_t*>(in + my_zeros + s * 2 + i * 64) : 0x0808;
        }
      }
      if (!(ok = w4_wait_warp(&free_a[ar.stage], ar.phase ^ 1u, p.status, a_ready))) break;
      tc_fence_after();
      {  // a look at what this warpgroup's next tile waits for
        Ring then = cr;
        next_c(then);
        c_ready = mbar_test(smem_u32(&cfull[then.stage]), then.phase);
        then = ar;
        next_a(then);
        a_ready = mbar_test(smem_u32(&free_a[then.stage]), then.phase ^ 1u);
      }
      // The scales move to a slot of their own.  The slot's last tile was SLOTS = A_TILES + 2 tiles ago; the products of the
      // tile that had this place have ended, so an accumulator was free when the last of them began, so the
      // sums of every tile at least 2 before it are taken.
      {
        const int i = w * 32 + lane, h = i / (groups * 8), j = i % (groups * 8);
        if (h < halves)
          reinterpret_cast<uint4*>(scales + slot * slot_bytes + h * groups * 128)[j] =
              reinterpret_cast<const uint4*>(in + h * a.tile_bytes + kW4Codes)[j];
      }
      if (kAhead) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&cempty[cr.stage]);
      }
      if (half < halves) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (!kAhead) c[s][b] = *reinterpret_cast<const uint4*>(in + my_codes + s * 1024 + b * 512);
            uint32_t v[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t zz = z[s][(b * 64 + j * 16) / G];
              uint32_t x[4];
              w4_widen<HALF>((&c[s][b].x)[j], w4_zero<HALF>(zz & 255), w4_zero_hi<HALF>(zz >> 8), x);
              v[4 * j] = x[0];  // row g, k and k + 2; row g + 8
              v[4 * j + 1] = x[2];
              v[4 * j + 2] = x[1];
              v[4 * j + 3] = x[3];
            }
            tmem_st_frags(to + ar.stage * kACols + ((uint32_t)(s * 16) << 16) + b * 32, v);
          }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&told[ar.stage]);
        if (!kAhead) mbar_arrive(&cempty[cr.stage]);
      }
      if (C::LEADS && leads) {  // the tile's place is filled again once all four warps have read it
        int t = tile, k = kt;
        further(t, k, a.code_stages);
        if (t < a.tiles && (ok = w4_wait(&cempty[cr.stage], cr.phase, p.status))) copy_codes(t, k, cr.stage);
      }
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      next_a(ar);
      next_c(cr);
      if ((slot += C::TURNS) >= C::SLOTS) slot -= C::SLOTS;
    }
    if (C::LEADS && !ok && leads)  // no copy is under way when the block ends (where a wait gave up)
      for (int i = 0; i < a.code_stages && tile < a.tiles; i += C::TURNS, next_c(cr), further(tile, kt, C::TURNS))
        w4_wait(&cfull[cr.stage], cr.phase, p.status);
    __syncwarp();
    if (a.split > 1) {
      if constexpr (NX == 256) {
        cluster_pass();
      } else {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        finish_cluster<HALF, NX>(a, smem, first_tile, rank, threadIdx.x - 128, 128 * (C::TURNS + C::H));
        __syncwarp();
        cluster_arrive();
        cluster_wait();
      }
    }
  } else {
    regs_inc<C::R_SUM>();
    const int w = warp - 4 - C::WIDEN, part = w >> 2, r = (warp & 3) * 32 + lane;  // half of the tile, row of W in it
    // With kOne a half's accumulator is full when its products have ended.  One that has been taken is free for the number
    // ACCS later, whose barrier is told; the first ACCS are free from the start (told by the warpgroup whose turn it would be).
    constexpr int kTold = kOne ? C::STAGES : kFree;
    uint64_t* told = kOne ? full : dempty;
    if (lane == 0) {
#pragma unroll
      for (int v = 0; v < C::ACCS; ++v)
        if ((v + C::ACCS) % C::H == part) mbar_arrive(&told[v]);
    }
    pdl_wait();
    const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint16_t* my_scales = reinterpret_cast<const uint16_t*>(scales + (r >> 6) * groups * 128) + w4_place(r & 63);
    Ring dr, er, pr;
    er.stage = dr.stage = part;
    int tell = (part + C::ACCS) % kTold, slot = 0;
    auto give_back = [&]() {  // the accumulator taken last
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&told[tell]);
      if ((tell += C::H) >= kTold) tell -= kTold;
    };
    bool ok = true, ready = false;
    for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step) {
      const int m0 = (tile / a.tiles_n) * NX + part * C::U;
      const int64_t packed = (int64_t)(tile % a.tiles_n) * kM + r;  // row of the packed weight
      float acc[C::U];
      int held = 0;  // the last group's accumulator
#pragma unroll
      for (int c = 0; c < C::U; ++c) acc[c] = 0.f;
      for (int kt = span.first; kt < span.end && ok; ++kt) {
        for (int gr = 0; gr < groups; ++gr) {
          // (with a look at the next one's barrier)
          if (kOne) {
            if (!(ok = w4_wait_warp(&empty[er.stage], er.phase, p.status, ready))) break;
            er.next(C::STAGES, C::H);
            ready = mbar_test(smem_u32(&empty[er.stage]), er.phase);
          } else {
            if (!(ok = w4_wait_warp(&dfull[part * C::ACCS + pr.stage], pr.phase, p.status, ready))) break;
            pr.next(C::ACCS);
            ready = mbar_test(smem_u32(&dfull[part * C::ACCS + pr.stage]), pr.phase);
          }
          tc_fence_after();
          const float s = w4_scale(my_scales[slot * (slot_bytes / 2) + gr * 64], p.scale_half);
          const float2 s2 = make_float2(s, s);
          constexpr int kLoad = C::U == 64 ? 64 : 32;
#pragma unroll
          for (int c = 0; c < C::U; c += kLoad) {
            float v[kLoad];
            if constexpr (kLoad == 64) {
              tmem_ld32x2(taddr + dr.stage * C::U, v);
            } else {
              tmem_ld32(taddr + dr.stage * C::U + c, v);
            }
#pragma unroll
            for (int i = 0; i < kLoad; i += 2) {
              const float2 q = fma2(s2, make_float2(v[i], v[i + 1]), make_float2(acc[c + i], acc[c + i + 1]));
              acc[c + i] = q.x;
              acc[c + i + 1] = q.y;
            }
          }
          held = dr.stage;
          if (a.split > 1 || kt + 1 < span.end || gr + 1 < groups) give_back();
          dr.next(C::ACCS, C::H);
        }
        if (++slot == C::SLOTS) slot = 0;
      }
      const int cols = min(C::U, p.rows - m0);
      if (a.split > 1) {  // one tile a cluster
        // [column][row] in the stages' place: every product and copy of this block is complete (of both halves, once both
        // warpgroups are here; each comes, also where a wait gave up, and waits for nothing that the other has to give).
        if (C::H == 2) named_sync(2, 128 * C::H);
        float* sums = reinterpret_cast<float*>(smem) + part * C::U * kM + r;
#pragma unroll
        for (int c = 0; c < C::U; ++c) sums[c * kM] = acc[c];
        break;
      }
      if (!ok) break;
      // The sums go into the accumulator taken last and come back a few columns at a time: what follows is a short loop
      // then, where all columns in a row would be ten thousand bytes of code that no instruction cache has in time.
      const uint32_t own = taddr + held * C::U;
#pragma unroll
      for (int c = 0; c < C::U; c += 32) tmem_st32(own + c, acc + c);
      tmem_st_wait();
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
        for (int c0 = 0; c0 < C::U; c0 += kChunk) {
          float v[kChunk];
          __syncwarp();  // (lanes without outputs have gone other ways)
          tmem_ld8(own + c0, v);
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
        for (int c0 = 0; c0 < C::U; c0 += kChunk) {
          float v[kChunk];
          __syncwarp();
          tmem_ld8(own + c0, v);
#pragma unroll
          for (int c = 0; c < kChunk; c += 2) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[c] : v[c + 1], 8);
            const float y = w4_act(up ? other : v[c], p.act) * (up ? v[c + 1] : other);
            if (c0 + c < count) out[(int64_t)(c0 + c) * p.n] = W4Num<HALF>::from_float(y);
          }
        }
      }
      give_back();
    }
    if (a.split > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      constexpr int kThreads = NX == 256 ? 128 * C::H : 128 * (C::TURNS + C::H);  // the widening warps help where they have registers
      finish_cluster<HALF, NX>(a, smem, first_tile, rank, (int)threadIdx.x - (C::THREADS - kThreads), kThreads);
      __syncwarp();
      cluster_arrive();  // no block leaves while another reads its sums
      cluster_wait();
    }
    tc_fence_before();
    named_sync(1, 32 + 128 * C::H);
  }
}

// Tiles of 128 rows of W x nx rows of x.
constexpr int64_t tiles_of(int blocks, int rows, int nx) { return ((int64_t)blocks + 1) / 2 * (((int64_t)rows + nx - 1) / nx); }
static_assert(tiles_of(1, 0x7fffffff, 256) == 1 << 23 && tiles_of(3, 257, 256) == 4, "as many rows as a call may have");

template <bool HALF, int NX, int G>
int many_smem(bool zeros) {
  const int tile = w4_tile_bytes(G, zeros), fixed = (Cfg<NX>::fixed(G) + 127) / 128 * 128;
  // as many packed tiles under way as there is room for, in whole turns: so each has its warpgroup, which sees all its phases
  const int room = (kMaxSmem - fixed) / (2 * tile), stages = (room < kMaxCodes ? room : kMaxCodes) / Cfg<NX>::TURNS * Cfg<NX>::TURNS;
  return fixed + stages * 2 * tile;
}

// Clusters of `split` blocks that are resident at once.
template <bool HALF, int NX, int G>
int room_for(int split, bool zeros) {
  static std::atomic<uint64_t> done{0};
  if (smem_attr_once(k_w4_many<HALF, NX, G>, kMaxSmem, done) != cudaSuccess) return 0;
  static ClusterRoom room;
  return cluster_room(k_w4_many<HALF, NX, G>, split, Cfg<NX>::THREADS, many_smem<HALF, NX, G>(zeros), room);
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
  const int64_t tiles = tiles_of(p.blocks, p.rows, NX);
  if (tiles > (1 << 27)) return cudaErrorInvalidValue;
  a.tiles = (int)tiles;
  a.split = split;
  CUtensorMap map;
  if (!make_tmap_2d(&map, p.x, 2, p.rows, p.k, (uint64_t)p.x_ld * 2, C::U, 64)) return cudaErrorInvalidValue;
  const int smem = many_smem<HALF, NX, G>(zeros);
  a.code_stages = (smem - (C::fixed(G) + 127) / 128 * 128) / (2 * a.tile_bytes);
  if (a.code_stages < 2 * C::TURNS) return cudaErrorInvalidValue;
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

// The tile's width and the split of k with the least time by a rule of thumb (us, groups of 128): a tile of 128 k is taken to
// cost 0.45 for NX = 32, 0.47 for 64, 0.73 for 128 and 0.87 for 256 (with groups of 64 1.2 and of 32 1.7 times that), the
// end of a block's tile 1.5 to 5, and the cluster's joining 1.5 more.  Measured, in one round of 148 tiles: 0.43, 0.48, 0.61 and
// 0.77; with groups of 64 1.3 to 1.5 times that and of 32 1.9 to 2.4 times, so the rule is kind to narrow groups, all widths
// alike.  Blocks of a cluster have one tile, so all clusters have to be resident at once.
struct Choice {
  int nx = 0, split = 1;
  int64_t cost = INT64_MAX;
};
template <bool HALF, int NX, int G>
void consider(const W4Dev& p, bool zeros, Choice& best) {
  constexpr int kTile = (NX == 32 ? 45 : NX == 64 ? 47 : NX == 128 ? 73 : 87) * (G == 32 ? 17 : G == 64 ? 12 : 10) / 10, kEnd = NX == 32 ? 150 : NX == 64 ? 200 : NX == 128 ? 300 : 500;
  const int64_t tiles = tiles_of(p.blocks, p.rows, NX);
  for (int s = 1; s <= 8 && p.tiles_k >= 2 * s; s *= 2) {
    if (s > 1 && tiles > room_for<HALF, NX, G>(s, zeros)) break;
    const int64_t rounds = s > 1 ? 1 : (tiles + num_sms() - 1) / num_sms();
    const int64_t cost = rounds * ((int64_t)((p.tiles_k + s - 1) / s) * kTile + kEnd) + (s > 1 ? 150 : 0);
    if (cost < best.cost) best = {NX, s, cost};
  }
  if (p.tiles_k == 1) {  // (nothing to split)
    const int64_t cost = (tiles + num_sms() - 1) / num_sms() * (kTile + kEnd);
    if (cost < best.cost) best = {NX, 1, cost};
  }
}

template <bool HALF, int G>
cudaError_t pick(const W4Dev& p, bool zeros, bool gated, cudaStream_t st) {
  Choice best;
  consider<HALF, 32, G>(p, zeros, best);
  if (p.rows > 32) consider<HALF, 64, G>(p, zeros, best);
  if (p.rows > 64) consider<HALF, 128, G>(p, zeros, best);
  if (p.rows > 128) consider<HALF, 256, G>(p, zeros, best);
  if (best.nx == 32) return launch<HALF, 32, G>(p, zeros, gated, best.split, st);
  if (best.nx == 64) return launch<HALF, 64, G>(p, zeros, gated, best.split, st);
  if (best.nx == 128) return launch<HALF, 128, G>(p, zeros, gated, best.split, st);
  return launch<HALF, 256, G>(p, zeros, gated, best.split, st);
}
template <bool HALF>
cudaError_t pick_group(const W4Dev& p, int group, bool zeros, bool gated, cudaStream_t st) {
  if (group == 32) return pick<HALF, 32>(p, zeros, gated, st);
  if (group == 64) return pick<HALF, 64>(p, zeros, gated, st);
  return pick<HALF, 128>(p, zeros, gated, st);
}

}  // namespace

cudaError_t launch_w4_many(const W4Dev& p, int group, bool zeros, bool gated, bool half, cudaStream_t st) {
  return half ? pick_group<true>(p, group, zeros, gated, st) : pick_group<false>(p, group, zeros, gated, st);
}

}  // namespace t2w
