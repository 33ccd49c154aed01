// Attention over the paged 8-bit cache for more than 16 query rows to a key head, on tcgen05 tensor cores.
//
// A segment is (request, key head, query tile): its 128 rows are tq = 128 / group query tokens with their `group` heads,
// so that a key head's codes are read and widened once for all its query heads.  Keys come in tiles of 64:
//   S_t = Q K_t^T (M 128, N 64, K head_dim) into S buffer t % 2 of TMEM;
//   the row's thread reads its 64 scores, keeps the exponent M of x_j + log2 s_v (see paged_attn.cuh; when it is raised, the
//   row's O in TMEM is multiplied), and writes the weights as
//   halves back over the scores;
//   O += W_t V_t (M 128, N 64 for each 64 columns, K 64, W from TMEM, V MN-major).
//
// Operands are halves: e4m3 codes widen to them exactly, a page's scales go into the exponent of the row's 16-column
// chunks (a page holds 16 keys at least), and bf16 queries are brought into their range by a power of two for each row.
// fp8 operands would spare the widening, but not the rounding of queries and weights to 4 bits.
//
// Two blocks an SM, each three warpgroups.  Warps 0-3 softmax, a thread a row; a segment's output is finished during the
// next segment's first tile.  Warps 4-7 widen: they write a tile's codes as halves in the 128-byte swizzle that the tensor
// core reads, K a tile ahead of V, and bring a segment's queries.  Warp 8 issues the products, warp 10 walks the segments
// and sends for the tiles ahead (a bulk copy for each page).  Of the 80 registers that a thread of the block is launched
// with, the three warpgroups take 128, 56 and 56.
//
// What was in the way, in the order it was found (4 requests of 700 to 1024 tokens over histories to 4096, 16 query and 4
// key heads, head_dim 128): queries brought by one warp of their own, 20,000 clocks a segment (185 us, of which it was
// 30); code that does not fit the instruction caches, 62 KB at first, so that the roles are kept short (16-byte
// pieces read ahead while widening: 138 to 150); descriptors made for each product by a lane that the compiler could not
// know to be alone (152 us before, 148 after); spills of the products' warp (138 to 135).  Without the registers' split (96
// for each of 10 warps) it was 158.
//
// Segments of at most 64 rows (windows) lie in the upper rows of every other block's tiles: a warp's exponentials run on
// the SM quarter that its TMEM lanes belong to, and so the two blocks of an SM use all four.
//
// What bounds it: a tile takes an SM 1950 clocks.  The exponentials (16 a clock and SM) need 512 of them, the tensor core
// 256 (head_dim 64) or 512 (128), shared memory about 1100 (the products read queries, keys and values from it, and every
// code passes through it twice); 900 instructions issue on each of the SM's quarters, from two softmax and two widening
// warps, which is too few to hide what each waits for.  The chunks above: 130 us, 447 TFLOP/s, 26% of cuBLAS's bf16 rate.
#include "paged_attn.cuh"

namespace t2w {
namespace {

constexpr int kRows = 128, kKeys = 64;
constexpr int kThreads = 384;
constexpr int kTmem = 256;  // S / W buffers at 0 and 64, O at 128

// Rings by head_dim: query buffers, K and V tiles of halves, and tiles of codes on their way (Ahead; a tile's K codes are
// kept until they are widened, its V codes one step longer).
template <int HD>
struct Rings {
  static constexpr int Q = HD == 64 ? 2 : 1, K = HD == 64 ? 2 : 1, V = HD == 64 ? 2 : 1, Ahead = HD == 64 ? 3 : 1;
  static constexpr int RawK = Ahead + 1, RawV = Ahead + 2;
  static constexpr int q_bytes = kRows * HD * 2, tile_bytes = kKeys * HD * 2, raw_bytes = kKeys * HD;
  static constexpr int k_at = Q * q_bytes, v_at = k_at + K * tile_bytes, raw_k_at = v_at + V * tile_bytes;
  static constexpr int raw_v_at = raw_k_at + RawK * raw_bytes, aux_at = raw_v_at + RawV * raw_bytes;
};
// A segment, as the copies' warp tells the others; rows == 0: there are no more.
struct Seg {
  int row0, rows, head0;   // first token row, rows, first query head
  int before, kv;          // keys ahead of the first token's own (causal), keys
  int kt0, kt1, slot;      // key tiles; the part's slot, or -1 for a whole segment
};
constexpr int kMetas = 8, kSegs = 16;  // tiles' scales and segments that the copies' warp may have told (see Aux)
struct Aux {
  uint64_t q_full[2], q_free[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2];
  uint64_t o_free, idle;
  uint64_t meta_full[kMetas], shift_full[4];  // by tile: ks, vs; by segment: shift
  uint64_t raw_full[4], raw_k_empty[4], raw_v_empty[5], seg_full[kSegs];
  uint32_t tmem;
  int pad;
  // By tile: the scales of its 16-key chunks.  Tile t is sent for once V of t - RawV has been widened, that is once the
  // product of t - RawV - V is done and the softmax may read what belongs to the tile behind that.  Tile t - 1's scales are
  // told then: RawV + V - 2 tiles (5 at most) ahead of it.
  float ks[kMetas][4], lv[kMetas][4], unit[kMetas][4];  // K's; log2 of V's (0 where that is not finite) and 2^-lv
  uint32_t odd[kMetas];
  // By segment.  One that begins with tile t is told before that tile waits for anything, when the product of t - 1 - RawV -
  // V is done.  The softmax may then still have to look up, for that tile's rows, the segment it ended: where segments are of
  // one tile, RawV + V + 1 segments (8 where head_dim is 64) lie between the two.
  Seg seg[kSegs];
  int16_t shift[4][kRows];   // by segment: the power of two that a row's queries were multiplied by
};

T2W_DEV void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
T2W_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (+)= A B with A from TMEM (two halves to a 32-bit column) and B from shared memory.
T2W_DEV void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor, kind::f16: D fp32, A and B halves, A K-major.
__host__ __device__ constexpr uint32_t idesc_half(int M, int N, bool b_mn_major = false) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// mbar_wait() in as few instructions as it takes: each of the roles goes round its loop once a tile, and what of it is not
// in the instruction cache costs more than the wait's looser look at the time.
T2W_DEV bool bar_wait(uint64_t* bar, uint32_t parity, int* err) {
  const uint32_t a = smem_u32(bar);
  unsigned long long t0 = 0;
  for (uint32_t i = 1; !mbar_try_wait(a, parity); ++i) {
    if (i & 1023u) continue;
    const unsigned long long now = globaltimer();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      atomicExch(err, T2W_ERR_TIMEOUT);
      return false;
    }
  }
  return true;
}
// One lane of a converged warp: said so, the compiler need not expect several lanes' descriptors behind a product.
T2W_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p;
}
T2W_DEV void copy16_plain(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
T2W_DEV void bulk_load_hint(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// The tile row that a segment's first row has.
T2W_DEV int base_of(int rows) { return rows <= 64 && 2 * blockIdx.x >= gridDim.x ? 64 : 0; }

template <int HD, bool HALF>
__global__ void __launch_bounds__(kThreads, 2) k_paged_many(const AttnDev p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using R = Rings<HD>;
  Aux* const x = reinterpret_cast<Aux*>(smem + R::aux_at);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = blockIdx.x, group = p.group;
  constexpr int kPanels = HD / 64;
  static_assert(R::RawV + R::V - 2 < kMetas && R::RawV + R::V + 1 < kSegs, "nothing is told over what may still be read");
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&x->q_full[i], 4);
      mbar_init(&x->q_free[i], 1);
      mbar_init(&x->k_full[i], 4);
      mbar_init(&x->k_empty[i], 1);
      mbar_init(&x->v_full[i], 4);
      mbar_init(&x->v_empty[i], 1);
      mbar_init(&x->s_full[i], 1);
      mbar_init(&x->p_full[i], 4);
      mbar_init(&x->o_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&x->shift_full[i], 4);
      mbar_init(&x->raw_full[i], 1);
      mbar_init(&x->raw_k_empty[i], 4);
    }
    for (int i = 0; i < 5; ++i) mbar_init(&x->raw_v_empty[i], 4);
    for (int i = 0; i < kMetas; ++i) mbar_init(&x->meta_full[i], 1);
    for (int i = 0; i < kSegs; ++i) mbar_init(&x->seg_full[i], 1);
    mbar_init(&x->o_free, 4);
    mbar_init(&x->idle, 1);
    fence_mbar_init();
  }
  pdl_wait();
  if (warp == 8) {
    tmem_alloc(&x->tmem, kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch();
  const uint32_t tmem = x->tmem;
  bool ok = true;
  auto next_seg = [&](int s) -> const Seg* {  // nullptr: none, or the wait gave up
    if (!bar_wait(&x->seg_full[s & (kSegs - 1)], (s & kSegs) != 0, p.status)) {
      ok = false;
      return nullptr;
    }
    const Seg* const g = &x->seg[s & (kSegs - 1)];
    return g->rows ? g : nullptr;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 8) {
      // ---------------- S_n, then W V of tile n - 1 (the products of one thread are in order: S_n writes over W_{n-2})
      if (elect_one()) {
        constexpr uint32_t idesc_s = idesc_half(kRows, kKeys), idesc_o = idesc_half(kRows, 64, true);
        int s = -1, left = 0;              // the segment of S_n, and its tiles from n on
        int sp = 0;                        // the segment of tile n - 1, and whether that tile is its first
        bool first_p = false;
        const Seg* g = nullptr;
        for (int n = 0; ok; ++n) {
          const bool had = n > 0;
          if (left <= 1) {
            g = next_seg(++s);
            left = g ? g->kt1 - g->kt0 : 0;
            if (!ok || (g && !bar_wait(&x->q_full[s % R::Q], (s / R::Q) & 1, p.status))) break;
          } else {
            --left;
          }
          const bool first_n = g && left == g->kt1 - g->kt0;
          if (g) {
            if (!bar_wait(&x->k_full[n % R::K], (n / R::K) & 1, p.status)) break;
            tc_fence_after();
            // (the address field of a descriptor counts 16 bytes)
            const uint64_t q0 = sdesc_sw128(smem_u32(smem + (s % R::Q) * R::q_bytes), 1024, 16);
            const uint64_t k0 = sdesc_sw128(smem_u32(smem + R::k_at + (n % R::K) * R::tile_bytes), 1024, 16);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              umma_f16(tmem + 64 * (n & 1), q0 + (kk >> 2) * (kRows * 8) + 2 * (kk & 3), k0 + (kk >> 2) * (kKeys * 8) + 2 * (kk & 3),
                       idesc_s, kk ? 1u : 0u);
            umma_commit(&x->s_full[n & 1]);
            umma_commit(&x->k_empty[n % R::K]);
            if (left == 1) umma_commit(&x->q_free[s % R::Q]);
          }
          if (had) {
            const int t = n - 1;
            if (!bar_wait(&x->v_full[t % R::V], (t / R::V) & 1, p.status) || !bar_wait(&x->p_full[t & 1], (t >> 1) & 1, p.status)) break;
            // a segment's first product overwrites O: the softmax has read the previous segment's
            if (first_p && sp > 0 && !bar_wait(&x->o_free, (sp - 1) & 1, p.status)) break;
            tc_fence_after();
            const uint64_t v0 = sdesc_sw128(smem_u32(smem + R::v_at + (t % R::V) * R::tile_bytes), 1024, 8192);
#pragma unroll
            for (int c = 0; c < kPanels; ++c)
#pragma unroll
              for (int kk = 0; kk < kKeys / 16; ++kk)
                umma_f16_ts(tmem + 128 + 64 * c, tmem + 64 * (t & 1) + 8 * kk,
                            v0 + c * (kKeys * 8) + kk * 128, idesc_o, !first_p || kk ? 1u : 0u);
            umma_commit(&x->o_done[t & 1]);
            umma_commit(&x->v_empty[t % R::V]);
          }
          if (!g) break;
          first_p = first_n;
          sp = s;
        }
        umma_commit(&x->idle);
      }
      __syncwarp();
      bar_wait(&x->idle, 0, p.status);  // no product is under way when the block ends, not where a wait gave up either
    } else if (warp == 10) {
      // ---------------- segments, codes and scales: lane x * 4 + c has the c-th page of a tile's K (x 0) or V, and chunk
      // c's scale
      const int unit = min(p.page, kKeys), c = lane & 3, y = (lane >> 2) & 1;  // keys of a copy
      int t = 0, pg = 0, pg_scale = 0;
      auto page = [&](int g) -> long long {
        if ((unsigned)g < (unsigned)p.pages) return g;
        atomicExch(p.status, T2W_ERR_INVALID);
        return 0;
      };
      float scale = 0.f;  // of the tile before, which is on its way while that tile's codes are
      auto publish = [&](int n) {
        const bool odd = !(scale < INFINITY);
        const int e = odd ? 0 : (int)(__float_as_uint(scale) >> 23) - 127;
        const uint32_t of = __ballot_sync(~0u, lane < 8 && odd);
        if (lane < 4) x->ks[n & (kMetas - 1)][c] = scale;
        else if (lane < 8) x->lv[n & (kMetas - 1)][c] = (float)e, x->unit[n & (kMetas - 1)][c] = exp2i(-e);
        else if (lane == 8) x->odd[n & (kMetas - 1)] = (of >> 4 & 15u) | (of & 15u ? 16u : 0u);
        __syncwarp();
        if (lane == 0) mbar_arrive(&x->meta_full[n & (kMetas - 1)]);
      };
      const uint64_t policy = l2_policy_evict_first();
      Walk at;
      bool more = at.begin(p, w);
#pragma unroll 1
      for (int s = 0;; ++s) {
        if (lane == 0) {
          Seg* const g = &x->seg[s & (kSegs - 1)];
          g->rows = more ? at.rows(p, group) : 0;
          g->row0 = at.row0 + at.qt * p.tq;
          g->head0 = at.hk * group;
          g->before = at.kv - at.f + at.qt * p.tq;
          g->kv = at.kv;
          g->kt0 = at.kt0;
          g->kt1 = at.kt1;
          g->slot = at.kt0 == 0 && at.kt1 == at.nt ? -1 : 2 * w + (at.first ? 0 : 1);
          mbar_arrive(&x->seg_full[s & (kSegs - 1)]);
        }
        if (!more) break;
#pragma unroll 1
        for (int kt = at.kt0 - 1; kt < at.kt1; ++kt) {
          // (a pass before the first tile only looks up its pages)
          if (kt >= at.kt0) {
            const int kb = kt * kKeys, sk = t % R::RawK, sv = t % R::RawV;
            ok = bar_wait(&x->raw_k_empty[sk], ((t / R::RawK) & 1) ^ 1u, p.status) &&
                 bar_wait(&x->raw_v_empty[sv], ((t / R::RawV) & 1) ^ 1u, p.status);
            if (!(ok = __all_sync(~0u, ok))) break;
            const int units = max(0, min((at.kv - kb + unit - 1) / unit, kKeys / unit));
            if (lane == 0) mbar_expect_tx(&x->raw_full[sk], 2 * units * unit * HD);
            __syncwarp();
            if (lane < 8 && c < units) {
              const int key = kb + c * unit;
              bulk_load_hint(smem + (y ? R::raw_v_at + sv * R::raw_bytes : R::raw_k_at + sk * R::raw_bytes) + c * unit * HD,
                             p.codes[y] + page(pg) * p.page_ld[y] + ((long long)at.hk * p.page + (key & (p.page - 1))) * HD,
                             unit * HD, &x->raw_full[sk], policy);
            }
            if (t) publish(t - 1);
            scale = lane < 8 && kb < at.kv ? __ldg(p.scales[y] + page(pg_scale) * p.scale_ld[y] + at.hk) : 1.f;
            ++t;
          }
          if (kt + 1 < at.kt1) {
            const int* const table = p.table + (size_t)at.r * p.table_ld;
            const int kb = (kt + 1) * kKeys, key = kb + c * unit, key_s = kb + 16 * c;
            pg = lane < 8 && c * unit < kKeys && key < at.kv ? __ldg(table + (key >> p.shift)) : 0;
            pg_scale = lane < 8 && kb < at.kv ? __ldg(table + ((key_s < at.kv ? key_s : kb) >> p.shift)) : 0;
          }
        }
        if (!ok) break;
        more = at.next(p);
      }
      if (ok && t) publish(t - 1);
      // nor is a copy
      for (int n = max(0, t - R::RawK); n < t; ++n) bar_wait(&x->raw_full[n % R::RawK], (n / R::RawK) & 1, p.status);
    }
  } else if (warp >= 4) {
    // ---------------- widening: thread i has the 16-byte pieces i, i + 128, ... of a tile's K and of its V codes
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int i = threadIdx.x - 128;
    constexpr int kPieces = HD / 16, kN = kKeys * kPieces / 128, kStep = 128 / kPieces;  // pieces a row, a thread; rows between
    // Of 8 threads, whose 16 bytes are read or written together, the even row's four read the pieces of one half of the row
    // and the odd row's those of the other (HD 128): neither the codes nor the halves meet in a bank.
    const int row_i = HD == 64 ? i / 4 : 2 * (i / 16) + ((i >> 2) & 1);
    const int piece = HD == 64 ? i % 4 : (i & 3) + 4 * (((i >> 3) ^ (i >> 2)) & 1), c0 = (piece & 3) * 2;
    // the queries of a segment that begins at tile t are copied as they are to where their halves go, a thread a row, while
    // K of tile t is widened
    constexpr int kQPieces = HD / 8;
    auto q_place = [&](int c) { return (c >> 3) * (kRows * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4); };
    // K of tile t, then V of tile t - 1
    int s = 0, kt = 0, left = 0;  // the keys from the tile before's first one on
    const Seg* g = next_seg(0);
    if (g) kt = g->kt0;
#pragma unroll 1
    for (int t = 0; ok; ++t) {
      const bool enter = g && kt == g->kt0;
      const int qb = s % R::Q;
      uint8_t* const q_row = smem + qb * R::q_bytes;
      bool has = false, used = false;  // this thread's row, one of its warp's
      if (enter) {
        if (!(ok = __all_sync(~0u, bar_wait(&x->q_free[qb], ((s / R::Q) & 1) ^ 1u, p.status)))) break;
        const int row = i - base_of(g->rows), tok = over_group(p, max(row, 0));
        has = row >= 0 && row < g->rows;
        used = __any_sync(~0u, has);
        if (has) {
          const uint16_t* const from = static_cast<const uint16_t*>(p.q) + (long long)(g->row0 + tok) * p.q_row_ld +
                                       (long long)(g->head0 + row - group * tok) * p.q_head_ld;
#pragma unroll
          for (int c = 0; c < kQPieces; ++c) copy16_plain(smem_u32(q_row + q_place(c)), from + 8 * c);
        }
      }
      if (g && !(ok = bar_wait(&x->raw_full[t % R::RawK], (t / R::RawK) & 1, p.status))) break;
#pragma unroll 1
      for (int y = g ? 0 : 1; y < (t ? 2 : 1); ++y) {
        const int n = t - y, ring = y ? R::V : R::K, slot = n % ring;
        if (!(ok = bar_wait(y ? &x->v_empty[slot] : &x->k_empty[slot], ((n / ring) & 1) ^ 1u, p.status))) break;
        const uint8_t* const raw =
            smem + (y ? R::raw_v_at + (n % R::RawV) * R::raw_bytes : R::raw_k_at + (n % R::RawK) * R::raw_bytes) + row_i * HD + 16 * piece;
        uint8_t* const dst = smem + (y ? R::v_at : R::k_at) + slot * R::tile_bytes + (piece >> 2) * (kKeys * 128) + row_i * 128;
        const int x0 = (c0 ^ (row_i & 7)) << 4;  // (rows kStep apart are the same in the swizzle's 8)
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          uint4 c = *reinterpret_cast<const uint4*>(raw + j * 2048);
          // places past the last key may hold anything; a weight of 0 does not hide a NaN value
          if (y && row_i + j * kStep >= left) c = make_uint4(0, 0, 0, 0);
          const uint2 a = e4m3x4_to_f16x4(c.x), b = e4m3x4_to_f16x4(c.y), d = e4m3x4_to_f16x4(c.z), e = e4m3x4_to_f16x4(c.w);
          *reinterpret_cast<uint4*>(dst + j * (kStep * 128) + x0) = make_uint4(a.x, a.y, b.x, b.y);
          *reinterpret_cast<uint4*>(dst + j * (kStep * 128) + (x0 ^ 16)) = make_uint4(d.x, d.y, e.x, e.y);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(y ? &x->v_full[slot] : &x->k_full[slot]);
          mbar_arrive(y ? &x->raw_v_empty[n % R::RawV] : &x->raw_k_empty[n % R::RawK]);
        }
        if (enter && y == 0) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          if (used) {  // (of a warp without a row nobody reads the scores)
            uint32_t m = 0;
#pragma unroll 4
            for (int c = 0; c < kQPieces; ++c) {
              const uint4 v = has ? *reinterpret_cast<const uint4*>(q_row + q_place(c)) : make_uint4(0, 0, 0, 0);
              m = __vmaxu2(__vmaxu2(m, v.x & 0x7fff7fffu), v.y & 0x7fff7fffu);
              m = __vmaxu2(__vmaxu2(m, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu);
            }
            const int sh = row_shift<HALF>(max(m & 0xffffu, m >> 16));
            const bool neg = p.scale < 0.f;
#pragma unroll 2
            for (int c = 0; c < kQPieces; ++c) {
              uint4* const to = reinterpret_cast<uint4*>(q_row + q_place(c));
              const uint4 v = has ? *to : make_uint4(0, 0, 0, 0);
              *to = make_uint4(row_half2<HALF>(v.x, sh, neg), row_half2<HALF>(v.y, sh, neg), row_half2<HALF>(v.z, sh, neg),
                               row_half2<HALF>(v.w, sh, neg));
            }
            x->shift[s & 3][i] = (int16_t)sh;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&x->q_full[qb]);
            mbar_arrive(&x->shift_full[s & 3]);
          }
        }
      }
      if (!ok || !g) break;
      left = g->kv - kt * kKeys;
      if (++kt == g->kt1) {
        g = next_seg(++s);
        if (g) kt = g->kt0;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---------------- softmax: thread r has the tile's row r
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    const int r = threadIdx.x;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16, oreg = tmem + lanes + 128;
    // the segment (kt: its next tile), the row's keys, factor, exponent and sum
    int s = -1, kt = 0, kt1 = 0, row = 0, lim = 0;
    bool mine = false, idle = true, have = false;
    float c_row = 0.f, M = -INFINITY, l = 0.f;
    // the segment before: output row (-1: none), query head; the part's slot (-1: a whole segment) and row
    int o_row = -1, o_head = 0, o_slot = -1, o_part = 0;
    float o_M = 0.f, o_l = 0.f;
    const Seg* g = nullptr;
#pragma unroll 1
    for (int t = 0; ok; ++t) {
      const bool first = kt == kt1;
      if (first) {
        if (s >= 0) {
          o_row = mine ? g->row0 + over_group(p, row) : -1;
          o_head = g->head0 + row - group * over_group(p, row);
          o_slot = g->slot;
          o_part = row;
          o_M = l != l ? fmaxf(M, -1e30f) : M;  // a NaN counts, even where M saw nothing else
          o_l = l;
          have = true;
        }
        g = next_seg(++s);
        if (!ok) break;
        if (g) {
          kt = g->kt0;
          kt1 = g->kt1;
          row = r - base_of(g->rows);
          mine = row >= 0 && row < g->rows;
          // keys that it sees (a row that nobody reads sees all, so that a warp's others need no mask for it)
          lim = mine && p.causal ? g->before + over_group(p, row) + 1 : g->kv;
          idle = !__any_sync(~0u, mine);  // nobody reads such a warp's weights and outputs
          if (!(ok = bar_wait(&x->shift_full[s & 3], (s >> 2) & 1, p.status))) break;
          c_row = scaled(fabsf(p.scale) * kLog2e, -x->shift[s & 3][r]);
          M = -INFINITY;
          l = 0.f;
        }
      }
      if (g) {
        ok = bar_wait(&x->meta_full[t & (kMetas - 1)], (t & kMetas) != 0, p.status) && bar_wait(&x->s_full[t & 1], (t >> 1) & 1, p.status);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
      }
      if (g && !idle) {
        const uint32_t sbuf = tmem + lanes + 64 * (t & 1);
        const int kb = kt * kKeys;
        const float* const ks = x->ks[t & (kMetas - 1)];
        const uint32_t odd = x->odd[t & (kMetas - 1)];  // 1 << c: chunk c's value scale is not finite; 16: a key scale
        float ck[4], lv[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          ck[c] = c_row * ks[c];
          if (ck[c] == 0.f) ck[c] = 1.1754944e-38f;  // (-inf times 0)
          lv[c] = x->lv[t & (kMetas - 1)][c];
        }
        float w[2][32];
        tmem_ld32(sbuf, w[0]);
        tmem_ld32(sbuf + 32, w[1]);
        uint32_t v[64];  // the scores, then two weights each
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = __float_as_uint(w[i >> 5][i & 31]);
        // scores that the row does not see, and all of them where a scale is not finite: it may only meet what a row sees
        if (!__all_sync(~0u, kb + kKeys <= lim) || odd) {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            float f = __uint_as_float(v[i]);
            if (odd) f = fmaf(f, c_row * ks[i >> 4], lv[i >> 4]);
            v[i] = __float_as_uint(kb + i < lim ? f : -INFINITY);
          }
          if (odd) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              ck[c] = 1.f;
              lv[c] = 0.f;
            }
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t* const u = v + 16 * c;
          float m = fmax3(__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]));
#pragma unroll
          for (int i = 3; i < 15; i += 2) m = fmax3(m, __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
          mx = fmaxf(mx, fmaf(fmaxf(m, __uint_as_float(u[15])), ck[c], lv[c]));
        }
        const bool raise = mx > M + kRaise;
        const float m_old = M;
        M = raise ? mx - kBelow : M;
        const float ref = M == -INFINITY ? 0.f : M;
        float add = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 2 * h; c < 2 * h + 2; ++c) {
            const float d = lv[c] - ref;
            float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
            for (int i = 16 * c; i < 16 * c + 16; i += 4) {
              const float2 a = __ffma2_rn(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])),
                                          make_float2(ck[c], ck[c]), make_float2(d, d));
              const float2 b = __ffma2_rn(make_float2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])),
                                          make_float2(ck[c], ck[c]), make_float2(d, d));
              const float2 ea = make_float2(exp2_approx(a.x), exp2_approx(a.y)), eb = make_float2(exp2_approx(b.x), exp2_approx(b.y));
              s0 = __fadd2_rn(s0, ea);
              s1 = __fadd2_rn(s1, eb);
              v[i / 2] = pack_f16x2(ea.x, ea.y);
              v[i / 2 + 1] = pack_f16x2(eb.x, eb.y);
            }
            add = fmaf((s0.x + s1.x) + (s0.y + s1.y), x->unit[t & (kMetas - 1)][c], add);
          }
          if (odd) {  // values that are NaN, where the row sees them
#pragma unroll
            for (int i = 16 * h; i < 16 * h + 16; ++i)
              if (odd >> (i >> 3) & 1u)
                v[i] |= (kb + 2 * i < lim ? 0x7fffu : 0u) | (kb + 2 * i + 1 < lim ? 0x7fff0000u : 0u);
          }
          uint32_t u[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) u[i] = v[16 * h + i];
          tmem_st16(sbuf + 16 * h, u);
        }
        if (!first && __any_sync(~0u, raise)) {
          // O holds the tiles before relative to the old exponent
          if (!(ok = __all_sync(~0u, bar_wait(&x->o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, p.status)))) break;
          tc_fence_after();
          const float f = raise ? exp2_approx(m_old - M) : 1.f;
          l *= f;
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            float o[16];
            tmem_ld16(oreg + c, o);
            uint32_t ou[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) ou[i] = __float_as_uint(o[i] * f);
            tmem_st16(oreg + c, ou);
          }
        }
        l += add;
        tmem_st_wait();
      }
      if (first && have) {  // the segment before is finished
        if (!(ok = __all_sync(~0u, bar_wait(&x->o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, p.status)))) break;
        tc_fence_after();
        float* const part = part_of(p.ws, o_slot, kRows, HD);
        const float inv = o_l != 0.f ? 1.f / o_l : 0.f;
        uint16_t* const out = static_cast<uint16_t*>(p.out) + ((size_t)o_row * p.q_heads + o_head) * HD;
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          float o[16];
          tmem_ld16(oreg + c, o);
          if (o_row >= 0 && o_slot < 0) {
            uint32_t u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = o[2 * i] * inv, b = o[2 * i + 1] * inv;
              u[i] = HALF ? pack_f16x2(a, b) : pack_bf16x2(a, b);
            }
            reinterpret_cast<uint4*>(out + c)[0] = make_uint4(u[0], u[1], u[2], u[3]);
            reinterpret_cast<uint4*>(out + c)[1] = make_uint4(u[4], u[5], u[6], u[7]);
          } else if (o_row >= 0) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<float4*>(part + o_part * HD + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&x->o_free);
        if (o_row >= 0 && o_slot >= 0) {
          part[kRows * HD + o_part] = o_M;
          part[kRows * HD + kRows + o_part] = o_l;
        } else if (o_row >= 0 && p.lse) {
          p.lse[(size_t)o_row * p.q_heads + o_head] = o_l != 0.f ? (o_M + log2f(o_l)) * 0.6931471805599453f : -INFINITY;
        }
        have = false;
      }
      if (!g) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&x->p_full[t & 1]);
      ++kt;
    }
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmem);
  }
}

template <int HD, bool HALF>
cudaError_t launch_many(const AttnDev& p, const PagedCut& cut, cudaStream_t st) {
  constexpr int smem = Rings<HD>::aux_at + (int)sizeof(Aux);
  static_assert(2 * (smem + 1024) <= 228 * 1024, "two blocks an SM");
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = smem_attr_once(k_paged_many<HD, HALF>, smem, done);
  return e != cudaSuccess ? e : launch_k(k_paged_many<HD, HALF>, dim3(cut.workers), dim3(kThreads), smem, st, p);
}

}  // namespace

cudaError_t launch_paged_many(const AttnDev& p, const PagedCut& cut, int head_dim, bool half, cudaStream_t st) {
  if (head_dim == 64) return half ? launch_many<64, true>(p, cut, st) : launch_many<64, false>(p, cut, st);
  return half ? launch_many<128, true>(p, cut, st) : launch_many<128, false>(p, cut, st);
}

}  // namespace t2w
