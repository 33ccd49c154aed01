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
// Two blocks an SM, each 3 warpgroups: warps 0-3 softmax (a thread a row), 4-7 widen, 8 the MMA issuer (9-11 only give up
// their registers: 128 a softmax thread, 72 and 40 the others, of the 80 each that the block is launched with).  Warps
// 4-7 copy the codes of the tiles ahead into a ring of their own with asynchronous copies, a thread its own pieces, and write them as halves in the
// 128-byte swizzle that the tensor core reads.  K and V tiles have rings of their own, since a K tile is free as soon as
// its scores are there.  A segment's output is finished during the next segment's first tile.
//
// What bounds it: for windows of some ten rows HBM (the codes are read once; 8 KB a tile at 64 columns), for longer
// chunks the exponentials: 16 a clock and SM, 512 clocks a tile, against 256 (head_dim 64) or 512 (128) of the tensor
// core.
#include "paged_attn.cuh"

namespace t2w {
namespace {

constexpr int kRows = 128, kKeys = 64;
constexpr int kThreads = 384, kWiden = 128;  // threads; of them widening
constexpr int kTmem = 256;                   // S / W buffers at 0 and 64, O at 128

// Rings by head_dim: query buffers, K and V tiles of halves, tiles of codes on their way.
template <int HD>
struct Rings {
  static constexpr int Q = HD == 64 ? 2 : 1, K = HD == 64 ? 2 : 1, V = HD == 64 ? 2 : 1, Raw = HD == 64 ? 4 : 2;
  static constexpr int q_bytes = kRows * HD * 2, tile_bytes = kKeys * HD * 2, raw_bytes = 2 * kKeys * HD;
  static constexpr int k_at = Q * q_bytes, v_at = k_at + K * tile_bytes, raw_at = v_at + V * tile_bytes;
  static constexpr int aux_at = raw_at + Raw * raw_bytes;
};
struct Aux {
  uint64_t q_full[2], q_free[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2], o_free;
  uint64_t meta_full[4];  // by tile: ks, vs, and for a segment's first tile c_row
  uint32_t tmem;
  int pad;
  float c_row[4][kRows];  // by segment: scale * log2 e / the power of two that the row's queries were multiplied by
  float ks[4][4], vs[4][4];  // by tile: the scales of its 16-key chunks
  float scale_raw[4][8];     // the same on their way
};

T2W_DEV void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
T2W_DEV void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
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
T2W_DEV void cp16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
T2W_DEV void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// A worker's walk over its segments: every role makes it for itself.
struct Walk {
  int r, hk, qt;       // the segment
  int row0, f, kv;     // its request's first row, rows and keys
  int kt0, kt1, nt;    // the tiles of it that are this worker's, and all of them
  int zero, stop;      // the place of its tile 0; the end of the worker's places
  int extra;
  bool first;

  T2W_DEV void cut(const AttnDev& p, int from) {
    nt = seg_tiles(tile_keys(f, kv, p.causal, p.tq, qt), kKeys);
    kt0 = from;
    kt1 = min(nt, stop - zero);
  }
  T2W_DEV bool begin(const AttnDev& p, int w) {
    const int4 h = *reinterpret_cast<const int4*>(p.head);  // n_runs, places, per, workers
    const int4 s = p.starts[2 * w], of = p.starts[2 * w + 1];
    extra = p.head->extra;
    if (w >= h.w) return false;
    r = s.x;
    hk = s.y;
    qt = s.z;
    row0 = of.x;
    f = of.y;
    kv = of.z;
    stop = min((w + 1) * h.z, h.y);
    zero = w * h.z - s.w;
    first = true;
    cut(p, max(s.w, 0));
    return kt0 < kt1;
  }
  T2W_DEV bool next(const AttnDev& p) {
    if (kt1 < nt) return false;
    zero += nt + extra;
    if (zero >= stop) return false;
    first = false;
    if (++qt * p.tq >= f) {
      qt = 0;
      if (++hk == p.kv_heads) {
        hk = 0;
        do {
          r++;
          row0 = p.q_start[r];
          f = p.q_start[r + 1] - row0;
        } while (f == 0);  // places are left, so there is a request with rows
        kv = p.kv_len[r];
      }
    }
    cut(p, 0);
    return true;
  }
  // rows of the segment
  T2W_DEV int tokens(const AttnDev& p) const { return min(p.tq, f - qt * p.tq); }
};

template <int HD, bool HALF>
__global__ void __launch_bounds__(kThreads, 2) k_paged_many(const AttnDev p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using R = Rings<HD>;
  Aux* const x = reinterpret_cast<Aux*>(smem + R::aux_at);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = blockIdx.x, group = p.q_heads / p.kv_heads;
  constexpr int kPanels = HD / 64;
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
    for (int i = 0; i < 4; ++i) mbar_init(&x->meta_full[i], 4);
    mbar_init(&x->o_free, 4);
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
  Walk at;
  bool ok = at.begin(p, w);

  if (warp >= 4 && warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---------------- widening: 128 threads, thread i has the 16-byte pieces i, i + 128, ... of a tile's codes
    const int i = threadIdx.x - 128;
    constexpr int kPieces = HD / 16, kN = kKeys * kPieces / kWiden, kStep = kWiden / kPieces;  // pieces a row, a thread; rows between
    const int row_i = i / kPieces, piece = i % kPieces;
    const uint64_t policy = l2_policy_evict_first();
    const uint32_t raw0 = smem_u32(smem + R::raw_at) + 16 * i;
    Walk ahead = at;  // the tile that is sent for next
    int kt_a = at.kt0, sent = 0;
    bool live = ok;
    auto send = [&]() {
      if (live) {
        const int slot = sent % R::Raw;
        const int* const table = p.table + (size_t)ahead.r * p.table_ld;
        const int kb = kt_a * kKeys;
        auto page_of = [&](int key) {
          const int g = __ldg(table + (key >> p.shift));
          if ((unsigned)g < (unsigned)p.pages) return (long long)g;
          atomicExch(p.status, T2W_ERR_INVALID);
          return 0ll;
        };
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const int key = kb + row_i + j * kStep;
          if (key < ahead.kv) {
            const long long g = page_of(key);
            const long long in = ((long long)ahead.hk * p.page + (key & (p.page - 1))) * HD + 16 * piece;
            const uint32_t dst = raw0 + slot * R::raw_bytes + j * (16 * kWiden);
            cp16(dst, p.codes[0] + g * p.page_ld[0] + in, policy);
            cp16(dst + kKeys * HD, p.codes[1] + g * p.page_ld[1] + in, policy);
          }
        }
        if (i < 8) {  // chunk i & 3's scale of K or V; a chunk past the last key takes the first one's
          const int key = kb + 16 * (i & 3), y = i >> 2;
          if (kb < ahead.kv) {
            const long long g = page_of(key < ahead.kv ? key : kb);
            cp4(smem_u32(&x->scale_raw[slot][i]), p.scales[y] + g * p.scale_ld[y] + ahead.hk);
          } else {
            x->scale_raw[slot][i] = 1.f;
          }
        }
        ++sent;
        if (++kt_a == ahead.kt1) {
          live = ahead.next(p);
          kt_a = 0;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int j = 0; j < R::Raw - 1; ++j) send();
    int t = 0;  // tiles so far
    for (int s = 0; ok; ++s) {
      // queries: thread i has row i
      {
        const int qb = s % R::Q, tokens = at.tokens(p), tok = i / group;
        const bool has = tok < tokens;
        const uint16_t* const q = static_cast<const uint16_t*>(p.q) + (long long)(at.row0 + at.qt * p.tq + tok) * p.q_row_ld +
                                  (at.hk * group + i % group) * p.q_head_ld;
        uint4 v[HD / 8];
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          v[c] = has ? __ldg(reinterpret_cast<const uint4*>(q) + c) : make_uint4(0, 0, 0, 0);
          m = __vmaxu2(__vmaxu2(m, v[c].x & 0x7fff7fffu), v[c].y & 0x7fff7fffu);
          m = __vmaxu2(__vmaxu2(m, v[c].z & 0x7fff7fffu), v[c].w & 0x7fff7fffu);
        }
        const int sh = row_shift<HALF>(max(m & 0xffffu, m >> 16));
        if (!(ok = __all_sync(~0u, mbar_wait(&x->q_free[qb], ((s / R::Q) & 1) ^ 1u, p.status)))) break;
        uint8_t* const dst = smem + qb * R::q_bytes + i * 128;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          const bool neg = p.scale < 0.f;
          const uint4 u = make_uint4(row_half2<HALF>(v[c].x, sh, neg), row_half2<HALF>(v[c].y, sh, neg),
                                     row_half2<HALF>(v[c].z, sh, neg), row_half2<HALF>(v[c].w, sh, neg));
          *reinterpret_cast<uint4*>(dst + (c >> 3) * (kRows * 128) + (((c & 7) ^ (i & 7)) << 4)) = u;
        }
        x->c_row[s & 3][i] = scaled(fabsf(p.scale) * kLog2e, -sh);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&x->q_full[qb]);
      }
      for (int kt = at.kt0; kt < at.kt1; ++kt, ++t) {
        send();  // into the slot of the tile before this one
        asm volatile("cp.async.wait_group %0;" ::"n"(R::Raw - 1) : "memory");
        const uint8_t* const raw = smem + R::raw_at + (t % R::Raw) * R::raw_bytes + 16 * i;
        if (i < 8) (i < 4 ? x->ks : x->vs)[t & 3][i & 3] = x->scale_raw[t % R::Raw][i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&x->meta_full[t & 3]);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int n = y ? R::V : R::K, slot = t % n;
          if (!(ok = __all_sync(~0u, mbar_wait(y ? &x->v_empty[slot] : &x->k_empty[slot], ((t / n) & 1) ^ 1u, p.status)))) break;
          uint8_t* const dst = smem + (y ? R::v_at : R::k_at) + slot * R::tile_bytes;
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            const int row = row_i + j * kStep;
            uint4 c = *reinterpret_cast<const uint4*>(raw + y * (kKeys * HD) + j * (16 * kWiden));
            // places past the last key may hold anything; a weight of 0 does not hide a NaN value
            if (y && kt * kKeys + row >= at.kv) c = make_uint4(0, 0, 0, 0);
            const uint2 a = e4m3x4_to_f16x4(c.x), b = e4m3x4_to_f16x4(c.y), d = e4m3x4_to_f16x4(c.z), e = e4m3x4_to_f16x4(c.w);
            uint8_t* const to = dst + (piece >> 2) * (kKeys * 128) + row * 128;
            const int c0 = (piece & 3) * 2;
            *reinterpret_cast<uint4*>(to + ((c0 ^ (row & 7)) << 4)) = make_uint4(a.x, a.y, b.x, b.y);
            *reinterpret_cast<uint4*>(to + (((c0 + 1) ^ (row & 7)) << 4)) = make_uint4(d.x, d.y, e.x, e.y);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(y ? &x->v_full[slot] : &x->k_full[slot]);
        }
        if (!ok) break;
      }
      if (!ok || !at.next(p)) break;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // ---------------- MMA issuer: S_0, S_1, then W_t V_t followed by S_{t + 2}
    if (warp == 8 && lane == 0 && ok) {
      constexpr uint32_t idesc_qk = idesc_half(kRows, kKeys), idesc_pv = idesc_half(kRows, 64, true);
      Walk pv = at;  // the segment of the next W V; `at` is that of the next S
      int js = at.kt0, ts = 0, seg = 0, jp = pv.kt0, tp = 0, segp = 0;
      bool more_s = true, more_p = true;
      auto issue_s = [&]() -> bool {
        if (js == at.kt0 && !mbar_wait(&x->q_full[seg % R::Q], (seg / R::Q) & 1, p.status)) return false;
        if (!mbar_wait(&x->k_full[ts % R::K], (ts / R::K) & 1, p.status)) return false;
        tc_fence_after();
        const uint32_t q0 = smem_u32(smem + (seg % R::Q) * R::q_bytes);
        const uint32_t k0 = smem_u32(smem + R::k_at + (ts % R::K) * R::tile_bytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_f16(tmem + 64 * (ts & 1), sdesc_sw128(q0 + (kk >> 2) * (kRows * 128) + 32 * (kk & 3), 1024, 16),
                   sdesc_sw128(k0 + (kk >> 2) * (kKeys * 128) + 32 * (kk & 3), 1024, 16), idesc_qk, kk ? 1u : 0u);
        umma_commit(&x->s_full[ts & 1]);
        umma_commit(&x->k_empty[ts % R::K]);
        ++ts;
        if (++js == at.kt1) {
          umma_commit(&x->q_free[seg % R::Q]);
          more_s = at.next(p);
          js = 0;
          ++seg;
        }
        return true;
      };
      for (int i = 0; i < 2 && more_s && ok; ++i) ok = issue_s();
      while (more_p && ok) {
        if (!(ok = mbar_wait(&x->p_full[tp & 1], (tp >> 1) & 1, p.status))) break;
        if (!(ok = mbar_wait(&x->v_full[tp % R::V], (tp / R::V) & 1, p.status))) break;
        // a segment's first W V overwrites O: the softmax has read the previous segment's
        if (jp == pv.kt0 && segp > 0 && !(ok = mbar_wait(&x->o_free, (segp - 1) & 1, p.status))) break;
        tc_fence_after();
        const uint32_t v0 = smem_u32(smem + R::v_at + (tp % R::V) * R::tile_bytes);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
          for (int c = 0; c < kPanels; ++c)
            umma_f16_ts(tmem + 128 + 64 * c, tmem + 64 * (tp & 1) + 8 * kk,
                        sdesc_sw128(v0 + c * (kKeys * 128) + kk * 16 * 128, 1024, 8192), idesc_pv,
                        (jp > pv.kt0 || kk > 0) ? 1u : 0u);
        umma_commit(&x->o_done[tp & 1]);
        umma_commit(&x->v_empty[tp % R::V]);
        ++tp;
        if (++jp == pv.kt1) {
          more_p = pv.next(p);
          jp = 0;
          ++segp;
        }
        if (more_s) ok = issue_s();
      }
    }
  } else {
    // ---------------- softmax: thread r has row r
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    const int r = threadIdx.x;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t oreg = tmem + lanes + 128;
    int t = 0;
    struct Pending {
      int row, head, t_last, slot;  // output row (-1: none), query head; the part's slot, or -1 for a whole segment
      float l, M;
    } pend{-1, 0, 0, -1, 0.f, 0.f};
    bool have = false;
    auto finish = [&]() -> bool {
      if (!__all_sync(~0u, mbar_wait(&x->o_done[pend.t_last & 1], (pend.t_last >> 1) & 1, p.status))) return false;
      tc_fence_after();
      const float l = pend.l, M = l != l ? fmaxf(pend.M, -1e30f) : pend.M;  // a NaN counts, even where M saw nothing else
      float* const part = part_of(p.ws, pend.slot, kRows, HD);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        float o[32];
        tmem_ld32(oreg + 32 * c, o);
        if (c == HD / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&x->o_free);
        }
        if (pend.row >= 0 && pend.slot < 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) store_row8<HALF>(p, pend.row, pend.head, HD, 32 * c + i, o + i, M, l);
        } else if (pend.row >= 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(part + r * HD + 32 * c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
        __syncwarp();
      }
      if (pend.row >= 0 && pend.slot >= 0) {
        part[kRows * HD + r] = M;
        part[kRows * HD + kRows + r] = l;
      }
      return true;
    };
    for (int s = 0; ok; ++s) {
      const int tok = r / group, keys = at.tokens(p) > tok ? 1 : 0;
      const int pos = at.qt * p.tq + tok;  // the row's query in its request
      // keys that the row sees
      const int lim = !keys ? 0 : p.causal ? at.kv - at.f + pos + 1 : at.kv;
      const bool idle = __all_sync(~0u, !keys);  // its rows' weights and outputs are never read
      float c_row = 0.f;
      float M = -INFINITY, l = 0.f;
      for (int kt = at.kt0; kt < at.kt1; ++kt, ++t) {
        if (!(ok = __all_sync(~0u, mbar_wait(&x->meta_full[t & 3], (t >> 2) & 1, p.status) &&
                                       mbar_wait(&x->s_full[t & 1], (t >> 1) & 1, p.status))))
          break;
        tc_fence_after();
        if (kt == at.kt0) c_row = x->c_row[s & 3][r];
        const uint32_t sbuf = tmem + lanes + 64 * (t & 1);
        if (!idle) {
          uint32_t sr[64];
          tmem_ld32_nowait(sbuf, sr);
          tmem_ld32_nowait(sbuf + 32, sr + 32);
          float ck[4], lv[4], unit[4];
          bool odd = false;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float ks = x->ks[t & 3][c], vs = x->vs[t & 3][c];
            odd |= !(ks < INFINITY) || !(vs < INFINITY);
            const bool bad = !(vs < INFINITY);
            const int e = bad ? 0 : (int)(__float_as_uint(vs) >> 23) - 127;
            ck[c] = c_row * ks;
            if (ck[c] == 0.f) ck[c] = 1.1754944e-38f;  // (-inf times 0)
            lv[c] = (float)e;
            unit[c] = exp2i(-e);
          }
          tmem_ld_wait();
          const int kb = kt * kKeys;
          if (!__all_sync(~0u, kb + kKeys <= lim)) {
#pragma unroll
            for (int i = 0; i < kKeys; ++i)
              if (kb + i >= lim) sr[i] = __float_as_uint(-INFINITY);
          }
          if (odd) {  // a scale that is not finite: it may only meet what the row sees
#pragma unroll
            for (int i = 0; i < kKeys; ++i)
              if (kb + i < lim) sr[i] = __float_as_uint(fmaf(__uint_as_float(sr[i]), ck[i >> 4], lv[i >> 4]));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              ck[c] = 1.f;
              lv[c] = 0.f;
            }
          }
          float mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float m = fmax3(__uint_as_float(sr[16 * c]), __uint_as_float(sr[16 * c + 1]), __uint_as_float(sr[16 * c + 2]));
#pragma unroll
            for (int i = 3; i < 15; i += 2)
              m = fmax3(m, __uint_as_float(sr[16 * c + i]), __uint_as_float(sr[16 * c + i + 1]));
            m = fmaxf(m, __uint_as_float(sr[16 * c + 15]));
            mx = fmaxf(mx, fmaf(m, ck[c], lv[c]));
          }
          const bool raise = mx > M + kRaise;
          const float m_old = M;
          M = raise ? mx - kBelow : M;
          const float ref = M == -INFINITY ? 0.f : M;
          uint32_t u[32];
          float add = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float2 c2 = make_float2(ck[c], ck[c]), d2 = make_float2(lv[c] - ref, lv[c] - ref);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 a = fma2(make_float2(__uint_as_float(sr[16 * c + 2 * i]), __uint_as_float(sr[16 * c + 2 * i + 1])), c2, d2);
              const float2 e = make_float2(exp2_approx(a.x), exp2_approx(a.y));
              sum = add2(sum, e);
              u[8 * c + i] = pack_f16x2(e.x, e.y);
            }
            add = fmaf(sum.x + sum.y, unit[c], add);
          }
          if (odd) {  // values that are NaN, where the row sees them
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(x->vs[t & 3][i >> 3] < INFINITY)) {
                if (kb + 2 * i < lim) u[i] |= 0x7fffu;
                if (kb + 2 * i + 1 < lim) u[i] |= 0x7fff0000u;
              }
          }
          tmem_st32(sbuf, u);
          if (kt > at.kt0 && __any_sync(~0u, raise)) {
            // O holds the tiles before relative to the old exponent; S_t's completion implies that of every product
            // issued before it, so the waits skipped here never fall two phases behind
            if (!(ok = __all_sync(~0u, mbar_wait(&x->o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, p.status)))) break;
            tc_fence_after();
            const float f = raise ? exp2_approx(m_old - M) : 1.f;
            l *= f;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              float o[32];
              tmem_ld32(oreg + 32 * c, o);
              uint32_t ou[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) ou[i] = __float_as_uint(o[i] * f);
              tmem_st32(oreg + 32 * c, ou);
            }
          }
          l += add;
          tmem_st_wait();
        }
        if (kt == at.kt0 && have) {
          if (!(ok = finish())) break;
          have = false;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&x->p_full[t & 1]);
      }
      if (!ok) break;
      pend.row = keys ? at.row0 + pos : -1;
      pend.head = at.hk * group + r % group;
      pend.t_last = t - 1;
      pend.slot = at.kt0 == 0 && at.kt1 == at.nt ? -1 : 2 * w + (at.first ? 0 : 1);
      pend.l = l;
      pend.M = M;
      have = true;
      if (!at.next(p)) break;
    }
    if (ok && have) finish();
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
