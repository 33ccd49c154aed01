// Attention over the paged 8-bit cache.
//
// Mathematics: row i of request r and query head h sees the keys j < end(i) of key head h / group, with end(i) the
// request's key count, or where the call is causal the count less the queries behind i; x_j = scale q . k_j, and
// o = sum_j 2^(c x_j - m) v_j / sum_j 2^(c x_j - m), c = log2 e, with the running maximum m of one pass over the keys.
// A row that sees no key gives zeros and the log-sum -inf.
#include "paged_attn.cuh"

namespace t2w {
namespace {

T2W_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ---------------------------------------------------------------- at most 16 query rows to a key head
//
// What bounds it: the cache is read once, 2 HD bytes for each key against 4 HD flops a query row, so HBM does.  A
// worker is one warp with a contiguous share of the key tiles (32 keys), so that nothing waits for another warp; only
// where one segment fills the shares of a whole block do its 8 warps join what they have, so that a long history comes
// to an eighth of the parts.
//
// A tile's bytes come to the warp's own ring in shared memory by asynchronous copies, one tile or two ahead across the
// ends of segments, and from there in the tensor core's fragments.  Scores: Q is the A operand (16 rows x 16 dims; a
// thread's four dims of a step are any four that K's fragment has in the same place, so a thread takes 16 consecutive
// bytes of a key's row with one load), K the B operand (16 dims x 8 keys).  Output: O^T = V^T P^T, the scores'
// accumulator layout being that of P^T as B operand; V^T as A operand wants two keys' bytes of one dim in a register,
// which one byte permute of two rows' words gives.  So each byte is widened once (e4m3 to half, exact) and in a register.
// The 16-byte pieces of a 128-byte line are permuted (swizzle()) so that neither K's reads (8 rows' pieces t) nor V's (4
// rows two apart, piece g) meet in a bank.
//
// Exponents: key j with scales s_k, s_v of its page weighs 2^(x_j + log2 s_v - M) on its V codes, M a little
// below the running maximum of x_j + log2 s_v (kBelow): the weights of the largest contributions have all the bits that a
// half has whatever the scales.  The sum of exponentials is kept in units of 2^M too.
//
// Measured: 64 requests of 40 to 4100 keys, 32 query and 8 key heads of 128: 272.6 MB in 59 us, 4.6 TB/s (72% of a copy);
// 3 requests of 90k to 150k keys, 16 and 2 heads: 184.5 MB in 45 us, 4.1 TB/s.  In the second the stream itself, between a
// worker's first tile and its last, runs at 7.5 TB/s; the rest is the launch, the plan's and the table's loads ahead of the
// first tile (5 us), the last workers' ends (3) and the joining (6).  Of the other splits, a block of 8 warps on one
// segment at a time took 167 and 68 us in its best form (short segments leave most of it idle), fragments loaded straight
// from global memory 75 and 54, rings of 2 or 6 tiles 66 and 49 or 76 and 52 (this one then 61 and 42 to 46).
template <int HD>
struct FewStage {
  uint8_t k[32 * HD], v[32 * HD];
  float ks[2], vs[2];  // of the tile's two halves
};
template <int HD>
T2W_DEV uint32_t swizzle(int row, int piece) {  // byte offset of 16-byte piece `piece` of row `row`
  if constexpr (HD == 128) return row * 128 + ((piece ^ (((row >> 1) & 3) << 1) ^ ((row & 1) << 2)) << 4);
  const int line = row >> 1;
  return line * 128 + ((((row & 1) * 4 + piece) ^ ((line & 3) << 1)) << 4);
}
T2W_DEV void copy16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
T2W_DEV void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// A lane's places in a stage: of what it copies of 1024 bytes of K or of V rows (of the first and the second 512, which
// repeat), of K's row g piece t (the pieces of the second 64 dims are 64 bytes on or back: xor), and of V's rows 2t and
// 2t + 1 piece g (8 bytes of it where HD is 64).
template <int HD>
T2W_DEV void stage_places(uint32_t (&put)[2], uint32_t& get_k, uint32_t (&get_v)[2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    put[i] = swizzle<HD>(i * (512 / HD) + lane / (HD / 16), lane % (HD / 16)) - i * 512;
    get_v[i] = 32 * HD + (HD == 128 ? swizzle<HD>(2 * t + i, g) : swizzle<HD>(2 * t + i, g >> 1) + 8 * (g & 1));
  }
  get_k = swizzle<HD>(g, t);
}

// A warp's 8 NQ query rows of a segment: thread (g, t) = (lane / 4, lane % 4) has of rows g, g + 8, ... what the scores'
// tiles give it, and columns 2t, 2t + 1 (+ 8 ...) of the transposed output.
template <int HD, int NQ>
struct Rows {
  uint32_t qa[HD / 16][4];         // queries as halves, as A operands
  float c[NQ];                     // scale * log2 e / the power of two that the row's queries were multiplied by
  int end[NQ];                     // keys that the row sees
  float M[NQ], l[NQ], o[NQ][HD / 16][4];
};
// Rows first .. of the segment that begins at row row0 and has `rows`; the segment's first row's query sees `before` + 1
// keys where the call is causal.
template <int HD, bool HALF, int NQ>
T2W_DEV void load_rows(const AttnDev& p, Rows<HD, NQ>& q, int row0, int first, int rows, int hk, int before, int kv) {
  constexpr int kC = HD / 64, kM = HD / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, group = p.group;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    if (n >= NQ) {
#pragma unroll
      for (int i = 0; i < kM; ++i) q.qa[i][n] = q.qa[i][2 + n] = 0;
      continue;
    }
    const int row = first + g + 8 * n;
    uint4 v[kC][2];
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[c][i] = make_uint4(0, 0, 0, 0);
        if (row < rows) {
          const uint16_t* x = static_cast<const uint16_t*>(p.q) + (row0 + over_group(p, row)) * p.q_row_ld +
                              (hk * group + row - group * over_group(p, row)) * p.q_head_ld;
          v[c][i] = __ldg(reinterpret_cast<const uint4*>(x + 64 * c + 16 * t + 8 * i));
        }
        const uint4 u = v[c][i];
        m = __vmaxu2(__vmaxu2(m, u.x & 0x7fff7fffu), u.y & 0x7fff7fffu);
        m = __vmaxu2(__vmaxu2(m, u.z & 0x7fff7fffu), u.w & 0x7fff7fffu);
      }
    m = max(m & 0xffffu, m >> 16);
    m = max(m, __shfl_xor_sync(~0u, m, 1));
    m = max(m, __shfl_xor_sync(~0u, m, 2));
    const int sh = row_shift<HALF>(m);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const uint32_t u[8] = {v[c][0].x, v[c][0].y, v[c][0].z, v[c][0].w, v[c][1].x, v[c][1].y, v[c][1].z, v[c][1].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) q.qa[4 * c + j][2 * i + n] = row_half2<HALF>(u[2 * j + i], sh, p.scale < 0.f);
    }
    q.c[n] = scaled(fabsf(p.scale) * kLog2e, -sh);
    q.end[n] = p.causal ? before + over_group(p, row) + 1 : kv;
    q.M[n] = -INFINITY;
    q.l[n] = 0.f;
#pragma unroll
    for (int i = 0; i < kM; ++i) q.o[n][i][0] = q.o[n][i][1] = q.o[n][i][2] = q.o[n][i][3] = 0.f;
  }
}
// 32 keys from kb on: their scores, weights and products.  get_k, get_v: the lane's places in a stage (stage_places()).
template <int HD, int NQ, bool P16>
T2W_DEV void tile_step(Rows<HD, NQ>& q, const FewStage<HD>& st, uint32_t get_k, const uint32_t (&get_v)[2],
                       int kb, int kv, int all_see) {
  constexpr int kC = HD / 64, kM = HD / 16, kH = P16 ? 2 : 1;  // kH: pages of the tile
  const int t = threadIdx.x & 3;
  const uint8_t* const bytes = st.k;
  float d[4][4] = {};
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    uint4 kr[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kr[j] = *reinterpret_cast<const uint4*>(bytes + 8 * HD * j + (get_k ^ (64 * c)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t(&qa)[4] = q.qa[4 * c + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 u = e4m3x4_to_f16x4(i == 0 ? kr[j].x : i == 1 ? kr[j].y : i == 2 ? kr[j].z : kr[j].w);
        mma_f16(d[j], qa[0], qa[1], qa[2], qa[3], u.x, u.y);
      }
    }
  }
  float ks[kH], lv[kH], unit[kH];
  bool odd = false;
#pragma unroll
  for (int i = 0; i < kH; ++i) {
    const float vs = st.vs[i];
    ks[i] = st.ks[i];
    odd |= !(vs < INFINITY) || !(ks[i] < INFINITY);
    const int e = vs < INFINITY ? (int)(__float_as_uint(vs) >> 23) - 127 : 0;
    lv[i] = (float)e;
    unit[i] = exp2i(-e);
  }
  const bool part = kb + 32 > all_see;  // some row does not see all of the tile
  uint32_t pw[NQ][4];
  float fac[NQ];
  bool raised = false;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float s[4][2], ck[kH], add[kH];
#pragma unroll
    for (int i = 0; i < kH; ++i) {
      ck[i] = q.c[n] * ks[i];
      if (ck[i] == 0.f) ck[i] = 1.1754944e-38f;  // (-inf times 0)
      add[i] = lv[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[j][i] = d[j][2 * n + i];
    if (part) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (kb + 8 * j + 2 * t + i >= q.end[n]) s[j][i] = -INFINITY;
    }
    if (odd) {  // a scale that is not finite may only meet what the row sees
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (kb + 8 * j + 2 * t + i < q.end[n]) s[j][i] = fmaf(s[j][i], ck[P16 ? j >> 1 : 0], add[P16 ? j >> 1 : 0]);
#pragma unroll
      for (int i = 0; i < kH; ++i) {
        ck[i] = 1.f;
        add[i] = 0.f;
      }
    }
    float mx;
    if constexpr (P16) {
      mx = fmaxf(fmaf(fmaxf(fmax3(s[0][0], s[0][1], s[1][0]), s[1][1]), ck[0], add[0]),
                 fmaf(fmaxf(fmax3(s[2][0], s[2][1], s[3][0]), s[3][1]), ck[kH - 1], add[kH - 1]));
    } else {
      mx = fmaf(fmax3(fmax3(s[0][0], s[0][1], s[1][0]), fmax3(s[1][1], s[2][0], s[2][1]), fmaxf(s[3][0], s[3][1])), ck[0], add[0]);
    }
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
    const bool raise = mx > q.M[n] + kRaise;
    raised |= raise;
    const float m_new = raise ? mx - kBelow : q.M[n];
    fac[n] = raise ? exp2_approx(q.M[n] - m_new) : 1.f;  // 2^-inf = 0 the first time
    q.M[n] = m_new;
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    float2 sum[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float c = ck[P16 ? j >> 1 : 0], b = add[P16 ? j >> 1 : 0] - ref;
      const float2 a = __ffma2_rn(make_float2(s[j][0], s[j][1]), make_float2(c, c), make_float2(b, b));
      const float2 e = make_float2(exp2_approx(a.x), exp2_approx(a.y));
      sum[j >> 1] = j & 1 ? __fadd2_rn(sum[j >> 1], e) : e;
      pw[n][j] = pack_f16x2(e.x, e.y);
    }
    // the exponentials without their values' scale: 2^(x - M) = w 2^-lv
    if constexpr (P16) {
      q.l[n] = fmaf(q.l[n], fac[n], fmaf(sum[0].x + sum[0].y, unit[0], (sum[1].x + sum[1].y) * unit[kH - 1]));
    } else {
      const float2 u = __fadd2_rn(sum[0], sum[1]);
      q.l[n] = fmaf(q.l[n], fac[n], (u.x + u.y) * unit[0]);
    }
    if (odd) {  // values that are NaN, where the row sees them
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!(st.vs[P16 ? j >> 1 : 0] < INFINITY)) {
          if (kb + 8 * j + 2 * t < q.end[n]) pw[n][j] |= 0x7fffu;
          if (kb + 8 * j + 2 * t + 1 < q.end[n]) pw[n][j] |= 0x7fff0000u;
        }
    }
  }
  if (__any_sync(~0u, raised)) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {  // the factors lie with the rows, the output has them as columns 2t, 2t + 1
      const float f0 = __shfl_sync(~0u, fac[n], 8 * t), f1 = __shfl_sync(~0u, fac[n], 8 * t + 4);
#pragma unroll
      for (int i = 0; i < kM; ++i) {
        q.o[n][i][0] *= f0;
        q.o[n][i][1] *= f1;
        q.o[n][i][2] *= f0;
        q.o[n][i][3] *= f1;
      }
    }
  }
  const bool tail = kb + 32 > kv;  // places of the page past the last key may hold anything, NaN codes too
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t vw[4][HD / 32];  // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the half
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t* const v = bytes + (16 * i + 8 * (j >> 1)) * HD + get_v[j & 1];
      if constexpr (HD == 128) {
        const uint4 u = *reinterpret_cast<const uint4*>(v);
        vw[j][0] = u.x;
        vw[j][1] = u.y;
        vw[j][HD / 32 - 2] = u.z;
        vw[j][HD / 32 - 1] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(v);
        vw[j][0] = u.x;
        vw[j][1] = u.y;
      }
    }
    if (tail) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (kb + 16 * i + 2 * t + (j & 1) + 8 * (j >> 1) >= kv)
#pragma unroll
          for (int x = 0; x < HD / 32; ++x) vw[j][x] = 0;
    }
#pragma unroll
    for (int x = 0; x < HD / 32; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint2 lo = e4m3x4_to_f16x4(__byte_perm(vw[0][x], vw[1][x], y ? 0x7362 : 0x5140));
        const uint2 hi = e4m3x4_to_f16x4(__byte_perm(vw[2][x], vw[3][x], y ? 0x7362 : 0x5140));
#pragma unroll
        for (int n = 0; n < NQ; ++n) mma_f16(q.o[n][2 * x + y], lo.x, lo.y, hi.x, hi.y, pw[n][2 * i], pw[n][2 * i + 1]);
      }
  }
}
// This thread's columns of queries 2t and 2t + 1, HD / 8 in a row: finished rows (part nullptr) or a part's.
template <int HD, bool HALF, int NQ>
T2W_DEV void store_rows(const AttnDev& p, const Rows<HD, NQ>& q, int row0, int from, int rows, int hk, float* part, int part_rows) {
  constexpr int kM = HD / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, group = p.group;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float sum = q.l[n];
    sum += __shfl_xor_sync(~0u, sum, 1);
    sum += __shfl_xor_sync(~0u, sum, 2);
    const float top = sum != sum ? fmaxf(q.M[n], -1e30f) : q.M[n];  // a NaN counts, even where M saw nothing else
    if (part && t == 0 && from + 8 * n + g < rows) {
      part[part_rows * HD + from + 8 * n + g] = top;
      part[part_rows * HD + part_rows + from + 8 * n + g] = sum;
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row = from + 8 * n + 2 * t + y;
      const float ls = __shfl_sync(~0u, sum, 8 * t + 4 * y), Ms = __shfl_sync(~0u, top, 8 * t + 4 * y);
      if (row < rows && part) {
#pragma unroll
        for (int i = 0; i < kM; i += 2)
          *reinterpret_cast<float4*>(part + row * HD + g * (HD / 8) + 2 * i) =
              make_float4(q.o[n][i][y], q.o[n][i][2 + y], q.o[n][i + 1][y], q.o[n][i + 1][2 + y]);
      } else if (row < rows) {
        const float inv = ls != 0.f ? 1.f / ls : 0.f;
        const int tok = over_group(p, row);
        const size_t at = (size_t)(row0 + tok) * p.q_heads + hk * group + row - group * tok;
        uint4* const out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at * HD + g * (HD / 8));
#pragma unroll
        for (int i = 0; i < kM; i += 4) {
          uint32_t u[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float a = q.o[n][i + x][y] * inv, b = q.o[n][i + x][2 + y] * inv;
            u[x] = HALF ? pack_f16x2(a, b) : pack_bf16x2(a, b);
          }
          out[i / 4] = make_uint4(u[0], u[1], u[2], u[3]);
        }
        if (g == 0 && p.lse) p.lse[at] = ls != 0.f ? (Ms + log2f(ls)) * 0.6931471805599453f : -INFINITY;
      }
      __syncwarp();
    }
  }
}

template <int HD, bool HALF, int NQ, bool P16>
__global__ void __launch_bounds__(32 * few_warps, few_blocks(HD, NQ)) k_paged_few(const AttnDev p) {
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr int kS = few_stages;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w = few_warps * blockIdx.x + warp, group = p.group;
  const FewStage<HD>* const stage = reinterpret_cast<const FewStage<HD>*>(ring) + warp * kS;
  const uint32_t ring0 = smem_u32(stage);
  const uint64_t policy = l2_policy_evict_first();
  uint32_t put[2], get_k, get_v[2];
  stage_places<HD>(put, get_k, get_v);
  pdl_wait();
  pdl_launch();
  const int4 head4 = *reinterpret_cast<const int4*>(p.head);  // n_runs, tiles, per, workers
  int4 seg = p.starts[2 * w], of = p.starts[2 * w + 1];  // request, key head, query tile (always 0), key tile; rows, lengths
  const int extra = p.head->extra;
  const int4 seg0 = p.starts[2 * few_warps * blockIdx.x], of0 = p.starts[2 * few_warps * blockIdx.x + 1];  // the block's first worker's
  if (w >= head4.w) return;
  // one segment over all of the block's places (its key count is that of the few rows' only query tile)
  const bool filled = seg0.w >= 0 && few_warps * blockIdx.x + few_warps - 1 < head4.w &&
                      seg_tiles(of0.z, 32) - seg0.w >= few_warps * head4.z;
  const int stop = min((w + 1) * head4.z, head4.y);
  int zero = w * head4.z - seg.w;  // the place of the segment's tile 0

  // ---- the copies, which run ahead: tiles lkt .. lkt1 - 1 of the segment with tile 0 at lzero, then the next segments'
  int lr = seg.x, lhk = seg.y, lkt = max(seg.w, 0), lkt1 = 0, lnt = 0, lkv = 0, lzero = zero, base = -64;
  int pgA = 0, pgB = 0;  // lane i: the pages of tile base + i
  bool live = true;
  auto open = [&](int kv) {
    lkv = kv;
    lnt = seg_tiles(lkv, 32);
    lkt1 = min(lnt, stop - lzero);
    base = -64;
    live = lkt < lkt1;
  };
  auto send = [&](int at) {
    if (live) {
      if (lkt - base >= 32) {
        base = lkt;
        const int mine = lkt + lane;
        if (mine < lkt1) {
          const int b = (mine * 32) >> p.shift;
          const int* const table = p.table + (size_t)lr * p.table_ld;
          pgA = mine * 32 < lkv ? table[b] : 0;
          pgB = P16 && mine * 32 + 16 < lkv ? table[b + 1] : pgA;
          if ((unsigned)pgA >= (unsigned)p.pages || (unsigned)pgB >= (unsigned)p.pages) {
            atomicExch(p.status, T2W_ERR_INVALID);
            pgA = pgB = 0;
          }
        }
      }
      const uint32_t to = ring0 + at * (uint32_t)sizeof(FewStage<HD>);
      const long long a = __shfl_sync(~0u, pgA, lkt - base), b = P16 ? (long long)__shfl_sync(~0u, pgB, lkt - base) : a;
      const long long in = ((long long)lhk * p.page + (P16 ? 0 : (lkt * 32) & (p.page - 1))) * HD + 16 * lane;
#pragma unroll
      for (int x = 0; x < 2; ++x) {  // a half tile's rows lie one after the other: the warp copies 512 bytes at a time
        const uint8_t* const lo = p.codes[x] + a * p.page_ld[x] + in;
        const uint8_t* const hi = P16 ? p.codes[x] + b * p.page_ld[x] + in : lo + 16 * HD;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
          copy16(to + x * 32 * HD + i * 512 + put[i & 1], i < HD / 32 ? lo + i * 512 : hi + (i - HD / 32) * 512, policy);
      }
      if (lane < 4)
        copy4(to + 64 * HD + 4 * lane,  // ks, vs
              p.scales[lane >> 1] + (lane & 1 ? b : a) * p.scale_ld[lane >> 1] + lhk);
      if (++lkt == lkt1) {
        lzero += lnt + extra;
        if (lkt1 < lnt || lzero >= stop) {
          live = false;
        } else {
          lkt = 0;
          if (++lhk == p.kv_heads) {
            lhk = 0;
            do lr++;
            while (p.q_start[lr + 1] == p.q_start[lr]);  // (tiles are left, so there is a request with rows)
            open(p.kv_len[lr]);
          } else {  // the same pages
            lkt1 = min(lnt, stop - lzero);
            if (base != 0) base = -64;
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  open(of.z);
#pragma unroll
  for (int i = 0; i < kS - 1; ++i) send(i);

  // ---- the segments
  int at = 0;  // the stage of the next tile
  bool first = true;
  while (zero < stop) {
    const int hk = seg.y, row0 = of.x, f = of.y, kv = of.z;
    const int rows = f * group, nt = seg_tiles(kv, 32);
    const int kt0 = max(seg.w, 0), kt1 = min(nt, stop - zero);
    if (kt1 <= kt0) break;
    Rows<HD, NQ> q;
    load_rows<HD, HALF, NQ>(p, q, row0, 0, rows, hk, kv - f, kv);
    const int all_see = p.causal ? kv - f + 1 : kv;  // keys that every row sees
    for (int kt = kt0; kt < kt1; ++kt) {
      __syncwarp();  // every lane is done with the stage that is filled again
      send(at ? at - 1 : kS - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kS - 1) : "memory");
      __syncwarp();
      const FewStage<HD>& st = stage[at];
      at = at + 1 == kS ? 0 : at + 1;
      tile_step<HD, NQ, P16>(q, st, get_k, get_v, kt * 32, kv, all_see);
    }
    const bool whole = kt0 == 0 && kt1 == nt;
    float* const part = whole    ? nullptr
                        : filled ? reinterpret_cast<float*>(ring + warp * kS * sizeof(FewStage<HD>))
                                 : part_of(p.ws, 2 * w + (first ? 0 : 1), 16, HD);
    if (filled) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();  // the warp's ring is read to the end
    }
    store_rows<HD, HALF, NQ>(p, q, row0, 0, rows, hk, part, 16);
    if (filled) {  // all the block's warps come here, each with its one segment
      __syncthreads();
      float* const out = part_of(p.ws, 2 * few_warps * blockIdx.x, 16, HD);
      const float* const in = reinterpret_cast<const float*>(ring);
      constexpr int kLd = kS * (int)sizeof(FewStage<HD>) / 4;
      for (int i = threadIdx.x; i < rows * (HD / 4); i += 32 * few_warps) {
        const int row = i / (HD / 4), d = i % (HD / 4) * 4;
        float m[few_warps], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int x = 0; x < few_warps; ++x) {
          m[x] = in[x * kLd + 16 * HD + row];
          top = fmaxf(top, m[x]);
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (top > -INFINITY) {
#pragma unroll
          for (int x = 0; x < few_warps; ++x) {
            const float e = exp2_approx(m[x] - top);
            const float4 v = *reinterpret_cast<const float4*>(in + x * kLd + row * HD + d);
            acc.x = fmaf(e, v.x, acc.x);
            acc.y = fmaf(e, v.y, acc.y);
            acc.z = fmaf(e, v.z, acc.z);
            acc.w = fmaf(e, v.w, acc.w);
            sum = fmaf(e, in[x * kLd + 16 * HD + 16 + row], sum);
          }
        }
        *reinterpret_cast<float4*>(out + row * HD + d) = acc;
        if (d == 0) {
          out[16 * HD + row] = top;
          out[16 * HD + 16 + row] = sum;
        }
      }
      return;
    }
    first = false;
    zero += nt + extra;
    seg.w = 0;
    if (++seg.y == p.kv_heads && zero < stop) {
      seg.y = 0;
      do {
        seg.x++;
        of.x = p.q_start[seg.x];
        of.y = p.q_start[seg.x + 1] - of.x;
      } while (of.y == 0);
      of.z = p.kv_len[seg.x];
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------- 17 to 64 query rows to a key head
//
// A segment is a few tiles long, so what counts is that a block begins and ends one cheaply and that other blocks run
// meanwhile.  A worker is a block of 4 warps with 16 rows each; it takes 64 keys at a time, of which each warp copies a
// quarter (32 keys' K or V) into the block's ring and all four read all.  Tiles of 128 rows on tcgen05 (paged_attn_tc.cu)
// have the faster products, but half of their rows or more would be empty.
//
// What bounds it: instructions.  Every warp widens all the codes for its 16 rows, so 1 in 4 instructions is a product; an
// SM's quarters issue one in 48% of the clocks with 4 warps each, whose tiles are chains from the copies through widening,
// products and exponentials to products.  Measured: 128 windows of 50 tokens over 400 keys, 8 heads of 64: 65.7 MB and 5.2
// GFLOP in 54 us, 1.2 TB/s.  Dropped: 32 rows a warp (half the widening, but the output's registers leave 2 blocks an SM):
// 85 to 99 us.
template <bool HALF, bool P16>
__global__ void __launch_bounds__(32 * mid_warps, mid_blocks) k_paged_mid(const AttnDev p) {
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr int HD = 64, kS = mid_stages;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w = blockIdx.x, group = p.group;
  const FewStage<HD>* const stage = reinterpret_cast<const FewStage<HD>*>(ring);
  const uint64_t policy = l2_policy_evict_first();
  uint32_t put[2], get_k, get_v[2];
  stage_places<HD>(put, get_k, get_v);
  pdl_wait();
  pdl_launch();
  Walk at;
  if (!at.begin(p, w)) return;

  // ---- copies: a tile's quarters are K and V codes of its keys 0-31 and 32-63, a quarter a warp
  static_assert(mid_warps == 4, "a quarter a warp");
  const int half = warp >> 1, x = warp & 1;
  Walk ahead = at;
  int kt_a = at.kt0, pgA = 0, pgB = 0;
  bool live = true;
  auto look_up = [&]() {
    if (!live) return;
    const int key = kt_a * 64 + 32 * half;
    const int* const table = p.table + (size_t)ahead.r * p.table_ld + (key >> p.shift);
    pgA = key < ahead.kv ? __ldg(table) : 0;
    pgB = P16 && key + 16 < ahead.kv ? __ldg(table + 1) : pgA;
  };
  auto send = [&](int to_stage) {
    if (live) {
      if (kt_a * 64 + 32 * half < ahead.kv) {  // there are keys in this half
        if ((unsigned)pgA >= (unsigned)p.pages || (unsigned)pgB >= (unsigned)p.pages) {
          atomicExch(p.status, T2W_ERR_INVALID);
          pgA = pgB = 0;
        }
        const uint32_t to = smem_u32(ring) + (2 * to_stage + half) * (uint32_t)sizeof(FewStage<HD>);
        const long long in = ((long long)ahead.hk * p.page + (P16 ? 0 : (kt_a * 64 + 32 * half) & (p.page - 1))) * HD + 16 * lane;
        const uint8_t* const lo = p.codes[x] + pgA * p.page_ld[x] + in;
        const uint8_t* const hi = P16 ? p.codes[x] + pgB * p.page_ld[x] + in : lo + 16 * HD;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
          copy16(to + x * 32 * HD + i * 512 + put[i & 1], i < HD / 32 ? lo + i * 512 : hi + (i - HD / 32) * 512, policy);
        if (lane < 2)  // ks or vs
          copy4(to + 64 * HD + 8 * x + 4 * lane, p.scales[x] + (lane ? pgB : pgA) * p.scale_ld[x] + ahead.hk);
      }
      if (++kt_a == ahead.kt1) {
        live = ahead.next(p);
        kt_a = 0;
      }
      look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look_up();
#pragma unroll
  for (int i = 0; i < kS - 1; ++i) send(i);

  // ---- segments
  int st = 0;  // the stage of the next tile
  do {
    const int rows = at.rows(p, group), from = 16 * warp, row0 = at.row0 + at.qt * p.tq, before = at.kv - at.f + at.qt * p.tq;
    const bool mine = from < rows;
    // keys that all of the warp's rows see, and that one of them sees
    const int all_see = p.causal ? before + over_group(p, from) + 1 : at.kv;
    const int some_see = p.causal ? before + over_group(p, min(from + 16, rows) - 1) + 1 : at.kv;
    Rows<HD, 2> q;
    load_rows<HD, HALF, 2>(p, q, row0, from, rows, at.hk, before, at.kv);
    for (int kt = at.kt0; kt < at.kt1; ++kt) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kS - 2) : "memory");
      __syncthreads();  // every warp's copies of this tile are there, and nobody reads the stage before it any more
      send(st ? st - 1 : kS - 1);
      if (mine)
#pragma unroll 1
        for (int i = 0; i < 2; ++i)
          if (kt * 64 + 32 * i < some_see)
            tile_step<HD, 2, P16>(q, stage[2 * st + i], get_k, get_v, kt * 64 + 32 * i, at.kv, all_see);
      st = st + 1 == kS ? 0 : st + 1;
    }
    float* const part = at.kt0 == 0 && at.kt1 == at.nt ? nullptr : part_of(p.ws, 2 * w + (at.first ? 0 : 1), 16 * mid_warps, HD);
    if (mine) store_rows<HD, HALF, 2>(p, q, row0, from, rows, at.hk, part, 16 * mid_warps);
  } while (at.next(p));
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------- segments that were cut
// Where worker w's start is the first cut of a segment, that segment's parts are joined: up to 4 parts by the start's
// warp, a thread four columns of a row, more of them by the 8 warps of the block, a row at a time and every eighth part a
// warp.  The order is fixed, so the bits are too.  What it costs is a chain of loads after the kernel in front of it has
// ended: so all that the plan tells is read before that, the parts' rows are sent for together with their exponents, and
// the blocks are resident at once.  It ends 6 us after that kernel for single tokens (3 requests of 150k keys: 38 parts
// each; row by row in one warp it was 11), 5 for windows, 12 for chunks (39 MB of parts, from L2).  A share of the rows for
// each 8 of a part: with twice or half as many the windows take 56.5 or 55.4 us for 54.0, the chunks 160 at a quarter and
// 142 at half for 132.
struct Parts {
  const float* ws;
  int rows_ld, hd;
  int w0, second;     // the first part's worker, and whether it is that worker's second
  int lead, mid, b0;  // parts of single workers, of blocks (from block b0, block_workers each), and of single workers again
  int block_workers, tail0, n;
  T2W_DEV const float* at(int i) const {
    const int slot = i == 0 && lead ? 2 * w0 + second
                     : i < lead     ? 2 * (w0 + i)
                     : i < lead + mid ? 2 * block_workers * (b0 + i - lead)
                                      : 2 * (tail0 + i - lead - mid);
    return ws + (size_t)slot * rows_ld * (hd + 2);
  }
};
template <int HD>
struct Joined {
  static constexpr int N = HD / 32;
  float acc[N], sum, top;
};
template <int N>
T2W_DEV void load_cols(float (&u)[N], const float* v) {
  if constexpr (N == 4) *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(v);
  else *reinterpret_cast<float2*>(u) = *reinterpret_cast<const float2*>(v);
}
// A row's parts first, first + 8, ...: a lane holds one part's exponent and sum of 32, and N columns of all of them.
template <int HD>
T2W_DEV void join_parts(Joined<HD>& j, const Parts& parts, int first, int row, int lane) {
  constexpr int N = HD / 32, K = 8;
  const int count = (parts.n - first + 7) / 8;
  j.top = -INFINITY;
  j.sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) j.acc[i] = 0.f;
  for (int x0 = 0; x0 < count; x0 += 32) {
    const int n = min(32, count - x0);
    float top = -INFINITY, sum = 0.f;
    if (lane < n) {
      const float* q = parts.at(first + 8 * (x0 + lane)) + parts.rows_ld * HD + row;
      top = __ldcg(q);
      sum = __ldcg(q + parts.rows_ld);
    }
    float m = 0.f, e = 0.f;
    for (int i0 = 0; i0 < n; i0 += K) {
      float u[K][N];
#pragma unroll
      for (int i = 0; i < K; ++i) {
#pragma unroll
        for (int y = 0; y < N; ++y) u[i][y] = 0.f;
        if (i0 + i < n) load_cols<N>(u[i], parts.at(first + 8 * (x0 + i0 + i)) + row * HD + lane * N);
      }
      if (i0 == 0) {
        m = fmaxf(j.top, top);
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
        const float ref = m == -INFINITY ? 0.f : m, old = exp2_approx(j.top - ref);
        e = exp2_approx(top - ref);
        j.top = m;
        j.sum = fmaf(j.sum, old, warp_sum(lane < n ? e * sum : 0.f));
#pragma unroll
        for (int i = 0; i < N; ++i) j.acc[i] *= old;
      }
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const float ei = __shfl_sync(~0u, e, i0 + i);
#pragma unroll
        for (int y = 0; y < N; ++y) j.acc[y] = fmaf(ei, u[i][y], j.acc[y]);
      }
    }
  }
}
struct Long {  // a segment of more than 4 parts
  Parts parts;
  int r0, rn, head0;
};
template <int HD, bool HALF>
__global__ void __launch_bounds__(256, 4) k_paged_merge(const AttnDev p) {
  __shared__ Long longs[8];
  __shared__ __align__(16) float joined[2][8][HD + 4];  // by warp: columns, exponent, sum

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = p.group;
  // The plan was complete before the kernel in front of this one began (it waited for it), so it is read ahead of the
  // wait, past this SM's L1.
  const int4 h0 = __ldcg(reinterpret_cast<const int4*>(p.head)), h1 = __ldcg(reinterpret_cast<const int4*>(p.head) + 1);
  const int per = h0.z, workers = h0.w, used = h1.y, extra = h1.w;
  // a warp has a start, and of its rows the share blockIdx.y of gridDim.y
  const int w = blockIdx.x * 8 + warp, share = blockIdx.y, shares = gridDim.y;
  bool mine = false;
  int r0 = 0, rn = 0, head0 = 0;
  Parts parts;
  parts.n = 0;
  if (w > 0 && w < workers) {
    const int4 seg = __ldcg(p.starts + 2 * w), of = __ldcg(p.starts + 2 * w + 1);  // of: first row, rows, keys
    const int at = of.w - seg.w, before = __ldcg(p.starts + 2 * w - 1).w;  // the place of the segment's tile 0; where w - 1 begins
    mine = seg.w > 0 && at >= before;
    const int end = at + seg_tiles(tile_keys(of.y, of.z, p.causal, p.tq, seg.z), p.kt);
    r0 = of.x + seg.z * p.tq;
    rn = min(p.tq, of.y - seg.z * p.tq) * group;
    head0 = seg.y * group;
    parts.ws = p.ws;
    parts.rows_ld = p.part_rows;
    parts.hd = HD;
    parts.w0 = w - 1;
    parts.second = at - extra > before;
    const int last = (end - 1) / per, bw = p.block_workers;
    const int b0 = (at + bw * per - 1) / (bw * per), b1 = end / (bw * per);  // blocks that the segment fills
    parts.block_workers = bw;
    parts.b0 = b0;
    parts.mid = bw > 1 && b1 > b0 ? b1 - b0 : 0;
    parts.lead = parts.mid ? b0 * bw - parts.w0 : last - parts.w0 + 1;
    parts.tail0 = b1 * bw;
    parts.n = parts.mid ? parts.lead + parts.mid + last - b1 * bw + 1 : parts.lead;
  }
  pdl_wait();
  pdl_launch();
  // Padding, and all rows where a page was met that the cache does not have (or the plan was void before): nobody's rows
  // are answered from other pages than their own.  (One answer for the block, whatever another stream's call with the same
  // plan writes meanwhile.  The look at it costs 0.2 to 0.8 us, and the same where the stores wait for it instead.)
  const bool is_void = __syncthreads_or(__ldcg(p.status) != T2W_OK);
  for (int row = (is_void ? 0 : used) + blockIdx.y * gridDim.x + blockIdx.x; row < p.rows; row += gridDim.x * gridDim.y)
    for (int i = threadIdx.x; i < p.q_heads * (HD / 4); i += blockDim.x)
      store_row<HALF>(p, row, i / (HD / 4), HD, i % (HD / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f);
  if (is_void) return;
  if (lane == 0) {
    longs[warp].parts = parts;
    longs[warp].r0 = r0;
    longs[warp].rn = mine && parts.n > 4 ? rn : 0;
    longs[warp].head0 = head0;
  }
  if (mine && parts.n <= 4) {  // a thread four columns of a row
    const float* part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) part[i] = parts.at(i);
#pragma unroll 2
    for (int i = share * 32 + lane; i < rn * (HD / 4); i += 32 * shares) {
      const int row = i / (HD / 4), d = i % (HD / 4) * 4;
      float m[4], l[4], top = -INFINITY;
      float4 v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
        m[x] = -INFINITY;
        l[x] = 0.f;
        if (x < parts.n) {
          v[x] = __ldcg(reinterpret_cast<const float4*>(part[x] + row * HD + d));
          m[x] = __ldcg(part[x] + p.part_rows * HD + row);
          l[x] = __ldcg(part[x] + p.part_rows * HD + p.part_rows + row);
        }
        top = fmaxf(top, m[x]);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
      if (top > -INFINITY) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float e = exp2_approx(m[x] - top);
          acc.x = fmaf(e, v[x].x, acc.x);
          acc.y = fmaf(e, v[x].y, acc.y);
          acc.z = fmaf(e, v[x].z, acc.z);
          acc.w = fmaf(e, v[x].w, acc.w);
          sum = fmaf(e, l[x], sum);
        }
      }
      store_row<HALF>(p, r0 + over_group(p, row), head0 + row - group * over_group(p, row), HD, d, acc, top, sum);
    }
  }
  __syncthreads();
  int turn = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const Long& g = longs[i];
#pragma unroll 1
    for (int row = share; row < g.rn; row += shares, turn ^= 1) {
      Joined<HD> j;
      join_parts<HD>(j, g.parts, warp, row, lane);
      float* const mine8 = joined[turn][warp];
#pragma unroll
      for (int y = 0; y < HD / 32; ++y) mine8[lane * (HD / 32) + y] = j.acc[y];
      if (lane == 0) {
        mine8[HD] = j.top;
        mine8[HD + 1] = j.sum;
      }
      __syncthreads();  // (the other turn's buffer is read until the next one)
      if (threadIdx.x < HD / 4) {
        const int d = threadIdx.x * 4;
        float top = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < 8; ++x) top = fmaxf(top, joined[turn][x][HD]);
        if (top > -INFINITY) {
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float e = exp2_approx(joined[turn][x][HD] - top);
            const float4 v = *reinterpret_cast<const float4*>(&joined[turn][x][d]);
            acc.x = fmaf(e, v.x, acc.x);
            acc.y = fmaf(e, v.y, acc.y);
            acc.z = fmaf(e, v.z, acc.z);
            acc.w = fmaf(e, v.w, acc.w);
            sum = fmaf(e, joined[turn][x][HD + 1], sum);
          }
        }
        store_row<HALF>(p, g.r0 + over_group(p, row), g.head0 + row - group * over_group(p, row), HD, d, acc, top, sum);
      }
    }
  }
}

}  // namespace
}  // namespace t2w

using namespace t2w;

namespace {

template <int HD, bool HALF>
cudaError_t launch_paged(const AttnDev& p, const PagedCut& cut, int max_rows, cudaStream_t st) {
  auto merge = [&](int shares) {
    return launch_k(k_paged_merge<HD, HALF>, dim3((cut.workers + 7) / 8, shares), dim3(256), 0, st, p);
  };
  if constexpr (HD == 64)
    if (cut.form == PagedForm::kMid) {
      constexpr int smem = 2 * mid_stages * (int)sizeof(FewStage<HD>);
      static std::atomic<uint64_t> done[2];
      auto mid = [&](auto* k, std::atomic<uint64_t>& d) {
        const cudaError_t r = smem_attr_once(k, smem, d);
        return r != cudaSuccess ? r : launch_k(k, dim3(cut.workers), dim3(32 * mid_warps), smem, st, p);
      };
      const cudaError_t e = p.page == 16 ? mid(k_paged_mid<HALF, true>, done[0]) : mid(k_paged_mid<HALF, false>, done[1]);
      return e != cudaSuccess ? e : merge(cut.part_rows / 8);
    }
  if (cut.form == PagedForm::kMany) {
    const cudaError_t e = launch_paged_many(p, cut, HD, HALF, st);
    return e != cudaSuccess ? e : merge(cut.part_rows / 8);
  }
  const int nq = max_rows > 8 ? 2 : 1;
  constexpr int smem = few_warps * few_stages * (int)sizeof(FewStage<HD>);
  static std::atomic<uint64_t> done[4];
  auto few = [&](auto* k, std::atomic<uint64_t>& d) {
    const cudaError_t r = smem_attr_once(k, smem, d);
    return r != cudaSuccess ? r : launch_k(k, dim3(cut.workers / few_warps), dim3(32 * few_warps), smem, st, p);
  };
  cudaError_t e;
  if (p.page == 16) e = nq == 1 ? few(k_paged_few<HD, HALF, 1, true>, done[0]) : few(k_paged_few<HD, HALF, 2, true>, done[1]);
  else e = nq == 1 ? few(k_paged_few<HD, HALF, 1, false>, done[2]) : few(k_paged_few<HD, HALF, 2, false>, done[3]);
  if (e != cudaSuccess) return e;
  return merge(max_rows < 8 ? max_rows : 8);
}

}  // namespace

extern "C" size_t t2w_paged_workspace_bytes(int32_t max_fresh, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  if (max_fresh <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
  const PagedCut c = paged_cut(max_fresh, q_heads, kv_heads, head_dim);
  return 2 * (size_t)c.workers * c.part_rows * (head_dim + 2) * sizeof(float);
}

extern "C" int t2w_paged_attn(const t2w_paged_attn_args* a, void* stream) {
  if (!a || !a->plan || !a->q || !a->k_codes || !a->v_codes || !a->k_scale || !a->v_scale || !a->table || !a->out)
    return T2W_ERR_INVALID;
  if (a->dtype != T2W_DT_BF16 && a->dtype != T2W_DT_FP16) return T2W_ERR_UNSUPPORTED;
  const int64_t ints = t2w_paged_plan_ints(a->requests, a->rows, a->max_fresh, a->page, a->q_heads, a->kv_heads,
                                           a->head_dim, nullptr);
  if (ints < 0) return (int)ints;
  if (a->pages <= 0 || a->table_ld <= 0 || !(a->scale == a->scale)) return T2W_ERR_INVALID;
  AttnDev p;
  p.q = a->q;
  p.q_row_ld = a->q_row_ld;
  p.q_head_ld = a->q_head_ld;
  p.codes[0] = static_cast<const uint8_t*>(a->k_codes);
  p.codes[1] = static_cast<const uint8_t*>(a->v_codes);
  p.scales[0] = a->k_scale;
  p.scales[1] = a->v_scale;
  p.page_ld[0] = a->k_page_ld;
  p.page_ld[1] = a->v_page_ld;
  p.scale_ld[0] = a->k_scale_ld;
  p.scale_ld[1] = a->v_scale_ld;
  for (int w = 0; w < 2; ++w)
    if ((reinterpret_cast<uintptr_t>(p.codes[w]) & 15) || p.page_ld[w] % 16 ||
        p.page_ld[w] < (int64_t)a->kv_heads * a->page * a->head_dim || p.scale_ld[w] < a->kv_heads)
      return T2W_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(a->q) & 15) || a->q_row_ld % 8 || a->q_head_ld % 8 ||
      (reinterpret_cast<uintptr_t>(a->out) & 15))
    return T2W_ERR_INVALID;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15)) return T2W_ERR_INVALID;
  if (a->workspace_bytes < t2w_paged_workspace_bytes(a->max_fresh, a->q_heads, a->kv_heads, a->head_dim))
    return T2W_ERR_WORKSPACE;
  const PagedCut cut = paged_cut(a->max_fresh, a->q_heads, a->kv_heads, a->head_dim);
  const PlanLayout l = paged_layout(a->requests, a->rows, a->page, cut);
  p.table = a->table;
  p.table_ld = a->table_ld;
  p.page = a->page;
  p.shift = a->page == 16 ? 4 : a->page == 32 ? 5 : a->page == 64 ? 6 : 7;
  p.pages = a->pages;
  p.rows = a->rows;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.causal = a->causal != 0;
  p.group = a->q_heads / a->kv_heads;
  p.group_mul = (65536 + p.group - 1) / p.group;
  p.scale = a->scale;
  p.head = reinterpret_cast<const PlanHead*>(a->plan);
  p.q_start = a->plan + l.q_start;
  p.kv_len = a->plan + l.kv_len;
  p.starts = reinterpret_cast<const int4*>(a->plan + l.starts);
  p.tq = cut.tq;
  p.kt = cut.kt;
  p.part_rows = cut.part_rows;
  p.block_workers = cut.form == PagedForm::kFew ? few_warps : 1;
  p.ws = static_cast<float*>(a->workspace);
  p.out = a->out;
  p.lse = a->lse;
  p.status = const_cast<int*>(&p.head->status);
  if (a->rows == 0) return T2W_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = a->dtype == T2W_DT_FP16;
  const int max_rows = a->max_fresh * (a->q_heads / a->kv_heads);
  cudaError_t e;
  if (a->head_dim == 64) e = half ? launch_paged<64, true>(p, cut, max_rows, st) : launch_paged<64, false>(p, cut, max_rows, st);
  else e = half ? launch_paged<128, true>(p, cut, max_rows, st) : launch_paged<128, false>(p, cut, max_rows, st);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return T2W_ERR_CUDA;
  }
  return T2W_OK;
}
