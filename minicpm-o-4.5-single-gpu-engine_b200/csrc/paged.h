// What the kernels of the paged 8-bit K/V cache share: the layout of a plan's buffer, the split of an attention call's
// key tiles over its workers, and the cache's number format.
//
// A value is code * scale: code e4m3, scale 2^e with e in [kScaleMin, kScaleMax], one scale per page and head (K and V
// each have their own).  A power of two because a page that is appended to may have to raise its scale: codes already
// written are then divided by a power of two, which is exact but for codes that become subnormal, and a floating-point
// code loses nothing by it against a scale of full precision.  A page and head that was given a value that is not finite
// has the scale NaN from then on: all of it reads as NaN, and rows that its mask hides from a query still cannot reach it.
#pragma once

#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace t2w {

constexpr int kScaleMin = -64, kScaleMax = 64;

// ---------------------------------------------------------------- a plan's buffer (int32)
// header, then q_start [B + 1], kv_len [B], slot [rows], request [rows], bases [B + 1] x 4 (new pages, runs, places,
// segments), starts 2 x int4 [workers], runs int4 [max_runs].  Every part begins on a 16-byte boundary.
struct PlanHead {
  int n_runs;   // runs of rows that go into one page
  int tiles;    // places of the attention's key tiles (see PagedCut)
  int per;      // places of a worker
  int workers;  // workers that have any
  int status;   // T2W_OK, or what made the plan void
  int used;     // rows that belong to a request (the rest is padding)
  int free_left;
  int extra;    // places before each segment's first tile
};
struct PlanLayout {
  int64_t q_start, kv_len, slot, request, new_base, run_base, tile_base, seg_base, starts, runs, total;  // in int32
  int max_runs, max_workers;
};

// How an attention call is cut.  A segment is what one softmax runs over: (request, key head, query tile); its keys come
// in tiles of `kt`.  The tiles of all segments, in that order, are numbered, and the places are dealt to the workers in
// equal contiguous shares, so that ragged lengths cost no balance; a segment that is cut by a share's end is finished by
// k_paged_merge.  Where the worker is a block and a segment is a good deal shorter than a share, the shares end at the
// nearest segment's end instead (whole segments).  In large calls each segment's first tile has `extra` empty places
// before it: what it costs a worker to begin a segment, in tiles, so that a share of many short segments is not the one
// that the others wait for.
enum class PagedForm {
  kFew,   // at most 16 query rows to a key head: a worker is a warp
  kMid,   // at most 64, head_dim 64: a worker is a block, with tiles of 64 rows
  kMany,  // a worker is a block, with tcgen05 tiles of 128 rows
};
struct PagedCut {
  PagedForm form;
  int part_rows;  // rows of a segment's part in the workspace
  int tq;     // query tokens of a tile (rows = tokens * group)
  int kt;     // keys of a tile
  int workers;  // workers at most
  int min_per;  // places of a worker at least
  int extra;
  bool whole;   // whether short segments are left whole
};

// Blocks of 8 warps that an SM holds of the kernel for few query rows.
constexpr int few_warps = 8;
constexpr int few_blocks(int hd, int nq) { return hd == 128 || nq == 2 ? 1 : 2; }
// The same of the form for middling numbers of rows (head_dim 64 alone), its warps, and the stages of a block's ring.
constexpr int mid_blocks = 4, mid_warps = 4, mid_stages = 3;
constexpr int few_stages = 3;  // tiles of a warp's ring (8 KB each, 4 KB where head_dim is 64): the SM's rings hold 196 KB

inline int64_t round4(int64_t n) { return (n + 3) & ~int64_t(3); }

PagedCut paged_cut(int max_fresh, int q_heads, int kv_heads, int head_dim);
PlanLayout paged_layout(int64_t requests, int64_t rows, int page, const PagedCut& cut);

// ---------------------------------------------------------------- tiles of a request (device)
// sum over i < n of floor((a i + b) / m), m a power of two (a key tile), a >= 1, b >= 0, a n + b < 2^32: the sum of the
// a i + b less that of their remainders, over m.  With g the largest power of two that divides a and m, the remainders come
// again after m / g terms, and until then each of b mod g, b mod g + g, .. below m comes once; only what is left of n after
// whole periods is gone through.  (a is the tokens of a query tile: where the heads to a key head are a power of two a period
// is 4 terms at most, else 64.)
T2W_DEV long long sum_of_quotients(unsigned n, unsigned m, unsigned a, unsigned b) {
  const int lm = __ffs(m) - 1, lg = min(__ffs(a) - 1, lm), lp = lm - lg;  // m = 2^lm, g = 2^lg, m / g = 2^lp
  const unsigned g = 1u << lg, period = 1u << lp, left = n & (period - 1);
  const unsigned one = (b & (g - 1)) * period + g * (period * (period - 1) / 2);  // the remainders of a period
  long long sum = (long long)a * ((unsigned long long)n * (n - 1) / 2) + (long long)b * n - (long long)(n >> lp) * one;
  for (unsigned i = n - left; i < n; ++i) sum -= (a * i + b) & (m - 1);
  return sum >> lm;
}
// Keys that the last query of query tile qt sees.
T2W_DEV int tile_keys(int f, int kv, int causal, int tq, int qt) {
  const int behind = f - (qt + 1) * tq;  // queries behind the tile (it may be the last, and not whole)
  return causal && behind > 0 ? max(kv - behind, 0) : kv;
}
// Key tiles of a segment: one at least, so that rows that see nothing are written too.
T2W_DEV int seg_tiles(int keys, int kt) { return keys > 0 ? (keys + kt - 1) / kt : 1; }
// Key tiles of the first x query tiles of one key head.
T2W_DEV long long tiles_before(int f, int kv, int causal, int tq, int kt, int x) {
  if (x <= 0) return 0;
  if (!causal) return (long long)x * seg_tiles(kv, kt);
  if (x == 1) return seg_tiles(tile_keys(f, kv, causal, tq, 0), kt);
  const int c = kv - f + tq;           // keys of query tile 0, were the last tile whole
  int none = c > 0 ? 0 : -c / tq + 1;  // query tiles that see nothing
  if (none > x) none = x;
  long long s = none;
  if (none < x) {
    s += sum_of_quotients(x - none, kt, tq, c + none * tq + kt - 1);
    const long long last = (long long)c + (long long)(x - 1) * tq;
    if (last > kv) s += seg_tiles(kv, kt) - (int)((last + kt - 1) / kt);
  }
  return s;
}

// ---------------------------------------------------------------- numbers
// The scale's exponent for a largest magnitude (finite): the least e with amax <= 448 2^e, kept in range.
T2W_DEV int scale_exp(float amax) {
  if (amax == 0.f) return kScaleMin;
  const int e = (int)ue8m0_for_amax(amax) - 127;
  return e < kScaleMin ? kScaleMin : e > kScaleMax ? kScaleMax : e;
}
T2W_DEV float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// Two e4m3 codes as two halves (exact).
T2W_DEV uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)v));
  return r;
}

// Four codes as two pairs of halves: lo of the lower two.
T2W_DEV uint2 e4m3x4_to_f16x4(uint32_t v) {
  uint2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(r.x), "=r"(r.y)
      : "r"(v));
  return r;
}

}  // namespace t2w
