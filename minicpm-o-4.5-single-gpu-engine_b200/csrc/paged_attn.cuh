// What the forms of the paged attention share: the arguments, a finished row's store, the queries as halves, and the
// parts of segments that were cut.
#pragma once

#include "paged.h"

namespace t2w {

struct AttnDev {
  const void* q;
  long long q_row_ld, q_head_ld;
  const uint8_t* codes[2];
  const float* scales[2];
  long long page_ld[2], scale_ld[2];
  const int* table;
  int table_ld, page, shift, pages, rows, q_heads, kv_heads, causal;
  int group, group_mul;  // query heads to a key head, and ceil(2^16 / group)
  float scale;
  const PlanHead* head;
  const int *q_start, *kv_len;
  const int4* starts;  // two entries for each worker
  int tq, kt, part_rows, block_workers;
  float* ws;  // the parts of cut segments, two for each worker
  void* out;
  float* lse;
  int* status;
};

// row / group for a row of a tile: exact below 128 rows, where row (group_mul group - 2^16) < 2^14.
T2W_DEV int over_group(const AttnDev& p, int row) { return row * p.group_mul >> 16; }

// Four columns of a finished row: O / l, and with the first columns its log-sum.
template <bool HALF>
T2W_DEV void store_row(const AttnDev& p, int row, int head, int hd, int d, float4 o, float M, float l) {
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint2 u;
  if constexpr (HALF) {
    const __half2 a = __floats2half2_rn(o.x * inv, o.y * inv), b = __floats2half2_rn(o.z * inv, o.w * inv);
    u = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    u = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + ((size_t)row * p.q_heads + head) * hd + d) = u;
  if (d == 0 && p.lse)
    p.lse[(size_t)row * p.q_heads + head] = l != 0.f ? (M + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// The cache streams through L2 (evicted first), so that the plan, the tables and the parts stay there.
T2W_DEV uint64_t l2_policy_evict_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
// x * 2^e for |e| up to 254 without leaving the range on the way.
T2W_DEV float scaled(float x, int e) {
  const int a = e / 2;
  return x * exp2i(a) * exp2i(e - a);
}
T2W_DEV uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One query row's factor for halves: the exponent shift that brings its largest magnitude into [2^14, 2^15), so that
// bf16 rows keep all their bits over 2^28 of range as halves.  Half rows and rows that are not finite stay as they are.
template <bool HALF>
T2W_DEV int row_shift(uint32_t max_bits16) {
  if (HALF || max_bits16 == 0 || max_bits16 >= 0x7f80u) return 0;
  return min(14 - ((int)(max_bits16 >> 7) - 127), 127);
}
template <bool HALF>
T2W_DEV uint32_t row_half2(uint32_t u, int shift, bool negate) {
  if constexpr (HALF) return negate ? u ^ 0x80008000u : u;
  const float f = negate ? -exp2i(shift) : exp2i(shift);
  return pack_f16x2(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f);
}

constexpr float kLog2e = 1.4426950408889634f;
// A weight is 2^(x + log2 s_v - M) in a half: M is set 9 below a row's largest exponent and again when that would pass M
// by more than 15 (65504 is the largest half), so that the largest weight is 2^9 or more and what falls under the halves'
// smallest, 2^-25, is 2^-34 of the largest contribution.
// The sum of exponentials is of fp32 numbers in units of 2^M, so a page with a value scale 2^s under the one that sets M loses
// terms below 2^(s - 117) of the largest.  From s = 90 on that shows: not with half values, whose scales span 2^72 (zeros
// have 2^-64), nor with bf16 values up to 3e10.
constexpr float kRaise = 15.f, kBelow = 9.f;

// A worker's unfinished rows of a segment: O [rows][HD], then the reference exponents [rows] and the sums [rows].
T2W_DEV float* part_of(float* ws, int slot, int rows, int hd) { return ws + (size_t)slot * rows * (hd + 2); }

// A block's walk over its segments.
struct Walk {
  int r, hk, qt;       // the segment
  int row0, f, kv;     // its request's first row, rows and keys
  int kt0, kt1, nt;    // the tiles of it that are this worker's, and all of them
  int zero, stop;      // the place of its tile 0; the end of the worker's places
  int extra;
  bool first;

  T2W_DEV void cut(const AttnDev& p, int from) {
    nt = seg_tiles(tile_keys(f, kv, p.causal, p.tq, qt), p.kt);
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
    stop = p.starts[2 * w + 3].w;
    zero = of.w - s.w;
    if (zero >= stop) return false;
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
  T2W_DEV int rows(const AttnDev& p, int group) const { return min(p.tq, f - qt * p.tq) * group; }
};

// Segments of up to 128 query rows on tcgen05 tiles (paged_attn_tc.cu): the parts of cut segments into p.ws.
cudaError_t launch_paged_many(const AttnDev& p, const PagedCut& cut, int head_dim, bool half, cudaStream_t st);

}  // namespace t2w
