// Rotary positions with one or more axes: pair i of each head turns by the angle p[axis_i][row] * f_i,
//   (x, y) -> (x cos - y sin, y cos + x sin),
// forward or back (the inverse rotation, which is also the gradient), for the heads of q and of k in one launch.  Bound by
// the bytes of q and k, read and written once.
//
// Angles: the table holds each frequency as a fraction of a turn in 64-bit fixed point, f_i / (2 pi) * 2^64.  A product
// with a whole position, taken modulo 2^64, is the angle modulo a turn, with no reduction and an error of |p| 2^-65
// turns; fp32 would be off by a tenth of a radian at a million.  Sine and cosine are taken once for each row and pair and shared by
// all heads through shared memory; a thread's first loads are under way meanwhile.
#include "common.cuh"
#include "kernels.h"
#include "w4.h"

#include <algorithm>
#include <cstdlib>

namespace t2w {
namespace {

constexpr int kMaxThreads = 256, kPieces = 1024;  // of a block

struct RotDev {
  const uint16_t* in[2];
  uint16_t* out[2];
  int64_t in_row[2], in_head[2], out_row[2], out_head[2];
  const void* positions;
  int64_t pos_ld;
  const uint64_t* table;  // [pairs] frequencies, [pairs] axes
  int rows, heads_q, heads, pairs, pieces, axes, wide, negate;
  int per_block;           // rows of a block
  int items;               // pieces of a row: (heads) x (rotated pieces of 16 values, then kept ones of 8)
  int turned;              // rotated pieces of a head
  uint32_t inv_items, inv_pieces;  // ceil(2^32 / .)
};

// n / d for n, d < 2^16 by d's reciprocal ceil(2^32 / d) (d > 1: for d = 1 it does not fit and is told by 0)
T2W_DEV int div16(int n, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)n, inv) : n; }

template <bool HALF>
T2W_DEV float2 widen2(uint32_t v) {
  if constexpr (HALF) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <bool HALF>
T2W_DEV uint32_t narrow2(float a, float b) {
  if constexpr (HALF) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(a, b);
}

struct Piece {
  const uint16_t* src;
  uint16_t* dst;
  int64_t second;  // distance of the second 8 values
  int row, pair;   // row of the block; first pair, -1: kept as it is
};

template <bool ADJACENT>
T2W_DEV Piece piece_of(const RotDev& p, int item, int64_t row0) {
  Piece r;
  r.row = div16(item, p.inv_items);
  const int in_row = item - r.row * p.items;
  const int head = div16(in_row, p.inv_pieces), c = in_row - head * p.pieces;
  const int which = head >= p.heads_q, h = which ? head - p.heads_q : head;
  const int64_t row = row0 + r.row;
  const bool turn = c < p.turned;
  const int first = turn ? (ADJACENT ? 16 * c : 8 * c) : 2 * p.pairs + 8 * (c - p.turned);
  r.src = p.in[which] + row * p.in_row[which] + h * p.in_head[which] + first;
  r.dst = p.out[which] + row * p.out_row[which] + h * p.out_head[which] + first;
  r.second = ADJACENT ? 8 : p.pairs;
  r.pair = turn ? 8 * c : -1;
  return r;
}

template <bool HALF, bool ADJACENT>
__global__ void __launch_bounds__(kMaxThreads, 6) k_rotary(const RotDev p) {
  extern __shared__ float2 turn[];  // [rows of the block][pairs] cosine, sine
  pdl_wait();
  pdl_launch();
  const int64_t row0 = (int64_t)blockIdx.x * p.per_block;
  const int rows = (int)(p.rows - row0 < p.per_block ? p.rows - row0 : p.per_block), total = rows * p.items;
  int item = threadIdx.x;
  Piece at = {};
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (item < total) {
    at = piece_of<ADJACENT>(p, item, row0);
    a = *reinterpret_cast<const uint4*>(at.src);
    if (at.pair >= 0) b = *reinterpret_cast<const uint4*>(at.src + at.second);
  }
  for (int i = threadIdx.x; i < rows * p.pairs; i += blockDim.x) {
    const int r = i / p.pairs, j = i - r * p.pairs;
    const int axis = min(max((int)p.table[p.pairs + j], 0), p.axes - 1);
    const int64_t from = axis * p.pos_ld + row0 + r;
    const int64_t pos = p.wide ? static_cast<const int64_t*>(p.positions)[from] : static_cast<const int32_t*>(p.positions)[from];
    const int32_t part = (int32_t)(((uint64_t)pos * p.table[j]) >> 32);  // of a turn, in 2^-32
    float s, c;
    sincospif((float)part * 0x1p-31f, &s, &c);
    turn[i] = make_float2(c, p.negate ? -s : s);
  }
  __syncthreads();
  while (item < total) {
    const int next = item + blockDim.x;
    Piece to = {};
    uint4 na = make_uint4(0, 0, 0, 0), nb = na;
    if (next < total) {
      to = piece_of<ADJACENT>(p, next, row0);
      na = *reinterpret_cast<const uint4*>(to.src);
      if (to.pair >= 0) nb = *reinterpret_cast<const uint4*>(to.src + to.second);
    }
    if (at.pair < 0) {
      *reinterpret_cast<uint4*>(at.dst) = a;
    } else {
      const float2* cs = turn + at.row * p.pairs + at.pair;
      uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
      if constexpr (ADJACENT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = widen2<HALF>(u[i]), y = widen2<HALF>(v[i]), e = cs[i], f = cs[i + 4];
          u[i] = narrow2<HALF>(x.x * e.x - x.y * e.y, x.y * e.x + x.x * e.y);
          v[i] = narrow2<HALF>(y.x * f.x - y.y * f.y, y.y * f.x + y.x * f.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = widen2<HALF>(u[i]), y = widen2<HALF>(v[i]), e = cs[2 * i], f = cs[2 * i + 1];
          u[i] = narrow2<HALF>(x.x * e.x - y.x * e.y, x.y * f.x - y.y * f.y);
          v[i] = narrow2<HALF>(y.x * e.x + x.x * e.y, y.y * f.x + x.y * f.y);
        }
      }
      *reinterpret_cast<uint4*>(at.dst) = make_uint4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<uint4*>(at.dst + at.second) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    item = next;
    at = to;
    a = na;
    b = nb;
  }
}

uint32_t inverse_of(int d) { return d > 1 ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u; }

// Whether [rows][heads][hd] at these pitches has no two values in one place.
bool apart(int64_t rows, int64_t heads, int64_t hd, int64_t row_ld, int64_t head_ld) {
  if (heads > 1 && head_ld < hd) return false;
  if (rows > 1 && row_ld < hd) return false;
  return rows == 1 || heads == 1 || row_ld >= (heads - 1) * head_ld + hd || head_ld >= (rows - 1) * row_ld + hd;
}

// Whether a stretch of hd values every q_ld from 0 on (q_heads of them) meets one of hd every k_ld from `at` on.
bool meet(int64_t q_heads, int64_t q_ld, int64_t k_heads, int64_t k_ld, int64_t at, int64_t hd) {
  for (int64_t h = 0; h < k_heads; ++h) {
    const int64_t from = at + h * k_ld;
    // the last of q's that begins at or before it, and the next
    const int64_t i = q_heads > 1 && from > 0 ? std::min(from / q_ld, q_heads - 1) : 0;
    for (int64_t j = i; j <= i + 1 && j < q_heads; ++j)
      if (j * q_ld < from + hd && from < j * q_ld + hd) return true;
  }
  return false;
}

// Whether the outputs of q and k share memory, as far as that shows: the same place, or rows at one pitch, head by head (heads of
// the two may alternate).  A row of k lies `column` behind one of q's and pitch - column before the next.
bool share(const t2w_rotary_rows& q, int64_t q_heads, const t2w_rotary_rows& k, int64_t k_heads, int64_t rows, int64_t hd) {
  if (q.out == k.out) return true;
  const int64_t pitch = q.out_row_ld, q_span = (q_heads - 1) * q.out_head_ld + hd, k_span = (k_heads - 1) * k.out_head_ld + hd;
  const int64_t apart = static_cast<const uint16_t*>(k.out) - static_cast<const uint16_t*>(q.out);
  auto at = [&](int64_t offset) { return meet(q_heads, q.out_head_ld, k_heads, k.out_head_ld, offset, hd); };
  if (rows == 1) return at(apart);
  if (pitch != k.out_row_ld || q_span > pitch || k_span > pitch) return false;
  const int64_t column = (apart % pitch + pitch) % pitch, behind = (apart - column) / pitch;  // k's row 0 in q's row `behind`
  return (std::abs(behind) < rows && at(column)) || (std::abs(behind + 1) < rows && at(column - pitch));
}

}  // namespace
}  // namespace t2w

using namespace t2w;

extern "C" int t2w_rotary(const t2w_rotary_args* a, void* stream) {
  if (!a) return T2W_ERR_INVALID;
  if (a->dtype != T2W_DT_BF16 && a->dtype != T2W_DT_FP16) return T2W_ERR_UNSUPPORTED;
  if (a->rows < 0 || a->q_heads < 0 || a->k_heads < 0 || a->head_dim <= 0 || a->head_dim % 8 || a->rotary_dim <= 0 ||
      a->rotary_dim % 16 || a->rotary_dim > a->head_dim || a->axes <= 0)
    return T2W_ERR_INVALID;
  const int64_t heads = (int64_t)a->q_heads + a->k_heads;
  if (a->rows == 0 || heads == 0) return T2W_OK;
  if (!a->positions || !a->table || (reinterpret_cast<uintptr_t>(a->table) & 7) ||
      (reinterpret_cast<uintptr_t>(a->positions) & (a->wide_positions ? 7 : 3)) || a->pos_ld < 0 ||
      (a->axes > 1 && a->pos_ld != 0 && a->pos_ld < a->rows))
    return T2W_ERR_INVALID;
  RotDev p = {};
  p.turned = a->rotary_dim / 16;
  const t2w_rotary_rows* s[2] = {&a->q, &a->k};
  const int64_t count[2] = {a->q_heads, a->k_heads};
  bool kept = false;  // values that do not turn and have to be copied
  for (int w = 0; w < 2; ++w) {
    if (count[w] == 0) continue;
    if (!s[w]->in || !s[w]->out || ((reinterpret_cast<uintptr_t>(s[w]->in) | reinterpret_cast<uintptr_t>(s[w]->out)) & 15) ||
        s[w]->in_row_ld % 8 || s[w]->in_head_ld % 8 || s[w]->out_row_ld % 8 || s[w]->out_head_ld % 8 || s[w]->in_row_ld < 0 ||
        s[w]->in_head_ld < 0 || !apart(a->rows, count[w], a->head_dim, s[w]->out_row_ld, s[w]->out_head_ld))
      return T2W_ERR_INVALID;
    if (s[w]->in == s[w]->out && ((a->rows > 1 && s[w]->in_row_ld != s[w]->out_row_ld) ||
                                  (count[w] > 1 && s[w]->in_head_ld != s[w]->out_head_ld)))
      return T2W_ERR_INVALID;
    if (s[w]->in != s[w]->out) kept = true;
    p.in[w] = static_cast<const uint16_t*>(s[w]->in);
    p.out[w] = static_cast<uint16_t*>(s[w]->out);
    p.in_row[w] = s[w]->in_row_ld;
    p.in_head[w] = s[w]->in_head_ld;
    p.out_row[w] = s[w]->out_row_ld;
    p.out_head[w] = s[w]->out_head_ld;
  }
  if (p.in[0] && p.in[1] && share(a->q, a->q_heads, a->k, a->k_heads, a->rows, a->head_dim)) return T2W_ERR_INVALID;
  p.pieces = p.turned + (kept ? (a->head_dim - a->rotary_dim) / 8 : 0);
  if (heads * p.pieces > 32767 || a->rotary_dim > 4096) return T2W_ERR_UNSUPPORTED;
  p.positions = a->positions;
  p.pos_ld = a->pos_ld;
  p.table = static_cast<const uint64_t*>(a->table);
  p.rows = a->rows;
  p.heads_q = a->q_heads;
  p.heads = (int)heads;
  p.pairs = a->rotary_dim / 2;
  p.axes = a->axes;
  p.wide = a->wide_positions != 0;
  p.negate = a->inverse != 0;
  p.items = (int)heads * p.pieces;
  p.inv_items = inverse_of(p.items);
  p.inv_pieces = inverse_of(p.pieces);
  // Rows of a block: as many as bring it about 1024 pieces (its threads then take about as many sines as it has threads, and
  // each has its next piece under way while it turns one), but no more than leave four blocks for each SM.
  p.per_block = std::max(1, std::min({kPieces / p.items, a->rows / (4 * num_sms()), 4096 / p.pairs}));
  const int total = std::min(p.per_block, a->rows) * p.items, rounds = (total + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((total + rounds - 1) / rounds + 31) / 32 * 32;
  const dim3 grid((unsigned)(((int64_t)a->rows + p.per_block - 1) / p.per_block));
  const size_t smem = (size_t)p.per_block * p.pairs * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == T2W_DT_FP16)
    e = a->adjacent ? launch_k(k_rotary<true, true>, grid, dim3(threads), smem, st, p)
                    : launch_k(k_rotary<true, false>, grid, dim3(threads), smem, st, p);
  else
    e = a->adjacent ? launch_k(k_rotary<false, true>, grid, dim3(threads), smem, st, p)
                    : launch_k(k_rotary<false, false>, grid, dim3(threads), smem, st, p);
  if (e == cudaSuccess) return T2W_OK;
  set_cuda_error(e);
  return T2W_ERR_CUDA;
}
