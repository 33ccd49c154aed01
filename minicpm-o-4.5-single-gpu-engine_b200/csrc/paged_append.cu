// New keys and values into the pages of the 8-bit cache.
//
// Mathematics, for each page and head that a step's rows go into: a = max |x| over the step's rows of that page and
// head, the scale s = max(s_old, 2^e) with e the least exponent for which a <= 448 2^e (448: the largest e4m3 number;
// s_old only where the page held rows before), the codes e4m3(x / s) rounded to nearest even, and the older codes c
// rounded again to e4m3(c s_old / s) where s grew.  A run (the rows of one request that go into one page, from the plan)
// and a head are written by one block alone, so nothing is added or compared across blocks: no atomics, and the same
// bits whatever the order.
//
// Bound: HBM for prompts (two bytes read for each element and one written; one read of the rows, which stay in
// registers between the search for the largest magnitude and the rounding), latency for single tokens.  Measured: 16 prompts
// of 1900 to 6300 rows, 8 heads of 128: 404 MB in 63.3 us, 6.4 TB/s, what a plain copy reaches; 128 windows of 50 rows, 8
// heads of 64: 23.9 MB in 7.3 us; 4 single rows 7.3 us, which is what the call costs on the host.
#include "paged.h"

namespace t2w {
namespace {

constexpr int kThreads = 128;

struct AppendDev {
  const void* x[2];   // K and V rows, [rows, heads, hd]
  long long row_ld[2], head_ld[2];
  uint8_t* codes[2];  // [pages][heads][page][hd]
  float* scales[2];   // [pages][heads]
  long long page_ld[2], scale_ld[2];
  int page, heads, pages;
  const PlanHead* head;
  const int4* runs;
  int* status;
};

// The largest magnitude of packed 16-bit floats, by their bit patterns (sign off): a pattern from the exponent's all
// ones up is an infinity or a NaN.
T2W_DEV uint32_t max_bits(uint32_t m, uint4 v) {
  m = __vmaxu2(m, v.x & 0x7fff7fffu);
  m = __vmaxu2(m, v.y & 0x7fff7fffu);
  m = __vmaxu2(m, v.z & 0x7fff7fffu);
  return __vmaxu2(m, v.w & 0x7fff7fffu);
}
template <bool HALF>
T2W_DEV float2 unpack(uint32_t u) {
  if constexpr (HALF) return __half22float2(*reinterpret_cast<__half2*>(&u));
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <bool HALF>
T2W_DEV uint2 quantised(uint4 v, float inv) {
  const float2 a = unpack<HALF>(v.x), b = unpack<HALF>(v.y), c = unpack<HALF>(v.z), d = unpack<HALF>(v.w);
  return make_uint2(e4m3x4(a.x * inv, a.y * inv, b.x * inv, b.y * inv), e4m3x4(c.x * inv, c.y * inv, d.x * inv, d.y * inv));
}

// One block: one run and head, of K (blockIdx.z 0) or of V.  The run's rows stay in registers between the maximum and
// the rounding: PER 16-byte pieces a thread, enough for a whole page.
template <int HD, bool HALF, int PER>
__global__ void __launch_bounds__(kThreads) k_append(const AppendDev p) {
  __shared__ uint32_t warp_max[kThreads / 32];
  constexpr int kPieces = HD / 8;  // 16-byte pieces of a row
  const int tid = threadIdx.x, h = blockIdx.y, w = blockIdx.z;
  pdl_wait();
  pdl_launch();
  if ((int)blockIdx.x >= p.head->n_runs) return;
  const int4 run = p.runs[blockIdx.x];  // first row, rows, page, place of the first row in the page
  // The plan's pages come off a free list that may be longer than this layer's codes: what lies past them is not written.
  if ((unsigned)run.z >= (unsigned)p.pages) {
    if (tid == 0) atomicExch(p.status, T2W_ERR_INVALID);
    return;
  }
  float* const sp = p.scales[w] + run.z * p.scale_ld[w] + h;
  uint8_t* const page = p.codes[w] + run.z * p.page_ld[w] + (size_t)h * p.page * HD;
  const float s_old = run.w > 0 ? *sp : exp2i(kScaleMin);
  const uint16_t* const x = static_cast<const uint16_t*>(p.x[w]) + run.x * p.row_ld[w] + h * p.head_ld[w];
  const int n = run.y * kPieces;
  uint4 v[PER];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = tid + i * kThreads;
    v[i] = make_uint4(0, 0, 0, 0);
    if (c < n) v[i] = __ldg(reinterpret_cast<const uint4*>(x + (c / kPieces) * p.row_ld[w] + (c % kPieces) * 8));
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) m = max_bits(m, v[i]);
  m = max(m & 0xffffu, m >> 16);
  m = __reduce_max_sync(~0u, m);
  if ((tid & 31) == 0) warp_max[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) m = max(m, warp_max[i]);
  const bool odd = m >= (HALF ? 0x7c00u : 0x7f80u) || s_old != s_old;
  const float s_new = exp2i(scale_exp(odd ? 0.f : unpack<HALF>(m).x));
  const float s = fmaxf(s_old, s_new);
  if (tid == 0) *sp = odd ? __int_as_float(0x7fffffff) : s;
  // rows that are not finite leave finite codes behind their NaN scale: what reads the codes never meets a NaN in them
  const float inv = odd ? 0.f : exp2i(-scale_exp(s * 448.f));
  if (run.w > 0 && (s > s_old || odd)) {
    const float ratio = odd ? 0.f : s_old * inv;  // both powers of two: exact
    uint2* const old = reinterpret_cast<uint2*>(page);
    for (int c = tid; c < run.w * kPieces; c += kThreads) {
      uint2 u = old[c];
      uint32_t r[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t f = e4m3x2_to_f16x2(r[i]);
        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&f));
        r[i] = e4m3x2(g.x * ratio, g.y * ratio);
      }
      old[c] = make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
    }
  }
  uint2* const out = reinterpret_cast<uint2*>(page + (size_t)run.w * HD);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = tid + i * kThreads;
    if (c < n) out[c] = odd ? make_uint2(0, 0) : quantised<HALF>(v[i], inv);
  }
}

template <int HD, bool HALF>
cudaError_t launch_append(const AppendDev& p, int max_runs, cudaStream_t st) {
  const dim3 grid(max_runs, p.heads, 2);
  const int per = p.page * (HD / 8) / kThreads;  // 1 .. 16
  if (per <= 1) return launch_k(k_append<HD, HALF, 1>, grid, dim3(kThreads), 0, st, p);
  if (per <= 2) return launch_k(k_append<HD, HALF, 2>, grid, dim3(kThreads), 0, st, p);
  if (per <= 4) return launch_k(k_append<HD, HALF, 4>, grid, dim3(kThreads), 0, st, p);
  if (per <= 8) return launch_k(k_append<HD, HALF, 8>, grid, dim3(kThreads), 0, st, p);
  return launch_k(k_append<HD, HALF, 16>, grid, dim3(kThreads), 0, st, p);
}

}  // namespace
}  // namespace t2w

using namespace t2w;

extern "C" int t2w_paged_append(const t2w_paged_append_args* a, void* stream) {
  if (!a || !a->plan || !a->k || !a->v || !a->k_codes || !a->v_codes || !a->k_scale || !a->v_scale) return T2W_ERR_INVALID;
  if (a->dtype != T2W_DT_BF16 && a->dtype != T2W_DT_FP16) return T2W_ERR_UNSUPPORTED;
  const int64_t ints = t2w_paged_plan_ints(a->requests, a->rows, a->max_fresh, a->page, a->q_heads, a->kv_heads,
                                           a->head_dim, nullptr);
  if (ints < 0) return (int)ints;
  if (a->kv_heads > 65535 || a->pages <= 0) return T2W_ERR_INVALID;
  AppendDev p;
  const void* x[2] = {a->k, a->v};
  void* codes[2] = {a->k_codes, a->v_codes};
  float* scales[2] = {a->k_scale, a->v_scale};
  for (int w = 0; w < 2; ++w) {
    p.x[w] = x[w];
    p.row_ld[w] = w ? a->v_row_ld : a->k_row_ld;
    p.head_ld[w] = w ? a->v_head_ld : a->k_head_ld;
    p.codes[w] = static_cast<uint8_t*>(codes[w]);
    p.scales[w] = scales[w];
    p.page_ld[w] = w ? a->v_page_ld : a->k_page_ld;
    p.scale_ld[w] = w ? a->v_scale_ld : a->k_scale_ld;
    // rows and pages are read and written in 16- and 8-byte pieces
    if ((reinterpret_cast<uintptr_t>(x[w]) & 15) || p.row_ld[w] % 8 || p.head_ld[w] % 8 ||
        (reinterpret_cast<uintptr_t>(codes[w]) & 15) || p.page_ld[w] % 16)
      return T2W_ERR_INVALID;
    if (p.page_ld[w] < (int64_t)a->kv_heads * a->page * a->head_dim || p.scale_ld[w] < a->kv_heads) return T2W_ERR_INVALID;
  }
  p.page = a->page;
  p.heads = a->kv_heads;
  p.pages = a->pages;
  const PlanLayout l = paged_layout(a->requests, a->rows, a->page,
                                    paged_cut(a->max_fresh, a->q_heads, a->kv_heads, a->head_dim));
  p.head = reinterpret_cast<const PlanHead*>(a->plan);
  p.runs = reinterpret_cast<const int4*>(a->plan + l.runs);
  p.status = &reinterpret_cast<PlanHead*>(a->plan)->status;
  if (l.max_runs == 0) return T2W_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = a->dtype == T2W_DT_FP16;
  cudaError_t e;
  if (a->head_dim == 64) e = half ? launch_append<64, true>(p, l.max_runs, st) : launch_append<64, false>(p, l.max_runs, st);
  else e = half ? launch_append<128, true>(p, l.max_runs, st) : launch_append<128, false>(p, l.max_runs, st);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return T2W_ERR_CUDA;
  }
  return T2W_OK;
}
