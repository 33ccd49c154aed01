// Attention over the paged 8-bit cache.
//
// Mathematics: row i of request r and query head h sees the keys j < end(i) of key head h / group, with end(i) the
// request's key count, or where the call is causal the count less the queries behind i; x_j = scale q . k_j, and
// o = sum_j 2^(c x_j - m) v_j / sum_j 2^(c x_j - m), c = log2 e, with the running maximum m of one pass over the keys.
// A row that sees no key gives zeros and the log-sum -inf.
#include "paged.h"

namespace t2w {
namespace {

struct AttnDev {
  const void* q;
  long long q_row_ld, q_head_ld;
  const uint8_t* codes[2];
  const float* scales[2];
  long long page_ld[2], scale_ld[2];
  const int* table;
  int table_ld, page, shift, pages, rows, q_heads, kv_heads, causal;
  float scale;
  const PlanHead* head;
  const int *q_start, *kv_len, *request;
  void* out;
  float* lse;
  int* status;
};

template <bool HALF>
T2W_DEV float load16(const uint16_t* p) {
  const uint32_t u = *p;
  if constexpr (HALF) return __half2float(*reinterpret_cast<const __half*>(&u));
  return __uint_as_float(u << 16);
}

// One warp: one row and query head; a lane scores one key of 32 and then holds HD / 32 columns of the output.
template <int HD, bool HALF>
__global__ void __launch_bounds__(128) k_paged_rows(const AttnDev p) {
  __shared__ float qs[4][HD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long unit = (long long)blockIdx.x * 4 + warp;
  pdl_wait();
  pdl_launch();
  if (unit >= (long long)p.rows * p.q_heads) return;
  const int row = (int)(unit / p.q_heads), h = (int)(unit % p.q_heads), hk = h / (p.q_heads / p.kv_heads);
  constexpr int N = HD / 32;
  float o[N] = {};
  float m = -INFINITY, l = 0.f;
  const bool used = row < p.head->used;
  if (used) {
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + row * p.q_row_ld + h * p.q_head_ld;
    for (int i = lane; i < HD; i += 32) qs[warp][i] = load16<HALF>(q + i) * p.scale * 1.4426950408889634f;
    __syncwarp();
    const int r = p.request[row];
    const int end = p.causal ? p.kv_len[r] - (p.q_start[r + 1] - row) + 1 : p.kv_len[r];
    for (int j0 = 0; j0 < end; j0 += 32) {
      const int j = j0 + lane;
      float x = -INFINITY, sv = 0.f;
      int g = 0;
      if (j < end) {
        g = p.table[(size_t)r * p.table_ld + (j >> p.shift)];
        if ((unsigned)g >= (unsigned)p.pages) {
          atomicExch(p.status, T2W_ERR_INVALID);
          g = 0;
        }
        const uint8_t* k = p.codes[0] + g * p.page_ld[0] + ((size_t)hk * p.page + (j & (p.page - 1))) * HD;
        float s = 0.f;
        for (int i = 0; i < HD; i += 2) {
          const uint32_t f = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(k + i));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&f));
          s += v.x * qs[warp][i] + v.y * qs[warp][i + 1];
        }
        x = s * p.scales[0][g * p.scale_ld[0] + hk];
        sv = p.scales[1][g * p.scale_ld[1] + hk];
      }
      float top = x;
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      const float m_new = fmaxf(m, top), f = m == -INFINITY ? 0.f : exp2f(m - m_new);
      const float e = j < end ? exp2f(x - (m_new == -INFINITY ? 0.f : m_new)) : 0.f;
      l = l * f + warp_sum(e);
      m = m_new;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] *= f;
      for (int t = 0; t < 32 && j0 + t < end; ++t) {
        const int gt = __shfl_sync(~0u, g, t);
        const float w = __shfl_sync(~0u, e * sv, t);
        const uint8_t* v = p.codes[1] + gt * p.page_ld[1] + ((size_t)hk * p.page + ((j0 + t) & (p.page - 1))) * HD;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t f2 = e4m3x2_to_f16x2(v[lane + 32 * i]);
          o[i] += w * __low2float(*reinterpret_cast<const __half2*>(&f2));
        }
      }
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint16_t* out = static_cast<uint16_t*>(p.out) + ((size_t)row * p.q_heads + h) * HD;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (HALF) reinterpret_cast<__half*>(out)[lane + 32 * i] = __float2half_rn(o[i] * inv);
    else reinterpret_cast<__nv_bfloat16*>(out)[lane + 32 * i] = __float2bfloat16_rn(o[i] * inv);
  }
  if (p.lse && lane == 0) p.lse[(size_t)row * p.q_heads + h] = l != 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace
}  // namespace t2w

using namespace t2w;

extern "C" size_t t2w_paged_workspace_bytes(int32_t max_fresh, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
  (void)max_fresh;
  (void)q_heads;
  (void)kv_heads;
  (void)head_dim;
  return 16;
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
  const PlanLayout l = paged_layout(a->requests, a->rows, a->page,
                                    paged_cut(a->max_fresh, a->q_heads, a->kv_heads, a->head_dim));
  p.table = a->table;
  p.table_ld = a->table_ld;
  p.page = a->page;
  p.shift = a->page == 16 ? 4 : a->page == 32 ? 5 : a->page == 64 ? 6 : 7;
  p.pages = a->pages;
  p.rows = a->rows;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.causal = a->causal != 0;
  p.scale = a->scale;
  p.head = reinterpret_cast<const PlanHead*>(a->plan);
  p.q_start = a->plan + l.q_start;
  p.kv_len = a->plan + l.kv_len;
  p.request = a->plan + l.request;
  p.out = a->out;
  p.lse = a->lse;
  p.status = const_cast<int*>(&p.head->status);
  if (a->rows == 0) return T2W_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)(((long long)a->rows * a->q_heads + 3) / 4));
  const bool half = a->dtype == T2W_DT_FP16;
  cudaError_t e;
  if (a->head_dim == 64) e = half ? launch_k(k_paged_rows<64, true>, grid, dim3(128), 0, st, p) : launch_k(k_paged_rows<64, false>, grid, dim3(128), 0, st, p);
  else e = half ? launch_k(k_paged_rows<128, true>, grid, dim3(128), 0, st, p) : launch_k(k_paged_rows<128, false>, grid, dim3(128), 0, st, p);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return T2W_ERR_CUDA;
  }
  return T2W_OK;
}
