// 4-bit weights: laying codes, scales and zeros out (once, when a weight is loaded), reading them back, and the C entries of
// the products.  The kernels here run at load time and are bound by their scattered byte reads; the products are in
// w4_few.cu and w4_many.cu.
#include "w4.h"

namespace t2w {
namespace {

struct PackDev {
  uint8_t* buffer;
  const uint8_t* codes[2];  // plain: [0]; gated: gate, up
  const uint16_t* scales[2];
  const uint8_t* zeros[2];
  int64_t code_ld[2], scale_ld[2], zero_ld[2];
  float* out[2];  // unpacking: fp32 [n][k]
  int64_t out_ld[2];
  int n, k, group, tiles_k, gated, has_zeros, scale_half;
  int64_t tiles;
};

// Source matrix and row of packed row r; row -1 past the end.
T2W_DEV void source_of(const PackDev& p, int64_t r, int& which, int64_t& row) {
  which = p.gated ? (int)(r >> 3) & 1 : 0;
  row = p.gated ? (r >> 4) * 8 + (r & 7) : r;
  if (row >= p.n) row = -1;
}

// A block for each tile: 1024 words of codes, then scales and zeros.
__global__ void __launch_bounds__(256) k_w4_pack(const PackDev p) {
  const int64_t tile = blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
  if (tile >= p.tiles) return;
  const int groups = kW4K / p.group, bytes = w4_tile_bytes(p.group, p.has_zeros);
  const int64_t rb = tile / p.tiles_k;
  const int k0 = (int)(tile % p.tiles_k) * kW4K;
  uint8_t* out = p.buffer + kW4Header + tile * bytes;
  if (tile == 0 && threadIdx.x < kW4Header / 4) reinterpret_cast<uint32_t*>(p.buffer)[threadIdx.x] = 0;
  for (int w = threadIdx.x; w < kW4Codes / 4; w += 256) {
    const int j = w & 3, lane = (w >> 2) & 31, kb = (w >> 7) & 1, strip = w >> 8;
    const int g = lane >> 2, t = lane & 3;
    uint32_t word = 0;
    for (int i = 0; i < 4; ++i) {
      int which;
      int64_t row;
      source_of(p, rb * kW4Rows + strip * 16 + (i & 1) * 8 + g, which, row);
      const int k = k0 + kb * 64 + 16 * j + 4 * t + (i >> 1) * 2;
      for (int e = 0; e < 2; ++e) {
        uint32_t c = p.has_zeros ? 0u : 8u;
        if (row >= 0 && k + e < p.k) c = p.codes[which][row * p.code_ld[which] + k + e] & 15u;
        word |= c << (4 * i + 16 * e);
      }
    }
    reinterpret_cast<uint32_t*>(out)[w] = word;
  }
  for (int i = threadIdx.x; i < groups * kW4Rows; i += 256) {
    const int r = i % kW4Rows, gr = i / kW4Rows;
    const int64_t at = (int64_t)k0 / p.group + gr;
    int which;
    int64_t row;
    source_of(p, rb * kW4Rows + r, which, row);
    const bool in = row >= 0 && at < p.k / p.group;
    reinterpret_cast<uint16_t*>(out + kW4Codes)[gr * kW4Rows + w4_place(r)] =
        in ? p.scales[which][row * p.scale_ld[which] + at] : (uint16_t)0;
    if (p.has_zeros)
      out[kW4Codes + groups * 128 + gr * kW4Rows + w4_place(r)] = in ? p.zeros[which][row * p.zero_ld[which] + at] & 15 : 0;
  }
}

// (code - zero) * scale, exact in fp32: 5 bits by 11.
__global__ void __launch_bounds__(256) k_w4_unpack(const PackDev p) {
  const int64_t tile = blockIdx.x + (int64_t)blockIdx.y * gridDim.x;
  if (tile >= p.tiles) return;
  const int groups = kW4K / p.group, bytes = w4_tile_bytes(p.group, p.has_zeros);
  const int64_t rb = tile / p.tiles_k;
  const int k0 = (int)(tile % p.tiles_k) * kW4K;
  const uint8_t* in = p.buffer + kW4Header + tile * bytes;
  for (int e = threadIdx.x; e < kW4Rows * kW4K; e += 256) {
    const int k = e % kW4K, r = e / kW4K;
    int which;
    int64_t row;
    source_of(p, rb * kW4Rows + r, which, row);
    if (row < 0 || k0 + k >= p.k) continue;
    const int kb = k >> 6, j = (k >> 4) & 3, t = (k >> 2) & 3, strip = r >> 4, g = r & 7;
    const int i = ((k >> 1) & 1) * 2 + ((r >> 3) & 1);
    const uint32_t word = reinterpret_cast<const uint32_t*>(in)[((strip * 2 + kb) * 32 + g * 4 + t) * 4 + j];
    const int code = (word >> (4 * i + 16 * (k & 1))) & 15, gr = k / p.group;
    const int zero = p.has_zeros ? in[kW4Codes + groups * 128 + gr * kW4Rows + w4_place(r)] : 8;
    const float s = w4_scale(reinterpret_cast<const uint16_t*>(in + kW4Codes)[gr * kW4Rows + w4_place(r)], p.scale_half);
    p.out[which][row * p.out_ld[which] + k0 + k] = (float)(code - zero) * s;
  }
}

bool sizes_ok(int32_t n, int32_t k, int32_t group) {
  return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128) && k % group == 0 && n <= (1 << 30) && k <= (1 << 24);
}

// The parts of pack and unpack that are alike; a status.
int fill(PackDev& p, const t2w_w4_weight* w) {
  if (!w || !w->buffer || (reinterpret_cast<uintptr_t>(w->buffer) & 127) || !sizes_ok(w->n, w->k, w->group) ||
      (w->scale_dtype != T2W_DT_BF16 && w->scale_dtype != T2W_DT_FP16))
    return T2W_ERR_INVALID;
  p.buffer = static_cast<uint8_t*>(w->buffer);
  p.n = w->n;
  p.k = w->k;
  p.group = w->group;
  p.gated = w->gated != 0;
  p.has_zeros = w->zeros != 0;
  p.scale_half = w->scale_dtype == T2W_DT_FP16;
  p.tiles_k = (w->k + kW4K - 1) / kW4K;
  p.tiles = (w4_rows(w->n, p.gated) + kW4Rows - 1) / kW4Rows * p.tiles_k;
  return T2W_OK;
}
dim3 tile_grid(int64_t tiles) { return dim3(65535 < tiles ? 65535 : (unsigned)tiles, (unsigned)((tiles + 65534) / 65535)); }

// Whether a pointer lies on `bytes` (a power of two).
bool lies_on(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int done(cudaError_t e) {
  if (e == cudaSuccess) return T2W_OK;
  set_cuda_error(e);
  return T2W_ERR_CUDA;
}

}  // namespace
}  // namespace t2w

using namespace t2w;

extern "C" int64_t t2w_w4_bytes(int32_t n, int32_t k, int32_t group, int32_t zeros, int32_t gated) {
  if (!sizes_ok(n, k, group)) return T2W_ERR_INVALID;
  return kW4Header + (w4_rows(n, gated != 0) + kW4Rows - 1) / kW4Rows * ((k + kW4K - 1) / kW4K) *
                         (int64_t)w4_tile_bytes(group, zeros != 0);
}

extern "C" int t2w_w4_pack(const t2w_w4_weight* w, const t2w_w4_source* a, const t2w_w4_source* b, void* stream) {
  PackDev p = {};
  if (const int e = fill(p, w)) return e;
  const t2w_w4_source* src[2] = {a, b};
  if (!a || (p.gated && !b)) return T2W_ERR_INVALID;
  for (int i = 0; i < (p.gated ? 2 : 1); ++i) {
    if (!src[i]->codes || !src[i]->scales || !lies_on(src[i]->scales, 2) || (p.has_zeros && !src[i]->zeros))
      return T2W_ERR_INVALID;
    p.codes[i] = static_cast<const uint8_t*>(src[i]->codes);
    p.scales[i] = static_cast<const uint16_t*>(src[i]->scales);
    p.zeros[i] = static_cast<const uint8_t*>(src[i]->zeros);
    p.code_ld[i] = src[i]->code_ld;
    p.scale_ld[i] = src[i]->scale_ld;
    p.zero_ld[i] = src[i]->zero_ld;
  }
  // no programmatic launch: what packs is complete before what follows it begins
  k_w4_pack<<<tile_grid(p.tiles), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return done(cudaGetLastError());
}

extern "C" int t2w_w4_unpack(const t2w_w4_weight* w, float* a, int64_t a_ld, float* b, int64_t b_ld, void* stream) {
  PackDev p = {};
  if (const int e = fill(p, w)) return e;
  if (!a || (p.gated && !b) || !lies_on(a, 4) || (p.gated && !lies_on(b, 4)) ||
      (p.n > 1 && (a_ld < p.k || (p.gated && b_ld < p.k))))
    return T2W_ERR_INVALID;
  p.out[0] = a;
  p.out[1] = b;
  p.out_ld[0] = a_ld;
  p.out_ld[1] = b_ld;
  k_w4_unpack<<<tile_grid(p.tiles), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return done(cudaGetLastError());
}

extern "C" int t2w_w4_status(const t2w_w4_weight* w, void* stream) {
  if (!w || !w->buffer) return T2W_ERR_INVALID;
  int32_t s = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(&s, w->buffer, sizeof(s), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && s != T2W_OK) {  // told once: products after it are judged by themselves
    e = cudaMemsetAsync(w->buffer, 0, sizeof(s), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e == cudaSuccess) return s;
  return done(e);
}

extern "C" int t2w_w4_linear(const t2w_w4_linear_args* a, void* stream) {
  if (!a) return T2W_ERR_INVALID;
  PackDev w = {};
  if (const int e = fill(w, &a->w)) return e;
  if (a->dtype != T2W_DT_BF16 && a->dtype != T2W_DT_FP16) return T2W_ERR_UNSUPPORTED;
  if (a->rows < 0 || (w.gated && a->act != T2W_ACT_SILU && a->act != T2W_ACT_GELU_TANH)) return T2W_ERR_INVALID;
  if (w.gated && (a->bias || a->residual)) return T2W_ERR_INVALID;
  if (a->rows == 0) return T2W_OK;
  // x is read in 16-byte pieces
  if (!a->x || !a->out || !lies_on(a->x, 16) || a->x_ld % 8 || a->x_ld < 0 || !lies_on(a->out, 2) || !lies_on(a->bias, 2) ||
      !lies_on(a->residual, 2) || (a->rows > 1 && a->x_ld < a->w.k) ||
      (a->residual && a->rows > 1 && a->res_ld < a->w.n))
    return T2W_ERR_INVALID;
  W4Dev p = {};
  p.tiles = w.buffer + kW4Header;
  p.status = reinterpret_cast<int*>(w.buffer);
  p.x = a->x;
  p.x_ld = a->x_ld;
  p.rows = a->rows;
  p.k = w.k;
  p.n = w.n;
  p.tiles_k = w.tiles_k;
  p.blocks = (int)(w.tiles / w.tiles_k);
  p.scale_half = w.scale_half;
  p.act = a->act;
  p.bias = a->bias;
  p.residual = a->residual;
  p.res_ld = a->res_ld;
  p.out = a->out;
  // A pass over the weights for every 8 rows against one for all, 16 rows in this form and 17 on tcgen05 (us): k x n 4096 x 6144 10.8
  // and 12.0, 11008 x 4096 15.4 and 15.5, 1024 x 1024 4.3 and 4.9, gated 4096 x 11008 25.6 and 33, 2048 x 5632 10.3 and 11.6; a
  // third pass is slower (32 x 4096 x 6144: 22 for 12).
  const auto launch = a->rows <= 16 ? launch_w4_few : launch_w4_many;
  return done(launch(p, w.group, w.has_zeros, w.gated, a->dtype == T2W_DT_FP16, static_cast<cudaStream_t>(stream)));
}
