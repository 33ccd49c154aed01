// torch custom ops over the C ABI of libt2w_b200.so: torch.ops.b200t2w.*.
//
// The reference engine calls its solver from torch code (BatchedToken2Wav -> FastDiT.solve,
// engine/runtime/token2wav_batch.py:335,356-357,518-519,549 -> engine/runtime/dit_fast.py:432-495).  These ops give
// that call site the B200 solve as registered torch operators (and the flow encoder before it, _flow_encode / _encoder,
// token2wav_batch.py:365-478): tensors in, the current torch CUDA stream of the
// tensors' device as the stream, a C-ABI call, and a RuntimeError carrying the status on failure.  No logic lives here:
// every op is argument conversion around one t2w_* call (include/t2w_b200.h).  Solver and slot-pool objects cross the
// boundary as int handles (their addresses), as the ctypes binding passes them.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <string>
#include <vector>

#include "t2w_b200.h"

namespace {

void check(const char* fn, int rc) {
  TORCH_CHECK(rc == T2W_OK, fn, " failed: status ", rc,
              rc == T2W_ERR_CUDA ? " (cudaError " + std::to_string(t2w_last_cuda_error()) + ")" : std::string());
}

void* stream_of(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "b200t2w ops take CUDA tensors");
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

std::vector<int32_t> i32(c10::IntArrayRef v) { return std::vector<int32_t>(v.begin(), v.end()); }

template <class T>
T* handle(int64_t h) {
  return reinterpret_cast<T*>(static_cast<intptr_t>(h));
}

const void* ptr(const std::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// ---- solver objects ------------------------------------------------------------------------------------------------

int64_t create(c10::IntArrayRef cfg_i, c10::ArrayRef<double> cfg_f, c10::ArrayRef<double> t_sched, at::TensorList weights,
               int64_t precision) {
  TORCH_CHECK(cfg_i.size() == 8 && cfg_f.size() == 7, "create: 8 integer and 7 float config fields");
  TORCH_CHECK(!weights.empty(), "create: no weights");
  t2w_config c{};
  c.mel = (int32_t)cfg_i[0];
  c.hidden = (int32_t)cfg_i[1];
  c.depth = (int32_t)cfg_i[2];
  c.heads = (int32_t)cfg_i[3];
  c.head_dim = (int32_t)cfg_i[4];
  c.ffn = (int32_t)cfg_i[5];
  c.steps = (int32_t)cfg_i[6];
  c.freq_dim = (int32_t)cfg_i[7];
  c.cfg_rate = (float)cfg_f[0];
  c.t_scale = (float)cfg_f[1];
  c.max_period = (float)cfg_f[2];
  c.eps_block = (float)cfg_f[3];
  c.eps_final = (float)cfg_f[4];
  c.eps_qk = (float)cfg_f[5];
  c.eps_conv = (float)cfg_f[6];
  std::vector<float> ts(t_sched.begin(), t_sched.end());
  std::vector<const float*> w;
  for (const at::Tensor& t : weights) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous(), "create: weights are contiguous fp32");
    w.push_back(t.data_ptr<float>());
  }
  t2w_solver* s = nullptr;
  check("t2w_create", t2w_create(&c, ts.empty() ? nullptr : ts.data(), w.data(), (int32_t)w.size(), (int32_t)precision,
                                 stream_of(weights[0]), &s));
  return static_cast<int64_t>(reinterpret_cast<intptr_t>(s));
}

void destroy(int64_t solver) { check("t2w_destroy", t2w_destroy(handle<t2w_solver>(solver))); }

int64_t workspace_bytes(int64_t solver, c10::IntArrayRef prompt_len, c10::IntArrayRef chunk_len) {
  TORCH_CHECK(prompt_len.size() == chunk_len.size(), "workspace_bytes: one prompt and chunk length per stream");
  const std::vector<int32_t> P = i32(prompt_len), T = i32(chunk_len);
  return (int64_t)t2w_workspace_bytes(handle<t2w_solver>(solver), (int32_t)P.size(), P.data(), T.data());
}

void solve_packed(int64_t solver, c10::IntArrayRef prompt_len, c10::IntArrayRef chunk_len, const at::Tensor& x0,
                  const at::Tensor& mu, const at::Tensor& cond, const at::Tensor& spk, at::Tensor& out,
                  at::Tensor& workspace, bool graph) {
  TORCH_CHECK(prompt_len.size() == chunk_len.size(), "solve_packed: one prompt and chunk length per stream");
  const std::vector<int32_t> P = i32(prompt_len), T = i32(chunk_len);
  t2w_batch b{};
  b.n_streams = (int32_t)P.size();
  b.prompt_len = P.data();
  b.chunk_len = T.data();
  b.x0 = x0.data_ptr<float>();
  b.mu = mu.data_ptr<float>();
  b.cond = cond.data_ptr<float>();
  b.spk = spk.data_ptr<float>();
  b.out = out.data_ptr<float>();
  check("t2w_solve_packed", t2w_solve_packed(handle<t2w_solver>(solver), &b, workspace.data_ptr(),
                                             (size_t)workspace.numel(), graph ? T2W_FLAG_GRAPH : 0u, stream_of(out)));
}

}  // namespace

namespace {

// ---- steady state: slot pools and the caches the library keeps ----------------------------------------------------

int64_t slots_create(int64_t solver, int64_t n_slots, int64_t n_rowslots) {
  t2w_slots* p = nullptr;
  check("t2w_slots_create", t2w_slots_create(handle<t2w_solver>(solver), (int32_t)n_slots, (int32_t)n_rowslots, &p));
  return static_cast<int64_t>(reinterpret_cast<intptr_t>(p));
}

void slots_destroy(int64_t slots) { check("t2w_slots_destroy", t2w_slots_destroy(handle<t2w_slots>(slots))); }

struct Cached {
  std::vector<int32_t> h, T;
  std::vector<uint8_t> keep;
  t2w_cached_batch b{};
};

Cached cached_batch(c10::IntArrayRef handles, c10::IntArrayRef chunk_len, c10::IntArrayRef keep, const at::Tensor& noise,
                    double temperature) {
  TORCH_CHECK(handles.size() == chunk_len.size() && handles.size() == keep.size(),
              "solve_cached: one handle, window length and keep flag per request");
  TORCH_CHECK(noise.dim() == 2 && noise.scalar_type() == at::kFloat && noise.is_contiguous(),
              "solve_cached: noise is contiguous fp32 [mel, frames]");
  Cached c;
  c.h = i32(handles);
  c.T = i32(chunk_len);
  c.keep.assign(keep.begin(), keep.end());
  c.b.n_streams = (int32_t)c.h.size();
  c.b.handle = c.h.data();
  c.b.chunk_len = c.T.data();
  c.b.keep = c.keep.data();
  c.b.noise = noise.data_ptr<float>();
  c.b.noise_frames = (int32_t)noise.size(1);
  c.b.temperature = (float)temperature;
  return c;
}

int64_t cached_workspace_bytes(int64_t solver, int64_t slots, c10::IntArrayRef handles, c10::IntArrayRef chunk_len,
                               c10::IntArrayRef keep, const at::Tensor& noise) {
  Cached c = cached_batch(handles, chunk_len, keep, noise, 1.0);
  return (int64_t)t2w_cached_workspace_bytes(handle<t2w_solver>(solver), handle<t2w_slots>(slots), &c.b);
}

void solve_cached(int64_t solver, int64_t slots, c10::IntArrayRef handles, c10::IntArrayRef chunk_len,
                  c10::IntArrayRef keep, const at::Tensor& noise, double temperature, const at::Tensor& mu,
                  const std::optional<at::Tensor>& cond, const at::Tensor& spk, at::Tensor& out, at::Tensor& workspace,
                  bool graph) {
  Cached c = cached_batch(handles, chunk_len, keep, noise, temperature);
  c.b.mu = mu.data_ptr<float>();
  c.b.cond = static_cast<const float*>(ptr(cond));
  c.b.spk = spk.data_ptr<float>();
  c.b.out = out.data_ptr<float>();
  check("t2w_solve_cached", t2w_solve_cached(handle<t2w_solver>(solver), handle<t2w_slots>(slots), &c.b,
                                             workspace.data_ptr(), (size_t)workspace.numel(),
                                             graph ? T2W_FLAG_GRAPH : 0u, stream_of(out)));
}

void solve_slots(int64_t solver, int64_t slots, c10::IntArrayRef chunk_len, c10::IntArrayRef kv_len,
                 c10::IntArrayRef kv_idx, c10::IntArrayRef cnn_rd, c10::IntArrayRef cnn_wr, const at::Tensor& x0,
                 const at::Tensor& mu, const std::optional<at::Tensor>& cond, const at::Tensor& spk, at::Tensor& out,
                 at::Tensor& workspace, bool graph) {
  const std::vector<int32_t> T = i32(chunk_len), kl = i32(kv_len), ki = i32(kv_idx), rd = i32(cnn_rd), wr = i32(cnn_wr);
  TORCH_CHECK(kl.size() == 2 * T.size() && rd.size() == kl.size() && wr.size() == kl.size(),
              "solve_slots: two key lists and conv rows (cond, uncond) per request");
  t2w_slot_batch b{};
  b.n_streams = (int32_t)T.size();
  b.chunk_len = T.data();
  b.kv_len = kl.data();
  b.kv_idx = ki.data();
  b.cnn_rd = rd.data();
  b.cnn_wr = wr.data();
  b.x0 = x0.data_ptr<float>();
  b.mu = mu.data_ptr<float>();
  b.cond = static_cast<const float*>(ptr(cond));
  b.spk = spk.data_ptr<float>();
  b.out = out.data_ptr<float>();
  const size_t need = t2w_slot_workspace_bytes(handle<t2w_solver>(solver), handle<t2w_slots>(slots), &b);
  TORCH_CHECK(need > 0, "solve_slots: invalid batch");
  TORCH_CHECK((size_t)workspace.numel() >= need, "solve_slots: workspace needs ", need, " bytes");
  check("t2w_solve_slots", t2w_solve_slots(handle<t2w_solver>(solver), handle<t2w_slots>(slots), &b,
                                           workspace.data_ptr(), (size_t)workspace.numel(),
                                           graph ? T2W_FLAG_GRAPH : 0u, stream_of(out)));
}

}  // namespace

namespace {

// ---- single kernels (the per-kernel entry points of the C ABI) -----------------------------------------------------

const uint8_t* pad_ptr(const std::optional<at::Tensor>& pad) { return static_cast<const uint8_t*>(ptr(pad)); }

void ln_mod(const at::Tensor& h, const at::Tensor& shift, const at::Tensor& scale1, double eps, at::Tensor& out,
            const std::optional<at::Tensor>& pad) {
  TORCH_CHECK(h.dim() == 2 && out.dim() == 2, "ln_mod: h [rows, C] fp32, out [rows, C] bf16");
  check("t2w_ln_mod", t2w_ln_mod(h.data_ptr<float>(), (int32_t)h.stride(0), shift.data_ptr<float>(),
                                 scale1.data_ptr<float>(), (float)eps, (int32_t)h.size(0), (int32_t)h.size(1),
                                 out.data_ptr(), (int32_t)out.stride(0), pad_ptr(pad), stream_of(h)));
}

void add_ln_mod(at::Tensor& h, const std::optional<at::Tensor>& y, const std::optional<at::Tensor>& g,
                const at::Tensor& shift, const at::Tensor& scale1, double eps, at::Tensor& out,
                const std::optional<at::Tensor>& pad) {
  TORCH_CHECK(h.dim() == 2, "add_ln_mod: h [rows, C] fp32");
  check("t2w_add_ln_mod", t2w_add_ln_mod(h.data_ptr<float>(), ptr(y), static_cast<const float*>(ptr(g)),
                                         shift.data_ptr<float>(), scale1.data_ptr<float>(), (float)eps,
                                         (int32_t)h.size(0), (int32_t)h.size(1), out.data_ptr(), pad_ptr(pad),
                                         stream_of(h)));
}

void ln_mish(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, double eps, at::Tensor& out,
             const std::optional<at::Tensor>& pad) {
  TORCH_CHECK(x.dim() == 2, "ln_mish: x [rows, C] bf16");
  check("t2w_ln_mish", t2w_ln_mish(x.data_ptr(), w.data_ptr<float>(), b.data_ptr<float>(), (float)eps,
                                   (int32_t)x.size(0), (int32_t)x.size(1), out.data_ptr(), pad_ptr(pad), stream_of(x)));
}

void gemm(const at::Tensor& A, const at::Tensor& W, const std::optional<at::Tensor>& bias, int64_t M, int64_t N, int64_t K,
          int64_t taps, int64_t tap_row0, int64_t epi, at::Tensor& out, int64_t ldo, at::TensorList qk, double qk_eps) {
  TORCH_CHECK(A.dim() == 2, "gemm: A [rows_a, lda] bf16");
  std::vector<const float*> q;
  for (const at::Tensor& t : qk) q.push_back(t.data_ptr<float>());
  check("t2w_gemm", t2w_gemm(A.data_ptr(), (int32_t)A.size(1), (int32_t)A.size(0), W.data_ptr(),
                             static_cast<const float*>(ptr(bias)), (int32_t)M, (int32_t)N, (int32_t)K, (int32_t)taps,
                             (int32_t)tap_row0, (int32_t)epi, out.data_ptr(), (int32_t)ldo, q.empty() ? nullptr : q.data(),
                             (float)qk_eps, stream_of(A)));
}

void attn_varlen(const at::Tensor& qkv, int64_t heads, c10::IntArrayRef seq_row, c10::IntArrayRef seq_len,
                 c10::IntArrayRef prompt_len, at::Tensor& out) {
  TORCH_CHECK(seq_row.size() == seq_len.size() && seq_len.size() == prompt_len.size(),
              "attn_varlen: one row, length and prompt length per sequence");
  const std::vector<int32_t> r = i32(seq_row), l = i32(seq_len), p = i32(prompt_len);
  check("t2w_attn_varlen", t2w_attn_varlen(qkv.data_ptr(), (int32_t)qkv.size(0), (int32_t)heads, (int32_t)r.size(),
                                           r.data(), l.data(), p.data(), out.data_ptr(), stream_of(qkv)));
}

void euler_cfg(at::Tensor& x, const at::Tensor& dphi, const at::Tensor& tok_row, int64_t half_rows, double dt, double w,
               const std::optional<at::Tensor>& hx, const std::optional<at::Tensor>& out) {
  TORCH_CHECK(x.dim() == 2 && dphi.dim() == 2 && tok_row.scalar_type() == at::kInt, "euler_cfg: x [n_tok, mel], "
              "dphi [rows, ld] fp32, tok_row int32 [n_tok]");
  check("t2w_euler_cfg", t2w_euler_cfg(x.data_ptr<float>(), dphi.data_ptr<float>(), (int32_t)dphi.size(1),
                                       tok_row.data_ptr<int32_t>(), (int32_t)x.size(0), (int32_t)x.size(1),
                                       (int32_t)half_rows, (float)dt, (float)w, const_cast<void*>(ptr(hx)),
                                       hx.has_value() ? (int32_t)hx->size(1) : 0,
                                       static_cast<float*>(const_cast<void*>(ptr(out))), stream_of(x)));
}

// ---- flow encoder ---------------------------------------------------------------------------------------------------

struct Enc {
  std::vector<int32_t> h, n, tok;
  std::vector<uint8_t> fin;
  t2w_enc_batch b{};
};

Enc enc_batch(c10::IntArrayRef handles, c10::IntArrayRef n_tokens, c10::IntArrayRef final_, c10::IntArrayRef tokens) {
  TORCH_CHECK(handles.size() == n_tokens.size() && handles.size() == final_.size(),
              "encode: one handle, token count and final flag per window");
  Enc e;
  e.h = i32(handles);
  e.n = i32(n_tokens);
  e.tok = i32(tokens);
  e.fin.assign(final_.begin(), final_.end());
  e.b.n_streams = (int32_t)e.h.size();
  e.b.handle = e.h.data();
  e.b.n_tokens = e.n.data();
  e.b.final = e.fin.data();
  e.b.tokens = e.tok.data();
  return e;
}

int64_t enc_workspace_bytes(int64_t encoder, c10::IntArrayRef handles, c10::IntArrayRef n_tokens,
                            c10::IntArrayRef final_, c10::IntArrayRef tokens) {
  Enc e = enc_batch(handles, n_tokens, final_, tokens);
  return (int64_t)t2w_enc_workspace_bytes(handle<t2w_encoder>(encoder), &e.b);
}

void encode(int64_t encoder, c10::IntArrayRef handles, c10::IntArrayRef n_tokens, c10::IntArrayRef final_,
            c10::IntArrayRef tokens, at::Tensor& mu, at::Tensor& workspace, bool graph) {
  TORCH_CHECK(mu.scalar_type() == at::kFloat && mu.is_contiguous(), "encode: mu is contiguous fp32");
  Enc e = enc_batch(handles, n_tokens, final_, tokens);
  e.b.mu = mu.data_ptr<float>();
  check("t2w_encode", t2w_encode(handle<t2w_encoder>(encoder), &e.b, workspace.data_ptr(), (size_t)workspace.numel(),
                                 graph ? T2W_FLAG_GRAPH : 0u, stream_of(mu)));
}

// ---- paged 8-bit K/V cache ------------------------------------------------------------------------------------------

const int32_t* i32_of(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like, int64_t n = -1) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == like.device() && (n < 0 || t.numel() == n),
              op, ": ", name, " is contiguous int32", n < 0 ? std::string() : " of " + std::to_string(n) + " entries",
              " on ", like.device().str());
  return t.data_ptr<int32_t>();
}

int32_t to_i32(const char* op, const char* name, int64_t v) {
  TORCH_CHECK(v >= 0 && v <= 0x7fffffff, op, ": ", name, " ", v, " does not fit 32 bits");
  return (int32_t)v;
}

// [requests, blocks] int32 whose rows may be strided (a view of a larger table)
void table_of(const char* op, const at::Tensor& t, const at::Tensor& like, int32_t& ld, int32_t& blocks) {
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt && t.device() == like.device() && (t.size(1) <= 1 || t.stride(1) == 1),
              op, ": table is int32 [requests, blocks] with contiguous rows on ", like.device().str());
  blocks = to_i32(op, "blocks", t.size(1));
  ld = t.size(0) > 1 ? to_i32(op, "the table's row stride", t.stride(0)) : blocks;
}

struct Pages {
  int32_t pages, heads, page, hd;
  void* codes[2];
  float* scale[2];
  int64_t page_ld[2], scale_ld[2];
};

Pages pages_of(const char* op, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs) {
  Pages p{};
  const at::Tensor* c[2] = {&kc, &vc};
  const at::Tensor* s[2] = {&ks, &vs};
  for (int w = 0; w < 2; ++w) {
    TORCH_CHECK(c[w]->is_cuda() && c[w]->dim() == 4 && c[w]->scalar_type() == at::kFloat8_e4m3fn && c[w]->sizes() == kc.sizes() &&
                    c[w]->device() == kc.device(),
                op, ": codes are float8_e4m3fn [pages, kv_heads, page, head_dim], K and V alike, on one GPU");
    const int64_t hd = c[w]->size(3), page = c[w]->size(2);
    TORCH_CHECK(c[w]->stride(3) == 1 && c[w]->stride(2) == hd && (c[w]->size(1) == 1 || c[w]->stride(1) == page * hd),
                op, ": a page's codes are contiguous [kv_heads, page, head_dim] (pages may lie at any pitch)");
    TORCH_CHECK(s[w]->dim() == 2 && s[w]->scalar_type() == at::kFloat && s[w]->size(0) == kc.size(0) && s[w]->size(1) == kc.size(1) &&
                    (s[w]->size(1) == 1 || s[w]->stride(1) == 1) && s[w]->device() == kc.device(),
                op, ": scales are fp32 [pages, kv_heads] with contiguous rows");
    p.codes[w] = c[w]->data_ptr();
    p.scale[w] = s[w]->data_ptr<float>();
    p.page_ld[w] = c[w]->size(0) > 1 ? c[w]->stride(0) : c[w]->size(1) * page * hd;
    p.scale_ld[w] = s[w]->size(0) > 1 ? s[w]->stride(0) : s[w]->size(1);
  }
  p.pages = to_i32(op, "pages", kc.size(0));
  p.heads = to_i32(op, "kv_heads", kc.size(1));
  p.page = to_i32(op, "page", kc.size(2));
  p.hd = to_i32(op, "head_dim", kc.size(3));
  return p;
}

int32_t dtype_of(const char* op, const at::Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": rows are bf16 or fp16");
  return t.scalar_type() == at::kHalf ? T2W_DT_FP16 : T2W_DT_BF16;
}

// [rows, heads, hd] with a contiguous last dimension
void rows_of(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like, int64_t rows, int64_t heads,
             int64_t hd, int64_t& row_ld, int64_t& head_ld) {
  TORCH_CHECK(t.dim() == 3 && t.size(0) == rows && t.size(1) == heads && t.size(2) == hd && t.stride(2) == 1 &&
                  t.device() == like.device(),
              op, ": ", name, " is [", rows, ", ", heads, ", ", hd, "] with contiguous head_dim on ", like.device().str());
  row_ld = rows > 1 ? t.stride(0) : heads * hd;
  head_ld = heads > 1 ? t.stride(1) : hd;
  TORCH_CHECK(row_ld >= 0 && head_ld >= 0 && row_ld % 8 == 0 && head_ld % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              op, ": ", name, " lies on 16-byte boundaries (strides a multiple of 8 elements)");
}

void plan_of(const char* op, const at::Tensor& plan, const at::Tensor& like, int32_t requests, int32_t rows, int32_t max_fresh,
             int32_t page, int32_t q_heads, int32_t kv_heads, int32_t hd) {
  const int64_t n = t2w_paged_plan_ints(requests, rows, max_fresh, page, q_heads, kv_heads, hd, nullptr);
  if (n < 0) check("t2w_paged_plan_ints", (int)n);
  i32_of(op, "a plan made for these sizes", plan, like, n);
}

std::vector<at::Tensor> paged_plan(const at::Tensor& fresh, const at::Tensor& length, at::Tensor& table, int64_t page, int64_t rows,
                      int64_t max_fresh, int64_t q_heads, int64_t kv_heads, int64_t head_dim, bool causal,
                      const std::optional<at::Tensor>& free_pages, const std::optional<at::Tensor>& free_count,
                      const std::optional<at::Tensor>& kv_len, const std::optional<at::Tensor>& free_left) {
  const char* op = "paged_plan";
  TORCH_CHECK(fresh.is_cuda(), "b200t2w ops take CUDA tensors");
  const c10::DeviceGuard guard(fresh.device());
  t2w_paged_plan_args a{};
  a.requests = to_i32(op, "requests", fresh.numel());
  a.rows = to_i32(op, "rows", rows);
  a.max_fresh = to_i32(op, "max_fresh", max_fresh);
  a.page = to_i32(op, "page", page);
  a.q_heads = to_i32(op, "q_heads", q_heads);
  a.kv_heads = to_i32(op, "kv_heads", kv_heads);
  a.head_dim = to_i32(op, "head_dim", head_dim);
  a.causal = causal;
  a.fresh = i32_of(op, "fresh", fresh, fresh);
  a.length = i32_of(op, "length", length, fresh, a.requests);
  table_of(op, table, fresh, a.table_ld, a.max_blocks);
  TORCH_CHECK(table.size(0) == a.requests, op, ": the table has a row for each request");
  a.table = table.data_ptr<int32_t>();
  TORCH_CHECK(free_pages.has_value() == free_count.has_value(), op, ": free_pages and free_count come together");
  a.pages = 1;
  if (free_pages) {
    a.free_pages = i32_of(op, "free_pages", *free_pages, fresh);
    a.free_count = i32_of(op, "free_count", *free_count, fresh, 1);
    a.pages = to_i32(op, "pages", free_pages->numel());
  }
  if (kv_len) a.kv_len = const_cast<int32_t*>(i32_of(op, "kv_len", *kv_len, fresh, a.requests));
  if (free_left) a.free_left = const_cast<int32_t*>(i32_of(op, "free_left", *free_left, fresh, 1));
  int64_t at[4];
  const int64_t n = t2w_paged_plan_ints(a.requests, a.rows, a.max_fresh, a.page, a.q_heads, a.kv_heads, a.head_dim, at);
  if (n < 0) check("t2w_paged_plan", (int)n);
  at::Tensor plan = at::empty({n}, fresh.options());
  a.plan = plan.data_ptr<int32_t>();
  check("t2w_paged_plan", t2w_paged_plan(&a, stream_of(fresh)));
  return {plan, plan.narrow(0, at[0], a.requests + 1), plan.narrow(0, at[1], a.requests), plan.narrow(0, at[2], a.rows),
          plan.narrow(0, at[3], a.rows), plan.narrow(0, 6, 1)};
}

void paged_append(const at::Tensor& k, const at::Tensor& v, at::Tensor& k_codes, at::Tensor& v_codes, at::Tensor& k_scale,
                  at::Tensor& v_scale, at::Tensor& plan, int64_t requests, int64_t max_fresh, int64_t q_heads) {
  const char* op = "paged_append";
  const Pages p = pages_of(op, k_codes, v_codes, k_scale, v_scale);
  const c10::DeviceGuard guard(k_codes.device());
  t2w_paged_append_args a{};
  a.requests = to_i32(op, "requests", requests);
  a.rows = to_i32(op, "rows", k.size(0));
  a.max_fresh = to_i32(op, "max_fresh", max_fresh);
  a.page = p.page;
  a.q_heads = to_i32(op, "q_heads", q_heads);
  a.kv_heads = p.heads;
  a.head_dim = p.hd;
  a.pages = p.pages;
  a.dtype = dtype_of(op, k);
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), op, ": k and v have one type");
  rows_of(op, "k", k, k_codes, a.rows, p.heads, p.hd, a.k_row_ld, a.k_head_ld);
  rows_of(op, "v", v, k_codes, a.rows, p.heads, p.hd, a.v_row_ld, a.v_head_ld);
  plan_of(op, plan, k_codes, a.requests, a.rows, a.max_fresh, a.page, a.q_heads, a.kv_heads, a.head_dim);
  if (a.rows == 0) return;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_codes = p.codes[0];
  a.v_codes = p.codes[1];
  a.k_scale = p.scale[0];
  a.v_scale = p.scale[1];
  a.k_page_ld = p.page_ld[0];
  a.v_page_ld = p.page_ld[1];
  a.k_scale_ld = p.scale_ld[0];
  a.v_scale_ld = p.scale_ld[1];
  a.plan = plan.data_ptr<int32_t>();
  check("t2w_paged_append", t2w_paged_append(&a, stream_of(k_codes)));
}

std::vector<at::Tensor> paged_attn(const at::Tensor& q, const at::Tensor& k_codes, const at::Tensor& v_codes,
                                   const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& table,
                                   at::Tensor& plan, int64_t requests, int64_t max_fresh, bool causal, double scale, bool lse) {
  const char* op = "paged_attn";
  const Pages p = pages_of(op, k_codes, v_codes, k_scale, v_scale);
  const c10::DeviceGuard guard(k_codes.device());
  TORCH_CHECK(q.dim() == 3, op, ": q is [rows, q_heads, head_dim]");
  t2w_paged_attn_args a{};
  a.requests = to_i32(op, "requests", requests);
  a.rows = to_i32(op, "rows", q.size(0));
  a.max_fresh = to_i32(op, "max_fresh", max_fresh);
  a.page = p.page;
  a.q_heads = to_i32(op, "q_heads", q.size(1));
  a.kv_heads = p.heads;
  a.head_dim = p.hd;
  a.causal = causal;
  a.pages = p.pages;
  a.dtype = dtype_of(op, q);
  a.scale = (float)scale;
  rows_of(op, "q", q, k_codes, a.rows, a.q_heads, p.hd, a.q_row_ld, a.q_head_ld);
  plan_of(op, plan, k_codes, a.requests, a.rows, a.max_fresh, a.page, a.q_heads, a.kv_heads, a.head_dim);
  int32_t blocks = 0;
  table_of(op, table, k_codes, a.table_ld, blocks);
  TORCH_CHECK(table.size(0) == a.requests, op, ": the table has a row for each request");
  at::Tensor out = at::empty({a.rows, a.q_heads, a.head_dim}, q.options());
  std::vector<at::Tensor> r{out};
  if (lse) r.push_back(at::empty({a.rows, a.q_heads}, q.options().dtype(at::kFloat)));
  if (a.rows == 0) return r;
  const size_t ws = t2w_paged_workspace_bytes(a.max_fresh, a.q_heads, a.kv_heads, a.head_dim);
  at::Tensor workspace = at::empty({(int64_t)ws}, q.options().dtype(at::kByte));
  a.q = q.data_ptr();
  a.k_codes = p.codes[0];
  a.v_codes = p.codes[1];
  a.k_scale = p.scale[0];
  a.v_scale = p.scale[1];
  a.k_page_ld = p.page_ld[0];
  a.v_page_ld = p.page_ld[1];
  a.k_scale_ld = p.scale_ld[0];
  a.v_scale_ld = p.scale_ld[1];
  a.table = table.data_ptr<int32_t>();
  a.plan = plan.data_ptr<int32_t>();
  a.out = out.data_ptr();
  a.lse = lse ? r[1].data_ptr<float>() : nullptr;
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = ws;
  check("t2w_paged_attn", t2w_paged_attn(&a, stream_of(k_codes)));
  return r;
}

void paged_release(const at::Tensor& done, at::Tensor& length, at::Tensor& table, int64_t page, at::Tensor& free_pages,
                   at::Tensor& free_count, at::Tensor& status) {
  const char* op = "paged_release";
  TORCH_CHECK(done.is_cuda(), "b200t2w ops take CUDA tensors");
  const c10::DeviceGuard guard(done.device());
  const int32_t n = to_i32(op, "requests", done.numel());
  int32_t ld = 0, blocks = 0;
  table_of(op, table, done, ld, blocks);
  TORCH_CHECK(table.size(0) == n, op, ": the table has a row for each request");
  check("t2w_paged_release",
        t2w_paged_release(i32_of(op, "done", done, done), const_cast<int32_t*>(i32_of(op, "length", length, done, n)),
                          table.data_ptr<int32_t>(), n, to_i32(op, "page", page), ld, blocks,
                          to_i32(op, "pages", free_pages.numel()), const_cast<int32_t*>(i32_of(op, "free_pages", free_pages, done)),
                          const_cast<int32_t*>(i32_of(op, "free_count", free_count, done, 1)),
                          const_cast<int32_t*>(i32_of(op, "status", status, done, 1)), stream_of(done)));
}

int64_t paged_status(const at::Tensor& plan) {
  const c10::DeviceGuard guard(plan.device());
  TORCH_CHECK(plan.numel() >= 8, "paged_status: a plan");
  return t2w_paged_status(i32_of("paged_status", "plan", plan, plan), stream_of(plan));
}

// ---- products with 4-bit weights --------------------------------------------------------------------------------------
// A weight crosses as its buffer (uint8, t2w_w4_bytes), its sizes and its kind: 1 zeros, 2 gated, 4 fp16 scales.

t2w_w4_weight weight_of(const char* op, const at::Tensor& buffer, int64_t n, int64_t k, int64_t group, int64_t kind) {
  TORCH_CHECK(buffer.is_cuda() && buffer.scalar_type() == at::kByte && buffer.dim() == 1 && buffer.is_contiguous(),
              op, ": a weight's buffer is contiguous uint8 on the GPU");
  t2w_w4_weight w{};
  w.n = to_i32(op, "n", n);
  w.k = to_i32(op, "k", k);
  w.group = to_i32(op, "group", group);
  w.zeros = (kind & 1) != 0;
  w.gated = (kind & 2) != 0;
  w.scale_dtype = kind & 4 ? T2W_DT_FP16 : T2W_DT_BF16;
  const int64_t bytes = t2w_w4_bytes(w.n, w.k, w.group, w.zeros, w.gated);
  if (bytes < 0) check("t2w_w4_bytes", (int)bytes);
  TORCH_CHECK(buffer.numel() == bytes, op, ": a weight of these sizes has ", bytes, " bytes, not ", buffer.numel());
  w.buffer = buffer.data_ptr();
  return w;
}

t2w_w4_source source_of(const char* op, const t2w_w4_weight& w, const at::Tensor& buffer, const at::Tensor& codes,
                        const at::Tensor& scales, const std::optional<at::Tensor>& zeros) {
  const int64_t groups = w.k / w.group;
  auto fits = [&](const at::Tensor& t, at::ScalarType type, int64_t cols) {
    return t.dim() == 2 && t.scalar_type() == type && t.size(0) == w.n && t.size(1) == cols &&
           (cols == 1 || t.stride(1) == 1) && t.stride(0) >= 0 && t.device() == buffer.device();
  };
  TORCH_CHECK(fits(codes, at::kByte, w.k), op, ": codes are uint8 [n, k] with contiguous rows on ", buffer.device().str());
  TORCH_CHECK(fits(scales, w.scale_dtype == T2W_DT_FP16 ? at::kHalf : at::kBFloat16, groups), op,
              ": scales are bf16 or fp16 [n, k / group] with contiguous rows on ", buffer.device().str());
  TORCH_CHECK(zeros.has_value() == (w.zeros != 0), op, ": zeros come where the weight has them");
  t2w_w4_source s{};
  s.codes = codes.data_ptr();
  s.scales = scales.data_ptr();
  s.code_ld = codes.stride(0);
  s.scale_ld = scales.stride(0);
  if (zeros) {
    TORCH_CHECK(fits(*zeros, at::kByte, groups), op, ": zeros are uint8 [n, k / group] with contiguous rows on ",
                buffer.device().str());
    s.zeros = zeros->data_ptr();
    s.zero_ld = zeros->stride(0);
  }
  return s;
}

void w4_pack(at::Tensor& buffer, int64_t n, int64_t k, int64_t group, int64_t kind, const at::Tensor& codes,
             const at::Tensor& scales, const std::optional<at::Tensor>& zeros, const std::optional<at::Tensor>& up_codes,
             const std::optional<at::Tensor>& up_scales, const std::optional<at::Tensor>& up_zeros) {
  const char* op = "w4_pack";
  const t2w_w4_weight w = weight_of(op, buffer, n, k, group, kind);
  const c10::DeviceGuard guard(buffer.device());
  TORCH_CHECK((w.gated != 0) == up_codes.has_value() && up_codes.has_value() == up_scales.has_value(), op,
              ": a gated weight has the up projection's codes and scales too");
  const t2w_w4_source a = source_of(op, w, buffer, codes, scales, zeros);
  t2w_w4_source b{};
  if (w.gated) b = source_of(op, w, buffer, *up_codes, *up_scales, up_zeros);
  check("t2w_w4_pack", t2w_w4_pack(&w, &a, w.gated ? &b : nullptr, stream_of(buffer)));
}

std::vector<at::Tensor> w4_unpack(const at::Tensor& buffer, int64_t n, int64_t k, int64_t group, int64_t kind) {
  const t2w_w4_weight w = weight_of("w4_unpack", buffer, n, k, group, kind);
  const c10::DeviceGuard guard(buffer.device());
  std::vector<at::Tensor> r;
  for (int i = 0; i < (w.gated ? 2 : 1); ++i) r.push_back(at::empty({n, k}, buffer.options().dtype(at::kFloat)));
  check("t2w_w4_unpack", t2w_w4_unpack(&w, r[0].data_ptr<float>(), k, w.gated ? r[1].data_ptr<float>() : nullptr, k,
                                       stream_of(buffer)));
  return r;
}

int64_t w4_status(at::Tensor& buffer, int64_t n, int64_t k, int64_t group, int64_t kind) {
  const t2w_w4_weight w = weight_of("w4_status", buffer, n, k, group, kind);
  const c10::DeviceGuard guard(buffer.device());
  return t2w_w4_status(&w, stream_of(buffer));
}

at::Tensor w4_product(const char* op, const at::Tensor& x, const at::Tensor& buffer, const t2w_w4_weight& w, int64_t act,
                      const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& residual) {
  const c10::DeviceGuard guard(buffer.device());
  t2w_w4_linear_args a{};
  a.w = w;
  a.dtype = dtype_of(op, x);
  a.act = (int32_t)act;
  TORCH_CHECK(x.dim() == 2 && x.size(1) == w.k && x.stride(1) == 1 && x.device() == buffer.device(), op, ": x is [rows, ", w.k,
              "] with contiguous rows on ", buffer.device().str());
  for (const at::Tensor* t : {&x, bias ? &*bias : nullptr, residual ? &*residual : nullptr})
    TORCH_CHECK(!t || !t->requires_grad() || !at::GradMode::is_enabled(), op, ": has no gradient");
  a.rows = to_i32(op, "rows", x.size(0));
  a.x_ld = a.rows > 1 ? x.stride(0) : w.k;
  TORCH_CHECK(a.x_ld >= w.k && a.x_ld % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0, op,
              ": x lies on 16-byte boundaries (a pitch of a multiple of 8 elements, at least k)");
  a.x = x.data_ptr();
  if (bias) {
    TORCH_CHECK(bias->dim() == 1 && bias->numel() == w.n && (w.n == 1 || bias->stride(0) == 1) &&
                    bias->scalar_type() == x.scalar_type() && bias->device() == x.device(),
                op, ": bias is contiguous [", w.n, "] of x's type and device");
    a.bias = bias->data_ptr();
  }
  if (residual) {
    TORCH_CHECK(residual->dim() == 2 && residual->size(0) == a.rows && residual->size(1) == w.n &&
                    (w.n == 1 || residual->stride(1) == 1) && (a.rows <= 1 || residual->stride(0) >= w.n) &&
                    residual->scalar_type() == x.scalar_type() && residual->device() == x.device(),
                op, ": residual is [", a.rows, ", ", w.n, "] with contiguous rows of x's type and device");
    a.residual = residual->data_ptr();
    a.res_ld = a.rows > 1 ? residual->stride(0) : w.n;
  }
  at::Tensor out = at::empty({a.rows, w.n}, x.options());
  if (a.rows == 0) return out;
  a.out = out.data_ptr();
  check("t2w_w4_linear", t2w_w4_linear(&a, stream_of(buffer)));
  return out;
}

at::Tensor w4_linear(const at::Tensor& x, const at::Tensor& buffer, int64_t n, int64_t k, int64_t group, int64_t kind,
                     const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& residual) {
  const t2w_w4_weight w = weight_of("w4_linear", buffer, n, k, group, kind);
  TORCH_CHECK(!w.gated, "w4_linear: the weight is a gated pair");
  return w4_product("w4_linear", x, buffer, w, T2W_ACT_SILU, bias, residual);
}

at::Tensor w4_gated(const at::Tensor& x, const at::Tensor& buffer, int64_t n, int64_t k, int64_t group, int64_t kind,
                    int64_t act) {
  const t2w_w4_weight w = weight_of("w4_gated", buffer, n, k, group, kind);
  TORCH_CHECK(w.gated, "w4_gated: the weight is not a gated pair");
  return w4_product("w4_gated", x, buffer, w, act, std::nullopt, std::nullopt);
}

// ---- rotary positions -------------------------------------------------------------------------------------------------

std::vector<at::Tensor> rotate(const char* op, const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions,
                               const at::Tensor& table, int64_t rotary_dim, int64_t axes, bool adjacent, bool inverse,
                               bool in_place) {
  TORCH_CHECK(q.is_cuda(), "b200t2w ops take CUDA tensors");
  const c10::DeviceGuard guard(q.device());
  TORCH_CHECK(q.dim() == 3, op, ": q is [rows, heads, head_dim]");
  t2w_rotary_args a{};
  a.rows = to_i32(op, "rows", q.size(0));
  a.head_dim = to_i32(op, "head_dim", q.size(2));
  a.rotary_dim = to_i32(op, "rotary_dim", rotary_dim);
  a.axes = to_i32(op, "axes", axes);
  a.adjacent = adjacent;
  a.inverse = inverse;
  a.dtype = dtype_of(op, q);
  TORCH_CHECK(table.scalar_type() == at::kLong && table.dim() == 1 && table.is_contiguous() && table.numel() == rotary_dim &&
                  table.device() == q.device(),
              op, ": the table is int64 [rotary_dim] on ", q.device().str());
  a.table = table.data_ptr();
  const bool wide = positions.scalar_type() == at::kLong;
  TORCH_CHECK(wide || positions.scalar_type() == at::kInt, op, ": positions are int32 or int64");
  const bool flat = positions.dim() == 1 && axes == 1;
  TORCH_CHECK((flat || (positions.dim() == 2 && positions.size(0) == axes)) && positions.size(flat ? 0 : 1) == a.rows &&
                  (a.rows <= 1 || positions.stride(flat ? 0 : 1) == 1) && positions.device() == q.device(),
              op, ": positions are [", axes, ", ", a.rows, "] with contiguous rows on ", q.device().str());
  a.wide_positions = wide;
  a.pos_ld = flat || axes == 1 ? a.rows : positions.stride(0);
  TORCH_CHECK(a.pos_ld == 0 || a.pos_ld >= a.rows, op, ": the axes of positions are apart, or one for all");
  a.positions = positions.data_ptr();
  std::vector<at::Tensor> r;
  auto fill = [&](const char* name, const at::Tensor& x, int32_t& heads, t2w_rotary_rows& rows) {
    TORCH_CHECK(x.dim() == 3 && x.scalar_type() == q.scalar_type(), op, ": q and k are [rows, heads, head_dim] of one type");
    TORCH_CHECK(!x.requires_grad() || !at::GradMode::is_enabled(), op, ": no gradient is recorded (`inverse` is the gradient)");
    heads = to_i32(op, "heads", x.size(1));
    if (heads == 0 || a.rows == 0) {
      TORCH_CHECK(x.size(0) == a.rows && x.size(2) == a.head_dim, op, ": q and k have the same rows and head_dim");
      r.push_back(in_place ? x : at::empty_like(x));
      return;
    }
    rows_of(op, name, x, q, a.rows, heads, a.head_dim, rows.in_row_ld, rows.in_head_ld);
    r.push_back(in_place ? x : at::empty({a.rows, heads, a.head_dim}, x.options()));
    rows.in = x.data_ptr();
    rows.out = r.back().data_ptr();
    rows.out_row_ld = in_place ? rows.in_row_ld : (int64_t)heads * a.head_dim;
    rows.out_head_ld = in_place ? rows.in_head_ld : a.head_dim;
  };
  fill("q", q, a.q_heads, a.q);
  if (k) fill("k", *k, a.k_heads, a.k);
  if (in_place && k && a.rows && a.q_heads && a.k_heads)
    TORCH_CHECK(q.data_ptr() != k->data_ptr(), op, ": q and k are one tensor");
  check("t2w_rotary", t2w_rotary(&a, stream_of(q)));
  return r;
}

std::vector<at::Tensor> rotary(const at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions,
                               const at::Tensor& table, int64_t rotary_dim, int64_t axes, bool adjacent, bool inverse) {
  return rotate("rotary", q, k, positions, table, rotary_dim, axes, adjacent, inverse, false);
}
void rotary_(at::Tensor& q, const std::optional<at::Tensor>& k, const at::Tensor& positions, const at::Tensor& table,
             int64_t rotary_dim, int64_t axes, bool adjacent, bool inverse) {
  rotate("rotary_", q, k, positions, table, rotary_dim, axes, adjacent, inverse, true);
}

}  // namespace

TORCH_LIBRARY(b200t2w, m) {
  m.def("create(int[] cfg_i, float[] cfg_f, float[] t_sched, Tensor[] weights, int precision) -> int", &create);
  m.def("destroy(int solver) -> ()", &destroy);
  m.def("workspace_bytes(int solver, int[] prompt_len, int[] chunk_len) -> int", &workspace_bytes);
  m.def("solve_packed(int solver, int[] prompt_len, int[] chunk_len, Tensor x0, Tensor mu, Tensor cond, Tensor spk, "
        "Tensor(a!) out, Tensor(b!) workspace, bool graph) -> ()",
        &solve_packed);
  m.def("slots_create(int solver, int n_slots, int n_rowslots) -> int", &slots_create);
  m.def("slots_destroy(int slots) -> ()", &slots_destroy);
  m.def("cached_workspace_bytes(int solver, int slots, int[] handles, int[] chunk_len, int[] keep, Tensor noise) -> int",
        &cached_workspace_bytes);
  m.def("solve_cached(int solver, int slots, int[] handles, int[] chunk_len, int[] keep, Tensor noise, "
        "float temperature, Tensor mu, Tensor? cond, Tensor spk, Tensor(a!) out, Tensor(b!) workspace, bool graph) -> ()",
        &solve_cached);
  m.def("solve_slots(int solver, int slots, int[] chunk_len, int[] kv_len, int[] kv_idx, int[] cnn_rd, int[] cnn_wr, "
        "Tensor x0, Tensor mu, Tensor? cond, Tensor spk, Tensor(a!) out, Tensor(b!) workspace, bool graph) -> ()",
        &solve_slots);
  m.def("ln_mod(Tensor h, Tensor shift, Tensor scale1, float eps, Tensor(a!) out, Tensor? pad) -> ()", &ln_mod);
  m.def("add_ln_mod(Tensor(a!) h, Tensor? y, Tensor? g, Tensor shift, Tensor scale1, float eps, Tensor(b!) out, "
        "Tensor? pad) -> ()",
        &add_ln_mod);
  m.def("ln_mish(Tensor x, Tensor w, Tensor b, float eps, Tensor(a!) out, Tensor? pad) -> ()", &ln_mish);
  m.def("gemm(Tensor A, Tensor W, Tensor? bias, int M, int N, int K, int taps, int tap_row0, int epi, Tensor(a!) out, "
        "int ldo, Tensor[] qk, float qk_eps) -> ()",
        &gemm);
  m.def("attn_varlen(Tensor qkv, int heads, int[] seq_row, int[] seq_len, int[] prompt_len, Tensor(a!) out) -> ()",
        &attn_varlen);
  m.def("euler_cfg(Tensor(a!) x, Tensor dphi, Tensor tok_row, int half_rows, float dt, float w, Tensor(b!)? hx, "
        "Tensor(c!)? out) -> ()",
        &euler_cfg);
  m.def("enc_workspace_bytes(int encoder, int[] handles, int[] n_tokens, int[] final, int[] tokens) -> int",
        &enc_workspace_bytes);
  m.def("encode(int encoder, int[] handles, int[] n_tokens, int[] final, int[] tokens, Tensor(a!) mu, "
        "Tensor(b!) workspace, bool graph) -> ()",
        &encode);
  m.def("paged_plan(Tensor fresh, Tensor length, Tensor(a!) table, int page, int rows, int max_fresh, int q_heads, "
        "int kv_heads, int head_dim, bool causal, Tensor? free_pages, Tensor? free_count, Tensor? kv_len, "
        "Tensor? free_left) -> Tensor[]",
        &paged_plan);
  m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k_codes, Tensor(b!) v_codes, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor(e!) plan, int requests, int max_fresh, int q_heads) -> ()",
        &paged_append);
  m.def("paged_attn(Tensor q, Tensor k_codes, Tensor v_codes, Tensor k_scale, Tensor v_scale, Tensor table, "
        "Tensor(a!) plan, int requests, int max_fresh, bool causal, float scale, bool lse) -> Tensor[]",
        &paged_attn);
  m.def("paged_release(Tensor done, Tensor(a!) length, Tensor(b!) table, int page, Tensor(c!) free_pages, "
        "Tensor(d!) free_count, Tensor(e!) status) -> ()",
        &paged_release);
  m.def("paged_status(Tensor plan) -> int", &paged_status);
  m.def("w4_pack(Tensor(a!) buffer, int n, int k, int group, int kind, Tensor codes, Tensor scales, Tensor? zeros, "
        "Tensor? up_codes, Tensor? up_scales, Tensor? up_zeros) -> ()",
        &w4_pack);
  m.def("w4_unpack(Tensor buffer, int n, int k, int group, int kind) -> Tensor[]", &w4_unpack);
  m.def("w4_status(Tensor(a!) buffer, int n, int k, int group, int kind) -> int", &w4_status);
  m.def("w4_linear(Tensor x, Tensor buffer, int n, int k, int group, int kind, Tensor? bias, Tensor? residual) -> Tensor",
        &w4_linear);
  m.def("w4_gated(Tensor x, Tensor buffer, int n, int k, int group, int kind, int act) -> Tensor", &w4_gated);
  m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor table, int rotary_dim, int axes, bool adjacent, bool inverse) "
        "-> Tensor[]",
        &rotary);
  m.def("rotary_(Tensor(a!) q, Tensor(b!)? k, Tensor positions, Tensor table, int rotary_dim, int axes, bool adjacent, "
        "bool inverse) -> ()",
        &rotary_);
}
