// fluxvla_b200._C: the thin torch C++ extension over the C ABI
// (include/fluxvla_b200.h) for the operator-level entry points that callers
// reach once per op outside a CUDA graph (the reference's atomic_ops /
// Triton call sites): tensors in, the C entry point on the current torch
// CUDA stream, arguments checked on entry (a Python ValueError for a bad
// argument, RuntimeError for an error the library reports), as the
// reference's own pybind extension checks its inputs
// (fluxvla/ops/cuda/matmul_bias/src/matmul_bias_forward.cpp:21-60).
// Nothing here allocates; every output is caller-allocated.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstring>
#include <sstream>
#include <stdexcept>
#include <string>

#include "../../include/fluxvla_b200.h"

namespace {

using OptT = c10::optional<at::Tensor>;

void* stream_ptr() {
  return reinterpret_cast<void*>(at::cuda::getCurrentCUDAStream().stream());
}

// Argument check: std::invalid_argument, which pybind11 raises as
// ValueError.  (Plain C++ exceptions rather than TORCH_CHECK: a c10::Error
// thrown from this module crashed the process on the error path.)
template <typename... Ts>
void require(bool ok, const Ts&... parts) {
  if (ok) return;
  std::ostringstream os;
  (os << ... << parts);
  throw std::invalid_argument(os.str());
}

void check(int rc, const char* what) {
  if (rc == FVB_OK) return;
  std::string msg = std::string("fluxvla_b200 ") + what + " error " + std::to_string(rc) +
                    ": " + fvb_last_error();
  throw std::runtime_error(msg);
}

template <typename T = void>
T* ptr(const OptT& t) {
  return t.has_value() && t->defined() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

int64_t rowmajor(const at::Tensor& t, at::ScalarType dt, const char* name) {
  require(t.scalar_type() == dt, name, ": expected ", dt, ", got ", t.scalar_type());
  require(t.is_cuda(), name, ": must be a CUDA tensor");
  require(t.dim() == 2 && t.stride(1) == 1, name, ": expected a 2-D row-major view");
  return t.stride(0);
}

void check_vec_f32(const OptT& t, const char* name) {
  if (!t.has_value() || !t->defined()) return;
  require(t->scalar_type() == at::kFloat && t->is_contiguous() && t->is_cuda(), name,
              ": expected a contiguous float32 CUDA tensor");
}

// C[M,N] = A[M,K] @ B[N,K]^T with the fused epilogue of fvb_gemm.
void gemm(const at::Tensor& a, const at::Tensor& b, const at::Tensor& out,
          int64_t epilogue, bool swap, int64_t act, const OptT& bias, const OptT& gate,
          double alpha, int64_t split_k, int64_t block_n, const OptT& row_add,
          int64_t row_add_mod, const OptT& k_out, const OptT& v_out, int64_t n_heads,
          int64_t head_dim, const OptT& rope_cs, const OptT& positions,
          const OptT& workspace, bool pair, const OptT& res, const OptT& gate_tok,
          bool rope_interleaved, int64_t norm_mode, const OptT& norm_out,
          const OptT& norm_w, const OptT& norm_b, double norm_eps,
          const OptT& norm_sync) {
  fvb_gemm_args g;
  memset(&g, 0, sizeof(g));
  g.lda = rowmajor(a, at::kBFloat16, "a");
  g.ldb = rowmajor(b, at::kBFloat16, "b");
  require(a.size(1) == b.size(1), "K mismatch ", a.sizes(), " ", b.sizes());
  const bool f32 = epilogue == FVB_EPI_F32_STORE || epilogue == FVB_EPI_F32_ACC;
  g.ldo = rowmajor(out, f32 ? at::kFloat : at::kBFloat16, "out");
  check_vec_f32(bias, "bias");
  check_vec_f32(gate, "gate");
  g.a = a.data_ptr(); g.b = b.data_ptr();
  g.m = (int32_t)a.size(0); g.n = (int32_t)b.size(0); g.k = (int32_t)a.size(1);
  g.swap = swap; g.epilogue = (int32_t)epilogue; g.act = (int32_t)act;
  g.split_k = (int32_t)split_k; g.block_n = (int32_t)block_n;
  g.out = out.data_ptr();
  g.bias = ptr<const float>(bias); g.gate = ptr<const float>(gate);
  g.alpha = (float)alpha;
  g.row_add = ptr(row_add); g.row_add_mod = (int32_t)row_add_mod;
  g.k_out = ptr(k_out); g.v_out = ptr(v_out);
  g.ld_kv = k_out.has_value() ? k_out->stride(0) : 0;
  g.n_heads = (int32_t)n_heads; g.head_dim = (int32_t)head_dim;
  g.rope_cs = ptr<const float>(rope_cs); g.positions = ptr<const int32_t>(positions);
  g.workspace = ptr(workspace);
  g.workspace_bytes = workspace.has_value() ? workspace->numel() * workspace->element_size() : 0;
  g.pair = pair;
  g.res = ptr(res);
  g.ld_res = res.has_value() ? rowmajor(*res, at::kBFloat16, "res") : 0;
  g.gate_tok = ptr(gate_tok);
  g.ld_gate_tok = gate_tok.has_value() ? rowmajor(*gate_tok, at::kBFloat16, "gate_tok") : 0;
  g.rope_interleaved = rope_interleaved;
  if (norm_out.has_value()) {
    g.norm_mode = (int32_t)norm_mode;
    g.norm_out = norm_out->data_ptr();
    g.ld_norm_out = rowmajor(*norm_out, at::kBFloat16, "norm_out");
    g.norm_w = ptr(norm_w); g.norm_b = ptr(norm_b);
    g.norm_eps = (float)norm_eps;
    g.norm_sync = ptr(norm_sync);
  }
  check(fvb_gemm(&g, stream_ptr()), "fvb_gemm");
}

// Row norms of f32 rows (fvb_norm), output bf16 or f32.
void norm(int64_t mode, const at::Tensor& x, const at::Tensor& out, const OptT& w,
          const OptT& b, const OptT& mod, double eps) {
  const int64_t ld_in = rowmajor(x, at::kFloat, "x");
  const bool out_f32 = out.scalar_type() == at::kFloat;
  const int64_t ld_out = rowmajor(out, out_f32 ? at::kFloat : at::kBFloat16, "out");
  check(fvb_norm((int32_t)mode, x.data_ptr<float>(), ld_in, out.data_ptr(), ld_out,
                 out_f32, (int32_t)x.size(0), (int32_t)x.size(1), ptr(w), ptr(b),
                 ptr<const float>(mod), (float)eps, stream_ptr()),
        "fvb_norm");
}

// Row norms of bf16 rows (fvb_norm_bf16).
void norm_bf16(int64_t mode, const at::Tensor& x, const at::Tensor& out, const OptT& w,
               const OptT& b, const OptT& style, const OptT& gate_out, double eps) {
  const int64_t ld_in = rowmajor(x, at::kBFloat16, "x");
  const int64_t ld_out = rowmajor(out, at::kBFloat16, "out");
  const int64_t ld_gate = gate_out.has_value() ? rowmajor(*gate_out, at::kBFloat16, "gate_out") : 0;
  check(fvb_norm_bf16((int32_t)mode, x.data_ptr(), ld_in, out.data_ptr(), ld_out,
                      (int32_t)x.size(0), (int32_t)x.size(1), ptr(w), ptr(b), ptr(style),
                      ptr(gate_out), ld_gate, (float)eps, stream_ptr()),
        "fvb_norm_bf16");
}

// bf16 softmax over the attended keys of f32 logits rows (fvb_softmax_rows).
void softmax_rows(const at::Tensor& logits, const at::Tensor& out, int64_t n_prefix,
                  const at::Tensor& valid_prefix) {
  require(valid_prefix.scalar_type() == at::kInt && valid_prefix.is_cuda(),
              "valid_prefix: expected an int32 CUDA tensor");
  const int64_t ld_in = rowmajor(logits, at::kFloat, "logits");
  const int64_t ld_out = rowmajor(out, at::kBFloat16, "out");
  check(fvb_softmax_rows(logits.data_ptr<float>(), ld_in, (int32_t)logits.size(0),
                         (int32_t)logits.size(1), (int32_t)n_prefix,
                         valid_prefix.data_ptr<int32_t>(), out.data_ptr(), ld_out,
                         stream_ptr()),
        "fvb_softmax_rows");
}

// y = act(x @ w[:, :k]^T + bias), f32 x, bf16 w (fvb_small_linear).
void small_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& out,
                  const OptT& bias, int64_t act, int64_t mode, double alpha, int64_t k) {
  const int64_t ldx = rowmajor(x, at::kFloat, "x");
  const int64_t ldw = rowmajor(w, at::kBFloat16, "w");
  const int64_t ldo = rowmajor(out, mode == 1 ? at::kBFloat16 : at::kFloat, "out");
  check_vec_f32(bias, "bias");
  check(fvb_small_linear(x.data_ptr<float>(), ldx, (int32_t)x.size(0),
                         (int32_t)(k > 0 ? k : x.size(1)), w.data_ptr(), ldw,
                         (int32_t)w.size(0), ptr<const float>(bias), (int32_t)act,
                         (int32_t)mode, (float)alpha, out.data_ptr(), ldo, stream_ptr()),
        "fvb_small_linear");
}

// ---- operators that serve several requests at once.  Their tensors may lie on
// any device: the call runs on that device and its current stream.

int64_t strided(const at::Tensor& t, at::ScalarType dt, int64_t dims, const char* name) {
  require(t.scalar_type() == dt, name, ": expected ", dt, ", got ", t.scalar_type());
  require(t.is_cuda(), name, ": must be a CUDA tensor");
  require(t.dim() == dims && (t.stride(dims - 1) == 1 || t.size(dims - 1) <= 1), name,
          ": expected ", dims, " dimensions, the last one contiguous");
  return dims == 2 && t.size(0) <= 1 ? std::max(t.stride(0), t.size(1)) : t.stride(0);
}

// stride of a dimension; one of size 1 has none that matters
int64_t step(const at::Tensor& t, int64_t dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

void same_device(const at::Tensor& a, const at::Tensor& b, const char* name) {
  require(a.device() == b.device(), name, ": on ", b.device(), ", expected ", a.device());
}

int32_t i32(int64_t v, const char* name) {
  require(v >= 0 && v <= INT32_MAX, name, ": ", v, " is out of range");
  return (int32_t)v;
}

bool f32_or_bf16(const at::Tensor& t, const char* name) {
  require(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name,
          ": expected float32 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat;
}

void norm_fp8(int64_t mode, const at::Tensor& x, const at::Tensor& q, const at::Tensor& scales,
              const OptT& delta, const OptT& res, const OptT& w, const OptT& mod, double eps) {
  fvb_norm_fp8_args a;
  memset(&a, 0, sizeof(a));
  a.mode = (int32_t)mode;
  a.x_f32 = f32_or_bf16(x, "x");
  a.ld_x = strided(x, x.scalar_type(), 2, "x");
  a.rows = i32(x.size(0), "rows");
  a.dim = i32(x.size(1), "dim");
  a.ld_q = strided(q, at::kFloat8_e4m3fn, 2, "out");
  a.ld_scales = strided(scales, at::kFloat, 2, "scales");
  require(q.sizes() == x.sizes(), "out: expected ", x.sizes(), ", got ", q.sizes());
  require(scales.size(0) == a.rows && scales.size(1) == (a.dim + 127) / 128,
          "scales: expected [", a.rows, ", ", (a.dim + 127) / 128, "], got ", scales.sizes());
  same_device(x, q, "out");
  same_device(x, scales, "scales");
  require(delta.has_value() == res.has_value(), "delta and res come together");
  if (delta.has_value()) {
    a.delta_f32 = f32_or_bf16(*delta, "delta");
    a.ld_delta = strided(*delta, delta->scalar_type(), 2, "delta");
    a.ld_res = strided(*res, x.scalar_type(), 2, "res");
    require(delta->sizes() == x.sizes() && res->sizes() == x.sizes(),
            "delta and res: expected ", x.sizes(), ", got ", delta->sizes(), " and ",
            res->sizes());
    same_device(x, *delta, "delta");
    same_device(x, *res, "res");
    a.delta = delta->data_ptr();
    a.res = res->data_ptr();
  }
  if (w.has_value()) {
    require(w->scalar_type() == at::kBFloat16 && w->is_contiguous() && w->numel() == a.dim,
            "w: expected ", a.dim, " contiguous bfloat16 values");
    same_device(x, *w, "w");
    a.w = w->data_ptr();
  }
  if (mod.has_value()) {
    require(mod->scalar_type() == at::kFloat && mod->is_contiguous() && mod->numel() == 2 * a.dim,
            "mod: expected ", 2 * (int64_t)a.dim, " contiguous float32 values");
    same_device(x, *mod, "mod");
    a.mod = mod->data_ptr<float>();
  }
  a.x = x.data_ptr();
  a.q = q.data_ptr();
  a.scales = scales.data_ptr<float>();
  a.eps = eps;
  if (a.rows == 0) return;
  c10::cuda::CUDAGuard guard(x.device());
  check(fvb_norm_fp8(&a, stream_ptr()), "fvb_norm_fp8");
}

void gemm_fp8(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b,
              const at::Tensor& b_scale, const at::Tensor& out, int64_t epilogue) {
  fvb_gemm_fp8_args g;
  memset(&g, 0, sizeof(g));
  g.lda = strided(a, at::kFloat8_e4m3fn, 2, "a");
  g.ldb = strided(b, at::kFloat8_e4m3fn, 2, "b");
  g.m = i32(a.size(0), "m");
  g.n = i32(b.size(0), "n");
  g.k = i32(a.size(1), "k");
  require(b.size(1) == g.k, "K mismatch ", a.sizes(), " ", b.sizes());
  const int64_t groups = (g.k + 127) / 128;
  g.ld_as = strided(a_scale, at::kFloat, 2, "a_scale");
  g.ld_bs = strided(b_scale, at::kFloat, 2, "b_scale");
  require(a_scale.size(0) == g.m && a_scale.size(1) == groups, "a_scale: expected [", g.m, ", ",
          groups, "], got ", a_scale.sizes());
  require(b_scale.size(0) == (g.n + 127) / 128 && b_scale.size(1) == groups,
          "b_scale: expected [", (g.n + 127) / 128, ", ", groups, "], got ", b_scale.sizes());
  const bool f32 = epilogue == FVB_EPI_F32_STORE;
  g.ldo = strided(out, f32 ? at::kFloat : at::kBFloat16, 2, "out");
  const int64_t nf = epilogue == FVB_EPI_GEGLU ? g.n / 2 : g.n;
  require(out.size(0) == g.m && out.size(1) == nf, "out: expected [", g.m, ", ", nf, "], got ",
          out.sizes());
  same_device(a, a_scale, "a_scale");
  same_device(a, b, "b");
  same_device(a, b_scale, "b_scale");
  same_device(a, out, "out");
  // a single row has no stride of its own to be aligned
  if (g.m == 1) g.lda = (g.lda + 15) / 16 * 16;
  if (g.n == 1) g.ldb = (g.ldb + 15) / 16 * 16;
  g.a = a.data_ptr();
  g.a_scale = a_scale.data_ptr<float>();
  g.b = b.data_ptr();
  g.b_scale = b_scale.data_ptr<float>();
  g.out = out.data_ptr();
  g.epilogue = (int32_t)epilogue;
  if (g.m == 0) return;
  c10::cuda::CUDAGuard guard(a.device());
  check(fvb_gemm_fp8(&g, stream_ptr()), "fvb_gemm_fp8");
}

// a cache [pages, page_size, kv_heads, dim] and its strides
void cache_strides(const at::Tensor& c, const char* name, int64_t* page, int64_t* row,
                   int64_t* head) {
  strided(c, at::kBFloat16, 4, name);
  *page = step(c, 0);
  *row = step(c, 1);
  *head = step(c, 2);
}

int32_t* int_vector(const at::Tensor& t, int64_t n, const char* name) {
  require(t.scalar_type() == at::kInt && t.is_cuda() && t.is_contiguous() && t.numel() == n, name,
          ": expected ", n, " contiguous int32 values on the GPU");
  return t.data_ptr<int32_t>();
}

void paged_append(const OptT& q, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& slots, const at::Tensor& k_cache, const at::Tensor& v_cache,
                  const OptT& q_out, const OptT& positions, const OptT& rope_cs,
                  bool rope_interleaved) {
  fvb_paged_append_args a;
  memset(&a, 0, sizeof(a));
  strided(k, at::kBFloat16, 3, "k");
  strided(v, at::kBFloat16, 3, "v");
  a.k_row_stride = step(k, 0);
  a.v_row_stride = step(v, 0);
  a.k_head_stride = step(k, 1);
  a.v_head_stride = step(v, 1);
  a.tokens = i32(k.size(0), "tokens");
  a.kv_heads = i32(k.size(1), "kv_heads");
  a.head_dim = i32(k.size(2), "head_dim");
  require(v.sizes() == k.sizes(), "v: expected ", k.sizes(), ", got ", v.sizes());
  cache_strides(k_cache, "k_cache", &a.kc_page_stride, &a.kc_row_stride, &a.kc_head_stride);
  cache_strides(v_cache, "v_cache", &a.vc_page_stride, &a.vc_row_stride, &a.vc_head_stride);
  require(k_cache.size(2) == a.kv_heads && k_cache.size(3) == a.head_dim &&
              v_cache.sizes() == k_cache.sizes(),
          "caches: expected [pages, page_size, ", a.kv_heads, ", ", a.head_dim, "], got ",
          k_cache.sizes(), " and ", v_cache.sizes());
  a.n_pages = i32(k_cache.size(0), "pages");
  a.page_size = i32(k_cache.size(1), "page_size");
  a.slots = int_vector(slots, a.tokens, "slots");
  for (const at::Tensor* t : {&v, &slots, &k_cache, &v_cache}) same_device(k, *t, "operand");
  require(q.has_value() == q_out.has_value(), "q and q_out come together");
  if (q.has_value()) {
    strided(*q, at::kBFloat16, 3, "q");
    strided(*q_out, at::kBFloat16, 3, "q_out");
    a.q_row_stride = step(*q, 0);
    a.q_out_row_stride = step(*q_out, 0);
    a.q_head_stride = step(*q, 1);
    a.q_out_head_stride = step(*q_out, 1);
    a.heads = i32(q->size(1), "heads");
    require(q->size(0) == a.tokens && q->size(2) == a.head_dim && q_out->sizes() == q->sizes(),
            "q and q_out: expected [", a.tokens, ", heads, ", a.head_dim, "], got ", q->sizes(),
            " and ", q_out->sizes());
    same_device(k, *q, "q");
    same_device(k, *q_out, "q_out");
    a.q = q->data_ptr();
    a.q_out = q_out->data_ptr();
  }
  require(positions.has_value() == rope_cs.has_value(), "positions and rope_cs come together");
  if (rope_cs.has_value()) {
    require(rope_cs->scalar_type() == at::kFloat && rope_cs->is_contiguous() &&
                rope_cs->dim() == 3 && rope_cs->size(0) > 0 &&
                rope_cs->size(1) * 2 == a.head_dim && rope_cs->size(2) == 2,
            "rope_cs: expected contiguous float32 [positions, head_dim / 2, 2]");
    same_device(k, *rope_cs, "rope_cs");
    same_device(k, *positions, "positions");
    a.rope_cs = rope_cs->data_ptr<float>();
    a.max_pos = i32(rope_cs->size(0), "positions");
    a.positions = int_vector(*positions, a.tokens, "positions");
  }
  a.rope_interleaved = rope_interleaved;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  if (a.tokens == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  check(fvb_paged_append(&a, stream_ptr()), "fvb_paged_append");
}

void paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& page_table, const at::Tensor& seq_lens,
                     const at::Tensor& out, double scale, const OptT& lse,
                     const at::Tensor& workspace) {
  fvb_paged_attn_args a;
  memset(&a, 0, sizeof(a));
  strided(q, at::kBFloat16, 3, "q");
  strided(out, at::kBFloat16, 3, "out");
  a.q_row_stride = step(q, 0);
  a.out_row_stride = step(out, 0);
  a.q_head_stride = step(q, 1);
  a.out_head_stride = step(out, 1);
  require(out.sizes() == q.sizes(), "out: expected ", q.sizes(), ", got ", out.sizes());
  a.batch = i32(q.size(0), "batch");
  a.heads = i32(q.size(1), "heads");
  a.head_dim = i32(q.size(2), "head_dim");
  cache_strides(k_cache, "k_cache", &a.kc_page_stride, &a.kc_row_stride, &a.kc_head_stride);
  cache_strides(v_cache, "v_cache", &a.vc_page_stride, &a.vc_row_stride, &a.vc_head_stride);
  require(k_cache.size(3) == a.head_dim && v_cache.sizes() == k_cache.sizes(),
          "caches: expected [pages, page_size, kv_heads, ", a.head_dim, "], got ",
          k_cache.sizes(), " and ", v_cache.sizes());
  a.n_pages = i32(k_cache.size(0), "pages");
  a.page_size = i32(k_cache.size(1), "page_size");
  a.kv_heads = i32(k_cache.size(2), "kv_heads");
  a.ld_table = strided(page_table, at::kInt, 2, "page_table");
  require(page_table.size(0) == a.batch, "page_table: expected ", a.batch, " rows, got ",
          page_table.sizes());
  a.max_pages = i32(page_table.size(1), "page_table columns");
  a.seq_lens = int_vector(seq_lens, a.batch, "seq_lens");
  require(workspace.is_cuda() && workspace.is_contiguous(),
          "workspace: expected a contiguous CUDA tensor");
  for (const at::Tensor* t : {&k_cache, &v_cache, &page_table, &seq_lens, &out, &workspace})
    same_device(q, *t, "operand");
  if (lse.has_value()) {
    a.lse_row_stride = strided(*lse, at::kFloat, 2, "lse");
    require(lse->size(0) == a.batch && lse->size(1) == a.heads, "lse: expected [", a.batch, ", ",
            a.heads, "], got ", lse->sizes());
    same_device(q, *lse, "lse");
    a.lse = lse->data_ptr<float>();
  }
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.page_table = page_table.data_ptr<int32_t>();
  a.out = out.data_ptr();
  a.scale = (float)scale;
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = workspace.numel() * workspace.element_size();
  if (a.batch == 0) return;
  c10::cuda::CUDAGuard guard(q.device());
  check(fvb_paged_attention(&a, stream_ptr()), "fvb_paged_attention");
}

// A C-ABI error surfaced as a Python exception without touching the GPU
// (fvb_get_device_status rejects a NULL pointer): used by the tests.
void error_path_probe() { check(fvb_get_device_status(nullptr, 0), "fvb_get_device_status"); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "fluxvla_b200 torch extension over the C ABI (include/fluxvla_b200.h)";
  m.def("gemm", &gemm);
  m.def("norm", &norm);
  m.def("norm_bf16", &norm_bf16);
  m.def("softmax_rows", &softmax_rows);
  m.def("small_linear", &small_linear);
  m.def("norm_fp8", &norm_fp8);
  m.def("gemm_fp8", &gemm_fp8);
  m.def("paged_append", &paged_append);
  m.def("paged_attention", &paged_attention);
  m.def("error_path_probe", &error_path_probe);
}
