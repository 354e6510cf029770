// Thin torch binding over the C ABI for the calls whose per-call host cost matters (a few rows through a Linear
// layer take less device time than Python + ctypes need to issue them).  It checks the tensors, allocates the
// output and the activation scratch from torch's allocator, takes torch's current stream and calls libmxq; nothing
// here computes.  mase_b200.gemm uses it when it is built and otherwise issues the same C calls through ctypes.

#include <algorithm>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "mxq.h"

namespace {

int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return MXQ_F32;
  if (t == at::kBFloat16) return MXQ_BF16;
  TORCH_CHECK_NOT_IMPLEMENTED(false, "mase_b200: dtype ", t, " is not supported (float32 and bfloat16 are)");
}

void check_rc(int rc, const char *what) {
  TORCH_CHECK(rc == MXQ_OK, what, " failed: ", mxq_error_string(rc), " (code ", rc, ")");
}

// LinearMXFP.forward on packed weights: quantize x along K into scratch, block-scaled GEMM, one C call.
at::Tensor mx_linear(const at::Tensor &x, const at::Tensor &w_codes, const at::Tensor &w_scales, int64_t w_format,
                     int64_t n_out, const c10::optional<at::Tensor> &bias, int64_t exp_bits, int64_t frac_bits,
                     c10::optional<at::ScalarType> out_dtype, int64_t floor_tab_ptr, const at::Tensor &status,
                     int64_t options_ptr) {
  TORCH_CHECK(x.is_cuda(), "mx_linear: tensor is on '", x.device(), "'; mase_b200 runs on CUDA devices only");
  const int64_t K = x.size(-1);
  at::Tensor a = x.reshape({-1, K});
  if (!a.is_contiguous()) a = a.contiguous();
  if (reinterpret_cast<uintptr_t>(a.data_ptr()) % 16) a = a.clone();
  const int64_t M = a.size(0);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t ws_bytes = mxq_mx_linear_workspace_bytes(M, K);
  TORCH_CHECK(ws_bytes >= 0, "mx_linear: bad shape");
  at::Tensor ws = at::empty({ws_bytes}, x.options().dtype(at::kByte));
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  at::Tensor out = at::empty({M, n_out}, x.options().dtype(odt));
  const void *bias_ptr = nullptr;
  int bias_dt = 0;
  at::Tensor b;
  if (bias.has_value() && bias->defined()) {
    b = bias->contiguous();
    bias_ptr = b.data_ptr();
    bias_dt = dtype_code(b.scalar_type());
  }
  const int rc = mxq_mx_linear(a.data_ptr(), dtype_code(a.scalar_type()), static_cast<const uint8_t *>(w_codes.data_ptr()),
                               static_cast<const uint8_t *>(w_scales.data_ptr()), (int)w_format, out.data_ptr(), bias_ptr,
                               dtype_code(odt), bias_dt, M, n_out, K, (int)exp_bits, (int)frac_bits,
                               reinterpret_cast<const uint8_t *>(floor_tab_ptr), ws.data_ptr(), ws_bytes,
                               static_cast<int *>(status.data_ptr()),
                               reinterpret_cast<const mxq_gemm_options *>(options_ptr),
                               at::cuda::getCurrentCUDAStream(x.device().index()).stream());
  check_rc(rc, "mxq_mx_linear");
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(n_out);
  return out.reshape(shape);
}

// F.linear on operands that already hold quantized values (bf16 exactly, fp32 as tf32).
at::Tensor dense_linear(const at::Tensor &x, const at::Tensor &weight, const c10::optional<at::Tensor> &bias,
                        c10::optional<at::ScalarType> out_dtype, const at::Tensor &status, int64_t options_ptr) {
  TORCH_CHECK(x.is_cuda(), "linear_forward: tensor is on '", x.device(), "'; mase_b200 runs on CUDA devices only");
  TORCH_CHECK(x.scalar_type() == weight.scalar_type(), "expected input and weight to have the same dtype");
  const int64_t K = x.size(-1), N = weight.size(0);
  TORCH_CHECK(weight.size(1) == K, "mat1 and mat2 shapes cannot be multiplied");
  TORCH_CHECK(K % (x.scalar_type() == at::kBFloat16 ? 8 : 4) == 0, "dense_linear: rows must be 16-byte multiples");
  at::Tensor a = x.reshape({-1, K});
  if (!a.is_contiguous()) a = a.contiguous();
  if (reinterpret_cast<uintptr_t>(a.data_ptr()) % 16) a = a.clone();
  at::Tensor w = weight.is_contiguous() ? weight : weight.contiguous();
  const int64_t M = a.size(0);
  const c10::cuda::CUDAGuard guard(x.device());
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  at::Tensor out = at::empty({M, N}, x.options().dtype(odt));
  const void *bias_ptr = nullptr;
  int bias_dt = 0;
  at::Tensor b;
  if (bias.has_value() && bias->defined()) {
    b = bias->contiguous();
    bias_ptr = b.data_ptr();
    bias_dt = dtype_code(b.scalar_type());
  }
  const int rc = mxq_gemm_dense(a.data_ptr(), w.data_ptr(), out.data_ptr(), bias_ptr, dtype_code(a.scalar_type()),
                                dtype_code(odt), bias_dt, M, N, K, static_cast<int *>(status.data_ptr()),
                                reinterpret_cast<const mxq_gemm_options *>(options_ptr),
                                at::cuda::getCurrentCUDAStream(x.device().index()).stream());
  check_rc(rc, "mxq_gemm_dense");
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(N);
  return out.reshape(shape);
}

// MXFP / MXINT quantize-dequantize of a tensor that already is a run of blocks (contiguous, blocks along the last
// dimension).  kind 0: MXFP (p0 = E, p1 = F, floor table); kind 1: MXINT (p0 = bits, ceil table of x's dtype).
at::Tensor mx_fake(const at::Tensor &x, int64_t kind, int64_t block, int64_t p0, int64_t p1,
                   c10::optional<at::ScalarType> out_dtype, int64_t tab_ptr) {
  TORCH_CHECK(x.is_cuda(), "mx_fake: tensor is on '", x.device(), "'; mase_b200 runs on CUDA devices only");
  TORCH_CHECK(x.is_contiguous() && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0, "mx_fake: contiguous, aligned input");
  const int64_t n = x.numel();
  TORCH_CHECK(block > 0 && n % block == 0, "Input tensor size ", n, " is not divisible by block size ", block, ".");
  const c10::cuda::CUDAGuard guard(x.device());
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  at::Tensor y = at::empty(x.sizes(), x.options().dtype(odt));
  void *stream = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
  const uint8_t *tab = reinterpret_cast<const uint8_t *>(tab_ptr);
  int rc;
  if (kind == 0)
    rc = mxq_mxfp_fake(x.data_ptr(), y.data_ptr(), dtype_code(x.scalar_type()), dtype_code(odt), n / block, (int)block,
                       (int)p0, (int)p1, tab, stream);
  else
    rc = mxq_mxint_fake(x.data_ptr(), y.data_ptr(), dtype_code(x.scalar_type()), dtype_code(odt), n / block, (int)block,
                        (int)p0, tab, stream);
  check_rc(rc, kind == 0 ? "mxq_mxfp_fake" : "mxq_mxint_fake");
  return y;
}

// ---- paged key/value cache -------------------------------------------------------------------------------------------
// The calls of mase_b200.kv_cache for arguments that need no copy and no complaint: everything else returns None (or
// false) and is left to the Python functions, which check in detail, copy what must be copied and raise.

bool on(const at::Tensor &t, int64_t device) { return t.is_cuda() && t.device().index() == device; }
bool float_type(const at::Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }

// a gradient or a tangent that the calls would drop
bool differentiated(const at::Tensor &t) {
  return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

bool plain_table(const at::Tensor &table, const at::Tensor &lengths, int64_t device) {
  return on(table, device) && on(lengths, device) && table.scalar_type() == at::kInt && lengths.scalar_type() == at::kInt &&
         table.dim() == 2 && lengths.dim() == 1 && table.size(0) == lengths.size(0) && table.size(0) > 0 &&
         table.size(1) > 0 && table.stride(1) == 1 && (table.size(0) == 1 || table.stride(0) >= table.size(1)) &&
         lengths.is_contiguous();
}
bool plain_vector(const c10::optional<at::Tensor> &t, int64_t n, int64_t device) {
  return !t.has_value() ||
         (on(*t, device) && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous());
}
bool plain_stats(const at::Tensor &t, at::ScalarType type, int64_t batch, int64_t heads, int64_t device) {
  return on(t, device) && t.scalar_type() == type && t.dim() == 3 && t.size(0) == batch && t.size(1) == heads &&
         t.size(2) > 0 && t.is_contiguous() && !differentiated(t);
}
void *ptr(const c10::optional<at::Tensor> &t) { return t.has_value() ? t->data_ptr() : nullptr; }

c10::optional<at::Tensor> paged_attention(int64_t cache, int64_t device, const at::Tensor &query, const at::Tensor &table,
                                          const at::Tensor &lengths, double scaling, const c10::optional<at::Tensor> &weights,
                                          const at::Tensor &status) {
  const auto *c = reinterpret_cast<const mxq_paged_cache *>(cache);
  const int64_t nd = query.dim();
  if (!on(query, device) || !float_type(query) || differentiated(query) ||
      !plain_table(table, lengths, device) || (nd != 3 && nd != 4) || (nd == 4 && query.size(2) != 1) ||
      query.size(0) != table.size(0) || query.size(nd - 1) != c->head_dim || query.stride(nd - 1) != 1 ||
      query.size(1) < 1 || query.size(1) % c->heads != 0)
    return c10::nullopt;
  const int64_t batch = query.size(0), heads = query.size(1);
  int64_t width = table.size(1);
  if (weights.has_value()) {
    if (!plain_stats(*weights, at::kFloat, batch, c->heads, device)) return c10::nullopt;
    width = std::min(width, (weights->size(2) + c->page_size - 1) / c->page_size);  // no scores behind the statistics
  }
  const c10::cuda::CUDAGuard guard(query.device());
  const int64_t n_ws = mxq_paged_attention_workspace_bytes(c, batch, heads, width, weights.has_value());
  if (n_ws < 0) return c10::nullopt;
  at::Tensor out = at::empty(query.sizes(), query.options());
  at::Tensor ws = at::empty({n_ws}, query.options().dtype(at::kByte));
  const int rc = mxq_paged_attention(
      c, query.data_ptr(), out.data_ptr(), dtype_code(query.scalar_type()), batch, heads, query.stride(0), query.stride(1),
      (float)scaling, static_cast<const int32_t *>(table.data_ptr()), width, table.stride(0),
      static_cast<const int32_t *>(lengths.data_ptr()), static_cast<float *>(ptr(weights)),
      weights.has_value() ? weights->size(2) : 0, ws.data_ptr(), n_ws, static_cast<int *>(status.data_ptr()),
      at::cuda::getCurrentCUDAStream(device).stream());
  check_rc(rc, "mxq_paged_attention");
  return out;
}

// every row on a 16-byte boundary, the last dimension contiguous
bool plain_rows(const at::Tensor &t) {
  const int64_t need = 16 / t.element_size();
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int d = 0; d < 3; ++d)
    if (t.size(d) > 1 && t.stride(d) % need) return false;
  return true;
}
int64_t step(const at::Tensor &t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

bool paged_append(int64_t cache, int64_t device, const at::Tensor &key, const at::Tensor &value, const at::Tensor &table,
                  const at::Tensor &lengths, const c10::optional<at::Tensor> &counts,
                  const c10::optional<at::Tensor> &positions, const c10::optional<at::Tensor> &next_position, int64_t tab,
                  const at::Tensor &status) {
  const auto *c = reinterpret_cast<const mxq_paged_cache *>(cache);
  if (!on(key, device) || !on(value, device) || !float_type(key) || value.scalar_type() != key.scalar_type() ||
      differentiated(key) || differentiated(value) ||
      !plain_table(table, lengths, device) || key.dim() != 4 || key.sizes() != value.sizes() ||
      key.size(0) != table.size(0) || key.size(1) != c->heads || key.size(3) != c->head_dim || key.numel() == 0 ||
      !plain_rows(key) || !plain_rows(value))
    return false;
  const int64_t batch = key.size(0);
  if (!plain_vector(counts, batch, device) || !plain_vector(next_position, batch, device) ||
      (positions.has_value() ? !plain_stats(*positions, at::kInt, batch, c->heads, device) : next_position.has_value()))
    return false;
  const c10::cuda::CUDAGuard guard(key.device());
  const int rc = mxq_paged_append(
      c, key.data_ptr(), value.data_ptr(), dtype_code(key.scalar_type()), batch, key.size(2), step(key, 0), step(key, 1),
      step(key, 2), step(value, 0), step(value, 1), step(value, 2), static_cast<const int32_t *>(table.data_ptr()),
      table.size(1), table.stride(0), static_cast<const int32_t *>(lengths.data_ptr()),
      static_cast<const int32_t *>(ptr(counts)), static_cast<int32_t *>(ptr(positions)),
      positions.has_value() ? positions->size(2) : 0, static_cast<const int32_t *>(ptr(next_position)),
      reinterpret_cast<const uint8_t *>(tab), static_cast<int *>(status.data_ptr()),
      at::cuda::getCurrentCUDAStream(device).stream());
  check_rc(rc, "mxq_paged_append");
  return true;
}

c10::optional<std::tuple<at::Tensor, at::Tensor>> paged_gather(int64_t cache, int64_t device, const at::Tensor &table,
                                                               const at::Tensor &lengths, int64_t max_length,
                                                               at::ScalarType dtype, const at::Tensor &status) {
  const auto *c = reinterpret_cast<const mxq_paged_cache *>(cache);
  if (!plain_table(table, lengths, device) || max_length < 1 || (dtype != at::kFloat && dtype != at::kBFloat16))
    return c10::nullopt;
  const c10::cuda::CUDAGuard guard(table.device());
  const int64_t batch = table.size(0);
  at::Tensor key = at::empty({batch, c->heads, max_length, c->head_dim}, table.options().dtype(dtype));
  at::Tensor value = at::empty_like(key);
  const int rc = mxq_paged_gather(c, key.data_ptr(), value.data_ptr(), dtype_code(dtype), batch, max_length,
                                  static_cast<const int32_t *>(table.data_ptr()), table.size(1), table.stride(0),
                                  static_cast<const int32_t *>(lengths.data_ptr()), static_cast<int *>(status.data_ptr()),
                                  at::cuda::getCurrentCUDAStream(device).stream());
  check_rc(rc, "mxq_paged_gather");
  return std::make_tuple(key, value);
}

c10::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor>> paged_evict(
    int64_t cache, int64_t device, const at::Tensor &table, const at::Tensor &lengths, const at::Tensor &weights,
    int64_t keep, int64_t recent, const c10::optional<at::Tensor> &positions,
    const c10::optional<at::Tensor> &next_position, const at::Tensor &status) {
  const auto *c = reinterpret_cast<const mxq_paged_cache *>(cache);
  if (!plain_table(table, lengths, device)) return c10::nullopt;
  const int64_t batch = table.size(0);
  if (!plain_stats(weights, at::kFloat, batch, c->heads, device) || keep < 1 || keep > INT32_MAX || recent < 0 ||
      recent > keep || positions.has_value() != next_position.has_value() || !plain_vector(next_position, batch, device) ||
      (positions.has_value() && (!plain_stats(*positions, at::kInt, batch, c->heads, device) ||
                                 positions->size(2) != weights.size(2))))
    return c10::nullopt;
  const c10::cuda::CUDAGuard guard(weights.device());
  const int64_t width = weights.size(2);
  const int64_t n_ws = mxq_paged_evict_workspace_bytes(c, batch, width, keep);
  if (n_ws < 0) return c10::nullopt;
  at::Tensor new_lengths = at::empty_like(lengths), new_weights = at::empty_like(weights);
  at::Tensor new_positions = at::empty(weights.sizes(), lengths.options());
  at::Tensor ws = at::empty({n_ws}, weights.options().dtype(at::kByte));
  const int rc = mxq_paged_evict(
      c, batch, static_cast<const int32_t *>(table.data_ptr()), table.size(1), table.stride(0),
      static_cast<const int32_t *>(lengths.data_ptr()), static_cast<const float *>(weights.data_ptr()),
      static_cast<const int32_t *>(ptr(positions)), static_cast<const int32_t *>(ptr(next_position)), width, keep, recent,
      static_cast<int32_t *>(new_lengths.data_ptr()), static_cast<float *>(new_weights.data_ptr()),
      static_cast<int32_t *>(new_positions.data_ptr()), ws.data_ptr(), n_ws, static_cast<int *>(status.data_ptr()),
      at::cuda::getCurrentCUDAStream(device).stream());
  check_rc(rc, "mxq_paged_evict");
  return std::make_tuple(new_lengths, new_weights, new_positions);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("paged_attention", &paged_attention, "attention of one new token per sequence over a paged cache");
  m.def("paged_append", &paged_append, "quantize new keys and values into a paged cache");
  m.def("paged_gather", &paged_gather, "the rows of a paged cache as dense tensors");
  m.def("paged_evict", &paged_evict, "eviction from a paged cache by accumulated attention weight");
  m.def("mx_fake", &mx_fake, "MXFP / MXINT quantize-dequantize of a contiguous run of blocks");
  m.def("mx_linear", &mx_linear, "LinearMXFP forward on packed weights (mxq_mx_linear)");
  m.def("dense_linear", &dense_linear, "F.linear of quantized bf16 / fp32 operands (mxq_gemm_dense)");
}
