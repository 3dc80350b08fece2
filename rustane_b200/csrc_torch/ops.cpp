// The torch side of rustane_b200.ops: checks of the tensors, outputs, the current stream, then one
// call of librustane_cuda.so's C ABI.  In C++ because a call's host time is what a small one costs:
// the same through Python and ctypes took 12 to 20 us, against 8 to 10 us on the GPU.
//
// Handles (rope tables, cache, workspace) are rustane_b200.ops objects; they pass the address of
// their C struct and the index of their device.  A wrong tensor raises ValueError, a status of the
// library RustaneError.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>
#include <tuple>

#include "rustane_cuda.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;
constexpr auto kBf16 = at::kBFloat16;
constexpr auto kF32 = at::kFloat;
constexpr auto kI32 = at::kInt;

c10::Device device_of(int64_t index) { return c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index)); }

// A [rows, cols] matrix with contiguous rows; its row stride, which torch leaves arbitrary where
// there are fewer than two rows.
int64_t rows(const char* name, const Tensor& t, int64_t cols, at::ScalarType type, c10::Device dev, int64_t n = -1) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == type && t.size(1) == cols && (n < 0 || t.size(0) == n), name,
                    ": expected a [", n < 0 ? std::string("T") : std::to_string(n), ", ", cols, "] ", type, " tensor, got ",
                    t.sizes(), " ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == dev && (t.size(0) == 0 || t.stride(1) == 1), name,
                    ": its rows have to be contiguous and on ", dev);
  return t.size(0) > 1 ? t.stride(0) : cols;
}
void vec(const char* name, const Tensor& t, int64_t n, at::ScalarType type, c10::Device dev) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.scalar_type() == type && (n < 0 || t.size(0) == n), name, ": expected ",
                    n < 0 ? std::string("a vector") : std::to_string(n), " of ", type, ", got ", t.sizes(), " ",
                    t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == dev && t.is_contiguous(), name, ": has to be contiguous and on ", dev);
}
template <class T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <class T>
T* ptr(const Opt& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
c10::Device cuda(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "a CUDA tensor is needed");
  return t.device();
}
// The device's error word, where one is given.
int* error_word(const Opt& t, c10::Device dev) {
  if (t)
    TORCH_CHECK_VALUE(t->scalar_type() == kI32 && t->numel() > 0 && t->device() == dev, "err: has to be an int32 tensor on ",
                      dev, ", got ", t->sizes(), " ", t->scalar_type(), " on ", t->device());
  return ptr<int>(t);
}
void* stream(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
void done(int rc, const char* name) {
  if (rc == RT_OK) return;
  const py::object cls = py::module_::import("rustane_b200._lib").attr("RustaneError");
  const py::object err = cls(rc, name);
  PyErr_SetObject(cls.ptr(), err.ptr());
  throw py::error_already_set();
}
Tensor like(const Tensor& t) { return at::empty_like(t, {}, at::MemoryFormat::Contiguous); }

void gammas(const Opt& q, const Opt& k, int64_t hd, c10::Device dev) {
  TORCH_CHECK_VALUE(q.has_value() == k.has_value(), "gamma_q and gamma_k: both or neither");
  if (!q) return;
  vec("gamma_q", *q, hd, kF32, dev);
  vec("gamma_k", *k, hd, kF32, dev);
}
void on(const char* name, int64_t index, c10::Device dev) {
  TORCH_CHECK_VALUE(index == dev.index(), name, ": has to be on ", dev);
}
// (hd, v heads) of q | k | v rows: hd from the column count, with or without the v part (the count
// fits one of the four: 128 without v would be 64 with v only for heads == 0).
std::pair<int64_t, int64_t> vectors(const Tensor& t, int64_t heads, int64_t kv_heads) {
  const int64_t cols = t.dim() == 2 ? t.size(1) : 0;
  if (heads > 0 && kv_heads > 0)
    for (const int64_t v : {kv_heads, int64_t(0)})
      for (const int64_t hd : {int64_t(128), int64_t(64)})
        if (cols == (heads + kv_heads + v) * hd) return {hd, v};
  TORCH_CHECK_VALUE(false, "rows of ", t.sizes(), " do not hold ", heads, " q and ", kv_heads,
                    " k (and v) heads of 64 or 128");
}

Tensor qk_norm_rope(const Tensor& qkv, const Tensor& positions, int64_t rope, int64_t rope_dev, int64_t heads,
                    int64_t kv_heads, const Opt& gamma_q, const Opt& gamma_k, double eps, const Opt& out_given,
                    const Opt& err) {
  const c10::Device dev = cuda(qkv);
  const auto [hd, nv] = vectors(qkv, heads, kv_heads);
  const int64_t T = qkv.size(0), cols = qkv.size(1);
  const int64_t ld = rows("qkv", qkv, cols, kBf16, dev);
  vec("positions", positions, T, kI32, dev);
  gammas(gamma_q, gamma_k, hd, dev);
  on("rope", rope_dev, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = out_given ? *out_given : like(qkv);
  const int64_t ldo = rows("out", out, cols, kBf16, dev, T);
  done(rt_kernel_qk_norm_rope_fwd(ptr<void>(qkv), ld, ptr<void>(out), ldo, ptr<int32_t>(positions),
                                  reinterpret_cast<const rt_rope*>(rope), ptr<float>(gamma_q), ptr<float>(gamma_k),
                                  static_cast<float>(eps), T, heads, kv_heads, nv, hd, error_word(err, dev), stream(dev)),
       "rt_kernel_qk_norm_rope_fwd");
  return out;
}

std::tuple<Tensor, Opt, Opt> qk_norm_rope_backward(const Tensor& dout, const Opt& qkv, const Tensor& positions,
                                                   int64_t rope, int64_t rope_dev, int64_t heads, int64_t kv_heads,
                                                   const Opt& gamma_q, const Opt& gamma_k, double eps,
                                                   const Opt& dqkv_given, const Opt& dgq_given, const Opt& dgk_given,
                                                   const Opt& err) {
  const c10::Device dev = cuda(dout);
  const auto [hd, nv] = vectors(dout, heads, kv_heads);
  const int64_t T = dout.size(0), cols = dout.size(1);
  const int64_t ld = rows("dout", dout, cols, kBf16, dev);
  vec("positions", positions, T, kI32, dev);
  gammas(gamma_q, gamma_k, hd, dev);
  on("rope", rope_dev, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor dqkv = dqkv_given ? *dqkv_given : like(dout);
  const int64_t lddx = rows("dqkv", dqkv, cols, kBf16, dev, T);
  Opt dgq, dgk, partials;
  int64_t ldx = 0;
  if (gamma_q) {
    TORCH_CHECK_VALUE(qkv.has_value(), "the gammas' backward reads qkv");
    ldx = rows("qkv", *qkv, cols, kBf16, dev, T);
    TORCH_CHECK_VALUE(dgq_given.has_value() == dgk_given.has_value(), "dgamma_q and dgamma_k: both or neither");
    dgq = dgq_given ? *dgq_given : like(*gamma_q);
    dgk = dgk_given ? *dgk_given : like(*gamma_k);
    vec("dgamma_q", *dgq, hd, kF32, dev);
    vec("dgamma_k", *dgk, hd, kF32, dev);
    partials = at::empty({rt_kernel_qk_norm_rope_bwd_partials(T, heads, kv_heads) * hd}, gamma_q->options());
  }
  done(rt_kernel_qk_norm_rope_bwd(ptr<void>(dout), ld, gamma_q ? ptr<void>(qkv) : nullptr, ldx, ptr<void>(dqkv), lddx,
                                  ptr<int32_t>(positions), reinterpret_cast<const rt_rope*>(rope), ptr<float>(gamma_q),
                                  ptr<float>(gamma_k), static_cast<float>(eps), ptr<float>(dgq), ptr<float>(dgk),
                                  gamma_q && dgq_given, ptr<float>(partials), T, heads, kv_heads, nv, hd,
                                  error_word(err, dev), stream(dev)),
       "rt_kernel_qk_norm_rope_bwd");
  return {dqkv, dgq, dgk};
}

Tensor kv_append(const Tensor& qkv, const Tensor& positions, const Tensor& slots, int64_t rope, int64_t rope_dev,
                 int64_t cache, int64_t cache_dev, int64_t err, int64_t heads, const Opt& gamma_q, const Opt& gamma_k,
                 double eps, const Opt& q_given) {
  const auto* c = reinterpret_cast<const rt_kv_pages*>(cache);
  const c10::Device dev = device_of(cache_dev);
  const int64_t ld = rows("qkv", qkv, (heads + 2 * c->kv_heads) * c->hd, kBf16, dev), T = qkv.size(0);
  vec("positions", positions, T, kI32, dev);
  vec("slots", slots, T, kI32, dev);
  gammas(gamma_q, gamma_k, c->hd, dev);
  on("rope", rope_dev, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor q = q_given ? *q_given : at::empty({T, heads * c->hd}, qkv.options());
  const int64_t ldq = rows("q_out", q, heads * c->hd, kBf16, dev, T);
  done(rt_kernel_kv_append(ptr<void>(qkv), ld, ptr<void>(q), ldq, ptr<int32_t>(positions), ptr<int32_t>(slots),
                           reinterpret_cast<const rt_rope*>(rope), ptr<float>(gamma_q), ptr<float>(gamma_k),
                           static_cast<float>(eps), c, T, heads, reinterpret_cast<int*>(err), stream(dev)),
       "rt_kernel_kv_append");
  return q;
}

std::tuple<Tensor, Tensor> kv_gather(int64_t cache, int64_t cache_dev, int64_t err, const Tensor& slots,
                                     const Opt& k_given, const Opt& v_given) {
  const auto* c = reinterpret_cast<const rt_kv_pages*>(cache);
  const c10::Device dev = device_of(cache_dev);
  const int64_t T = slots.dim() == 1 ? slots.size(0) : -1;
  vec("slots", slots, T, kI32, dev);
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t shape[3] = {T, c->kv_heads, c->hd};
  auto output = [&](const char* name, const Opt& given) {
    if (!given) return at::empty(shape, slots.options().dtype(kBf16));
    TORCH_CHECK_VALUE(given->sizes() == at::IntArrayRef(shape) && given->scalar_type() == kBf16 && given->device() == dev &&
                          given->is_contiguous(),
                      name, ": a contiguous bf16 [", T, ", ", c->kv_heads, ", ", c->hd, "] tensor on ", dev);
    return *given;
  };
  const Tensor k = output("k_out", k_given), v = output("v_out", v_given);
  done(rt_kernel_kv_gather(c, ptr<int32_t>(slots), ptr<void>(k), ptr<void>(v), int64_t(c->kv_heads) * c->hd, T,
                           reinterpret_cast<int*>(err), stream(dev)),
       "rt_kernel_kv_gather");
  return {k, v};
}

std::tuple<Tensor, Opt> attention_paged(const Tensor& q, int64_t cache, int64_t cache_dev, int64_t err,
                                        const Tensor& page_table, const Tensor& kv_lens, const Tensor& q_start,
                                        int64_t heads, int64_t workspace, int64_t workspace_bytes,
                                        int64_t workspace_dev, int64_t max_q, int64_t max_kv, int64_t window,
                                        double scale, const Opt& out_given, bool want_lse) {
  const auto* c = reinterpret_cast<const rt_kv_pages*>(cache);
  const c10::Device dev = device_of(cache_dev);
  const int64_t cols = heads * c->hd, ldq = rows("q", q, cols, kBf16, dev), T = q.size(0);
  const int64_t n = kv_lens.dim() == 1 ? kv_lens.size(0) : -1;
  vec("kv_lens", kv_lens, n, kI32, dev);
  vec("q_start", q_start, n + 1, kI32, dev);
  const int64_t pages = page_table.dim() == 2 ? page_table.size(1) : 0;  // of a row; its stride may be another number
  const int64_t ldt = rows("page_table", page_table, pages, kI32, dev, n);
  on("workspace", workspace_dev, dev);
  auto to_int = [](int64_t v) { return static_cast<int>(std::clamp<int64_t>(v, -1, INT32_MAX)); };
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = out_given ? *out_given : like(q);
  const int64_t ldo = rows("out", out, cols, kBf16, dev, T);
  Opt lse2;
  if (want_lse) lse2 = at::empty({T, heads}, q.options().dtype(kF32));
  done(rt_kernel_attention_paged_cols(ptr<void>(q), ldq, ptr<void>(out), ldo, ptr<float>(lse2), c,
                                      ptr<int32_t>(page_table), ldt, pages, ptr<int32_t>(kv_lens), ptr<int32_t>(q_start),
                                      n, T, to_int(max_q), to_int(max_kv), heads, to_int(window),
                                      static_cast<float>(scale), reinterpret_cast<void*>(workspace), workspace_bytes,
                                      reinterpret_cast<int*>(err), stream(dev)),
       "rt_kernel_attention_paged");
  return {out, lse2};
}

std::tuple<Tensor, Tensor> logits_adjust(const Tensor& logits, const Opt& hist, const Opt& hist_start,
                                         const Opt& n_prompt, const Opt& repetition, const Opt& presence,
                                         const Opt& frequency, const Opt& bias_ids, const Opt& bias_vals,
                                         const Opt& bias_start, const Opt& mask, const Opt& out_given, const Opt& err) {
  const c10::Device dev = cuda(logits);
  TORCH_CHECK_VALUE(logits.dim() == 2, "logits: [B, V]");
  const int64_t B = logits.size(0), V = logits.size(1), ldl = rows("logits", logits, V, kF32, dev);
  rt_logit_rules r{};
  if (hist) {
    TORCH_CHECK_VALUE(hist_start.has_value(), "hist needs hist_start");
    vec("hist", *hist, -1, kI32, dev);
    vec("hist_start", *hist_start, B + 1, kI32, dev);
    r.hist = ptr<int32_t>(hist);
    r.hist_start = ptr<int32_t>(hist_start);
    r.n_hist = hist->size(0);
    if (n_prompt) {
      vec("n_prompt", *n_prompt, B, kI32, dev);
      r.n_prompt = ptr<int32_t>(n_prompt);
    }
  }
  auto factor = [&](const char* name, const Opt& t) -> const float* {
    if (t) vec(name, *t, B, kF32, dev);
    return ptr<float>(t);
  };
  r.repetition = factor("repetition", repetition);
  r.presence = factor("presence", presence);
  r.frequency = factor("frequency", frequency);
  if (bias_ids) {
    TORCH_CHECK_VALUE(bias_vals && bias_start, "bias_ids needs bias_vals and bias_start");
    vec("bias_ids", *bias_ids, -1, kI32, dev);
    vec("bias_vals", *bias_vals, bias_ids->size(0), kF32, dev);
    vec("bias_start", *bias_start, B + 1, kI32, dev);
    r.bias_ids = ptr<int32_t>(bias_ids);
    r.bias_vals = ptr<float>(bias_vals);
    r.bias_start = ptr<int32_t>(bias_start);
    r.n_bias = bias_ids->size(0);
  }
  if (mask) {
    r.mask_ld = rows("mask", *mask, (V + 31) / 32, kI32, dev, B);
    r.mask = ptr<uint32_t>(mask);
  }
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = out_given ? *out_given : like(logits);
  const int64_t ldo = rows("out", out, V, kF32, dev, B);
  const Tensor token = at::empty({B}, logits.options().dtype(kI32));
  done(rt_kernel_logits_adjust(ptr<float>(logits), ldl, ptr<float>(out), ldo, ptr<int32_t>(token), B, V, &r,
                               error_word(err, dev), stream(dev)),
       "rt_kernel_logits_adjust");
  return {out, token};
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward);
  m.def("kv_append", &kv_append);
  m.def("kv_gather", &kv_gather);
  m.def("attention_paged", &attention_paged);
  m.def("logits_adjust", &logits_adjust);
}
