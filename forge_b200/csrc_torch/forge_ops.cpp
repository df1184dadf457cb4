// Direct calls of the loss, multi-tensor and 8-bit entry points of the C ABI from PyTorch, for calls that are so short
// that marshalling them in Python would take longer than the kernels run (a decoding step's log probabilities, the
// norm weights of a decoder).  Every function returns None for arguments that are not of the plain form it handles
// (another dtype or layout, a wrong shape, CPU tensors, a derivative carried forward or a trace being recorded); the Python
// wrappers then take over, which check, copy or refuse.
// Both paths issue the same library calls.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <array>
#include <vector>

#include "../../include/forge_b200.h"

namespace {

namespace py = pybind11;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the exceptions of forge_b200._lib.check
void check(int rc, const char* what) {
  if (rc == FORGE_OK) return;
  if (rc == FORGE_ERR_INVALID_ARG || rc == FORGE_ERR_SHAPE || rc == FORGE_ERR_UNSUPPORTED)
    TORCH_CHECK_VALUE(false, what, ": ", forge_last_error_string(), " (code ", rc, ")");
  const std::string message = c10::str(what, ": ", forge_last_error_string(), " (code ", rc, ")");
  py::gil_scoped_acquire gil;                // (a backward pass runs without it)
  py::set_error(py::module_::import("forge_b200._lib").attr("ForgeLibraryError"), message.c_str());
  throw py::error_already_set();
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

bool float_type(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
int dtype_id(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? FORGE_DT_BF16 : FORGE_DT_F32; }

// whether something besides x.requires_grad() follows what happens to x (forge_b200.native.followed)
bool followed(const at::Tensor& x) { return torch::jit::tracer::isTracing() || x._fw_grad(0).defined(); }

// an error for whoever differentiates a gradient again
at::Tensor once(const at::Tensor& g) {
  if (!at::GradMode::is_enabled()) return g;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that supports one derivative only", 1);
  return (*node)({g})[0];
}

// Saved tensors come back from whatever hooks are set on them (torch.autograd.graph.saved_tensors_hooks): in another layout,
// perhaps, or as something else altogether, which is refused here as it would be at the operator's own entry.
void check_saved(bool ok, const char* what) { TORCH_CHECK(ok, what, ": what was saved for the backward pass came back as something else"); }

// ----- token log probabilities ---------------------------------------------------------------------
struct Rows {
  int64_t rows, vocab, ld;
};

bool as_rows(const at::Tensor& x, Rows& r) {
  if (!x.is_cuda() || !float_type(x) || x.dim() < 1 || x.numel() == 0) return false;
  r.vocab = x.size(-1);
  r.rows = x.numel() / r.vocab;
  r.ld = r.vocab;
  if (x.is_contiguous()) return true;
  if (x.dim() != 2 || x.stride(1) != 1 || x.stride(0) < r.vocab) return false;
  r.ld = x.stride(0);
  return true;
}

ForgeLogprobsArgs loss_args(const at::Tensor& x, const Rows& r, const at::Tensor& t, int64_t top_k, double temperature, int64_t ignore) {
  ForgeLogprobsArgs a = {};
  a.logits = x.const_data_ptr();
  a.targets = t.defined() ? static_cast<const int64_t*>(t.const_data_ptr()) : nullptr;
  a.rows = r.rows;
  a.vocab = a.vocab_total = r.vocab;
  a.ld = r.ld;
  a.ignore_index = ignore;
  a.temperature = temperature;
  a.dtype = dtype_id(x);
  a.top_k = static_cast<int32_t>(top_k);
  return a;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

// {logprobs, entropy, top_logprobs, top_ids, and for the gradient row_max, log_sum}
std::array<at::Tensor, 6> loss_forward(const at::Tensor& x, const at::Tensor& t, int64_t top_k, double temperature, int64_t ignore,
                                       bool gradient) {
  Rows r;
  as_rows(x, r);
  const int dev = x.get_device();
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  ForgeLogprobsArgs a = loss_args(x, r, t, top_k, temperature, ignore);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  std::array<at::Tensor, 6> out;
  float** const per_row[6] = {&a.logprobs, &a.entropy, nullptr, nullptr, &a.row_max, &a.log_sum};
  for (int i : {0, 1, 4, 5}) {
    if (i >= 4 && !gradient) continue;
    out[i] = empty(lead, at::kFloat, x);
    *per_row[i] = static_cast<float*>(out[i].data_ptr());
  }
  if (top_k > 0) {
    c10::SmallVector<int64_t, 6> shape(lead.begin(), lead.end());
    shape.push_back(top_k);
    out[2] = empty(shape, at::kFloat, x);
    out[3] = empty(shape, at::kLong, x);
    a.top_logprobs = static_cast<float*>(out[2].data_ptr());
    a.top_ids = static_cast<int64_t*>(out[3].data_ptr());
  }
  check(forge_logprobs_forward(&a, stream_of(dev)), "forge_logprobs_forward");
  return out;
}

class TokenLogprobsFn : public torch::autograd::Function<TokenLogprobsFn> {
 public:
  // (no targets: none, since an undefined tensor is no argument that apply() takes)
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& targets, int64_t top_k,
                               double temperature, int64_t ignore) {
    const at::Tensor t = targets.value_or(at::Tensor());
    auto out = loss_forward(x, t, top_k, temperature, ignore, true);
    ctx->save_for_backward({x, t, out[1], out[4], out[5]});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    if (top_k > 0) {
      ctx->mark_non_differentiable({out[2], out[3]});
      return {out[0], out[1], out[2], out[3]};
    }
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    at::Tensor x = saved[0], t = saved[1];
    variable_list none(5);
    if (!g[0].defined() && !g[1].defined()) return none;
    at::Tensor gr[2];
    for (int i = 0; i < 2; ++i)
      if (g[i].defined()) gr[i] = g[i].detach().to(at::kFloat).contiguous();
    at::Tensor dx;
    {
      at::NoGradGuard no_grad;
      Rows r;
      x = as_rows(x, r) ? x : x.contiguous();
      check_saved(as_rows(x, r), "token_logprobs");
      const int dev = x.get_device();
      auto per_row_of = [&](const at::Tensor& s, at::ScalarType type) {
        return s.is_cuda() && s.get_device() == dev && s.scalar_type() == type && s.numel() == r.rows;
      };
      check_saved(!t.defined() || per_row_of(t, at::kLong), "token_logprobs");
      if (t.defined()) t = t.contiguous();
      c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
      ForgeLogprobsArgs a = loss_args(x, r, t, 0, ctx->saved_data["temperature"].toDouble(), ctx->saved_data["ignore"].toInt());
      float** const per_row[3] = {&a.entropy, &a.row_max, &a.log_sum};
      at::Tensor rows[3];
      for (int i = 0; i < 3; ++i) {
        check_saved(per_row_of(saved[2 + i], at::kFloat), "token_logprobs");
        rows[i] = saved[2 + i].contiguous();
        *per_row[i] = static_cast<float*>(const_cast<void*>(rows[i].const_data_ptr()));
      }
      dx = empty(x.sizes(), x.scalar_type(), x);
      check(forge_logprobs_backward(&a, gr[0].defined() ? static_cast<const float*>(gr[0].const_data_ptr()) : nullptr,
                                    gr[1].defined() ? static_cast<const float*>(gr[1].const_data_ptr()) : nullptr, dx.data_ptr(), r.vocab,
                                    stream_of(dev)),
            "forge_logprobs_backward");
    }
    none[0] = once(dx);
    return none;
  }
};

py::object token_logprobs(const at::Tensor& x, const c10::optional<at::Tensor>& targets, int64_t top_k, double temperature, int64_t ignore) {
  Rows r;
  if (!as_rows(x, r) || top_k < 0 || top_k > 32 || top_k > r.vocab || followed(x)) return py::none();
  at::Tensor t;
  if (targets.has_value() && targets->defined()) {
    t = *targets;
    if (t.scalar_type() != at::kLong || !t.is_cuda() || t.get_device() != x.get_device() || !t.is_contiguous() ||
        t.sizes() != x.sizes().slice(0, x.dim() - 1))
      return py::none();
  }
  const py::object none = py::none();
  auto wrap = [](const at::Tensor& v) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(v)); };
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    const auto out = TokenLogprobsFn::apply(x, t.defined() ? std::optional<at::Tensor>(t) : std::nullopt, top_k, temperature, ignore);
    return py::make_tuple(wrap(out[0]), wrap(out[1]), top_k ? wrap(out[2]) : none, top_k ? wrap(out[3]) : none);
  }
  const auto out = loss_forward(x, t, top_k, temperature, ignore, false);
  return py::make_tuple(wrap(out[0]), wrap(out[1]), top_k ? wrap(out[2]) : none, top_k ? wrap(out[3]) : none);
}

// ----- AdamW over a list of tensors -----------------------------------------------------------------
// a list or tuple of tensors -> pointers to them (no reference counts touched); false if it holds anything else
bool unpack(const py::handle& seq, std::vector<const at::Tensor*>& out) {
  PyObject* o = seq.ptr();
  const bool list = PyList_CheckExact(o);
  if (!list && !PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
  out.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* e = list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i);
    if (!THPVariable_Check(e)) return false;
    out[i] = &THPVariable_Unpack(e);
  }
  return true;
}

// a set of addresses in one flat table
class PointerSet {
 public:
  explicit PointerSet(size_t most) {
    while ((size_t(1) << bits_) < 2 * most) ++bits_;
    table_.assign(size_t(1) << bits_, nullptr);
  }
  // false if it was there already
  bool insert(const void* p) {
    const size_t mask = table_.size() - 1;
    for (size_t i = (reinterpret_cast<uintptr_t>(p) * 0x9E3779B97F4A7C15ull) >> (64 - bits_);; i = (i + 1) & mask) {
      if (table_[i] == p) return false;
      if (table_[i] == nullptr) {
        table_[i] = p;
        return true;
      }
    }
  }

 private:
  int bits_ = 4;
  std::vector<const void*> table_;
};

bool plain(const at::Tensor& t, int dev) {
  return t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided && t.is_contiguous();
}

// norm and (max_norm > 0) the factor that clips to it, as two elements of one tensor
at::Tensor norm_of(const std::vector<ForgeNormItem>& items, double max_norm, const at::Tensor& like, void* stream) {
  const int32_t n = static_cast<int32_t>(items.size());
  const size_t bytes = forge_multi_norm_scratch_bytes(items.data(), n);
  at::Tensor out = empty({2}, at::kFloat, like), scratch = empty({static_cast<int64_t>(bytes + 8)}, at::kByte, like);
  float* o = static_cast<float*>(out.data_ptr());
  check(forge_multi_norm(items.data(), n, max_norm, o, max_norm > 0 ? o + 1 : nullptr, scratch.data_ptr(), bytes, stream), "forge_multi_norm");
  return out;
}

// None: not of the plain form.  Otherwise (norm, factor or None).
py::object multi_norm(const py::object& grads, double max_norm) {
  const py::object none = py::none();
  std::vector<const at::Tensor*> g;
  if (!unpack(grads, g) || g.empty() || !g[0]->is_cuda()) return none;
  const int dev = g[0]->get_device();
  std::vector<ForgeNormItem> items(g.size());
  for (size_t i = 0; i < g.size(); ++i) {
    if (!plain(*g[i], dev) || !float_type(*g[i])) return none;
    items[i] = ForgeNormItem{g[i]->const_data_ptr(), g[i]->numel(), dtype_id(*g[i]), 0};
  }
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const at::Tensor out = norm_of(items, max_norm, *g[0], stream_of(dev));
  auto wrap = [](const at::Tensor& v) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(v)); };
  return py::make_tuple(wrap(out.select(0, 0)), max_norm > 0 ? wrap(out.select(0, 1)) : none);
}

// None: not of the plain form.  Otherwise (done, norm or None).
py::object multi_adamw(const py::object& params, const py::object& grads, const py::object& exp_avgs, const py::object& exp_avg_sqs,
                       const py::object& m_scales, const py::object& v_scales, double lr, double beta1, double beta2, double eps,
                       double weight_decay, int64_t step, double max_norm, int64_t hyper_device, const c10::optional<at::Tensor>& grad_coef) {
  const py::object none = py::none();
  std::vector<const at::Tensor*> p, g, m, v, ms, vs;
  if (!unpack(params, p) || !unpack(grads, g) || !unpack(exp_avgs, m) || !unpack(exp_avg_sqs, v)) return none;
  const size_t n = p.size();
  if (n == 0 || g.size() != n || m.size() != n || v.size() != n || !p[0]->is_cuda() || (hyper_device == 0 && step < 1)) return none;
  const int dev = p[0]->get_device();
  const auto sdt = m[0]->scalar_type();
  int mode;
  if (sdt == at::kFloat) mode = FORGE_ST_F32;
  else if (sdt == at::kBFloat16) mode = FORGE_ST_BF16;
  else if (sdt == at::kChar) mode = FORGE_ST_INT8;
  else if (sdt == at::kFloat8_e4m3fn) mode = FORGE_ST_FP8_BLOCK;
  else return none;
  const bool quant = mode == FORGE_ST_INT8 || mode == FORGE_ST_FP8_BLOCK;
  if (quant) {
    if (!unpack(m_scales, ms) || !unpack(v_scales, vs) || ms.size() != n || vs.size() != n) return none;
  } else if (!m_scales.is_none() || !v_scales.is_none()) {
    return none;
  }
  std::vector<ForgeMultiItem> items(n);
  PointerSet seen((quant ? 5 : 3) * n);
  for (size_t i = 0; i < n; ++i) {
    const int64_t num = p[i]->numel();
    if (!plain(*p[i], dev) || !plain(*g[i], dev) || !plain(*m[i], dev) || !plain(*v[i], dev) || !float_type(*p[i]) || !float_type(*g[i]) ||
        m[i]->scalar_type() != sdt || v[i]->scalar_type() != sdt || g[i]->sizes() != p[i]->sizes() || m[i]->numel() != num || v[i]->numel() != num)
      return none;
    ForgeMultiItem& it = items[i];
    it = ForgeMultiItem{};
    it.param = p[i]->mutable_data_ptr();
    it.grad = g[i]->const_data_ptr();
    it.m = m[i]->mutable_data_ptr();
    it.v = v[i]->mutable_data_ptr();
    it.numel = num;
    it.param_dtype = dtype_id(*p[i]);
    it.grad_dtype = dtype_id(*g[i]);
    if (quant) {
      const int64_t blocks = (num + 63) / 64;
      for (const at::Tensor* s : {ms[i], vs[i]})
        if (!plain(*s, dev) || s->scalar_type() != at::kFloat || s->numel() != blocks) return none;
      it.m_scale = static_cast<float*>(ms[i]->mutable_data_ptr());
      it.v_scale = static_cast<float*>(vs[i]->mutable_data_ptr());
    }
    if (num > 0 && !(seen.insert(it.param) && seen.insert(it.m) && seen.insert(it.v) &&
                     (!quant || (seen.insert(it.m_scale) && seen.insert(it.v_scale)))))
      return none;
  }
  ForgeMultiArgs a = {};
  if (grad_coef.has_value() && grad_coef->defined()) {
    if (!plain(*grad_coef, dev) || grad_coef->scalar_type() != at::kFloat || grad_coef->numel() != 1 || max_norm > 0) return none;
    a.grad_coef = static_cast<const float*>(grad_coef->const_data_ptr());
  }
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  void* stream = stream_of(dev);
  at::Tensor out;
  if (max_norm > 0) {
    std::vector<ForgeNormItem> gi(n);
    for (size_t i = 0; i < n; ++i) gi[i] = ForgeNormItem{items[i].grad, items[i].numel, items[i].grad_dtype, 0};
    out = norm_of(gi, max_norm, *p[0], stream);
    a.grad_coef = static_cast<float*>(out.data_ptr()) + 1;
  }
  a.items = items.data();
  a.count = static_cast<int32_t>(n);
  a.state_mode = mode;
  a.hyper = ForgeHyper{lr, beta1, beta2, eps, weight_decay, 0.0, 0, static_cast<int32_t>(step)};
  a.hyper_device = reinterpret_cast<const void*>(hyper_device);
  check(forge_multi_adamw(&a, stream), "forge_multi_adamw");
  // for autograd: a graph that has saved one of these tensors must not go on with other values
  for (const auto* list : {&p, &m, &v})
    for (const at::Tensor* t : *list)
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return py::make_tuple(true, max_norm > 0 ? py::reinterpret_steal<py::object>(THPVariable_Wrap(out.select(0, 0))) : none);
}

// ----- products in 8-bit floating point -------------------------------------------------------------
int32_t* g_status[64] = {};

bool code_matrix(const at::Tensor& t, int dev) {
  return t.defined() && t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kFloat8_e4m3fn && t.dim() == 2 && t.size(0) > 0 &&
         t.size(1) > 0 && t.stride(1) == 1 && t.stride(0) >= t.size(1) && t.stride(0) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}
bool scale_matrix(const at::Tensor& t, int dev, int64_t rows, int64_t cols) {
  return t.defined() && t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols;
}
int64_t blocks(int64_t n) { return (n + 127) / 128; }

// saved codes whose rows no longer start on 16-byte boundaries (save_on_cpu brings them back without their pitch) get them again
at::Tensor saved_codes(const at::Tensor& t, int dev) {
  if (code_matrix(t, dev)) return t;
  check_saved(t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kFloat8_e4m3fn && t.dim() == 2, "fp8_linear");
  at::Tensor q = empty({t.size(0), (t.size(1) + 15) / 16 * 16}, at::kFloat8_e4m3fn, t).narrow(1, 0, t.size(1));
  return q.copy_(t);
}

// contiguous x (..., K), quantised by rows, times the codes (N, K) of a weight -> (..., N) bf16
at::Tensor linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& ws) {
  const int dev = x.get_device();
  const int64_t M = x.numel() / w.size(1);
  const int64_t K = w.size(1), N = w.size(0), pitch = (K + 15) / 16 * 16, kb = blocks(K);
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  void* stream = stream_of(dev);
  // codes and scales of this call in one allocation: rows of `pitch` bytes, then M x kb floats
  at::Tensor buf = empty({M * pitch + M * kb * 4}, at::kByte, x);
  uint8_t* codes = static_cast<uint8_t*>(buf.data_ptr());
  float* scales = reinterpret_cast<float*>(codes + M * pitch);
  ForgeFp8QuantizeArgs q = {};
  q.x = x.const_data_ptr();
  q.rows = M; q.cols = K; q.ld_x = K;
  q.dtype = dtype_id(x);
  q.block_rows = 1;
  q.codes = codes;
  q.ld_codes = pitch;
  q.scales = scales;
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = empty(shape, at::kBFloat16, x);
  ForgeFp8ProductArgs a = {};
  a.x_codes = codes; a.x_scales = scales;
  a.w_codes = w.const_data_ptr(); a.w_scales = static_cast<const float*>(ws.const_data_ptr());
  a.y = y.data_ptr();
  a.M = M; a.N = N; a.K = K;
  a.ld_x = pitch; a.ld_w = w.stride(0); a.ld_y = N;
  a.x_scale_row = kb; a.x_scale_col = 1;
  a.w_scale_row = ws.stride(0); a.w_scale_col = ws.stride(1);
  a.status = g_status[dev];
  check(forge_fp8_linear(&q, &a, stream), "forge_fp8_linear");
  return y;
}

class Fp8LinearFn : public torch::autograd::Function<Fp8LinearFn> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& ws, const at::Tensor& wt,
                            const at::Tensor& wts) {
    ctx->save_for_backward({wt, wts});
    return linear(x, w, ws);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(5);
    if (!g[0].defined()) return out;
    at::Tensor dx;
    {
      at::NoGradGuard no_grad;
      const at::Tensor dy = g[0].contiguous(), codes = saved_codes(saved[0], dy.get_device());
      check_saved(codes.size(1) == dy.size(-1) && scale_matrix(saved[1], dy.get_device(), blocks(codes.size(0)), blocks(codes.size(1))),
                  "fp8_linear");
      dx = linear(dy, codes, saved[1]);
    }
    out[0] = once(dx);
    return out;
  }
};

py::object fp8_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& ws, const c10::optional<at::Tensor>& wt,
                      const c10::optional<at::Tensor>& wts) {
  if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || !x.is_contiguous() || x.dim() < 1 || x.numel() == 0 || followed(x)) return py::none();
  const int dev = x.get_device();
  if (dev >= 64 || g_status[dev] == nullptr || !code_matrix(w, dev) || x.size(-1) != w.size(1) ||
      !scale_matrix(ws, dev, blocks(w.size(0)), blocks(w.size(1))))
    return py::none();
  at::Tensor y;
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    if (!wt.has_value() || !wts.has_value() || !code_matrix(*wt, dev) || wt->size(0) != w.size(1) || wt->size(1) != w.size(0) ||
        !scale_matrix(*wts, dev, blocks(w.size(1)), blocks(w.size(0))))
      return py::none();
    y = Fp8LinearFn::apply(x, w, ws, *wt, *wts);
  } else {
    y = linear(x, w, ws);
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(y));
}

// (codes, scales[, codes of the transpose, its scales])
py::object quantize(const at::Tensor& x, int64_t block_rows, bool transposed) {
  if (!x.is_cuda() || !float_type(x) || x.dim() != 2 || x.numel() == 0 || !x.is_contiguous() || (block_rows != 1 && block_rows != 128) ||
      (transposed && block_rows == 1) || torch::jit::tracer::isTracing())
    return py::none();
  const int dev = x.get_device();
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const int64_t R = x.size(0), C = x.size(1), sr = block_rows == 1 ? R : blocks(R), sc = blocks(C);
  auto codes = [&](int64_t r, int64_t c) {
    const int64_t pitch = (c + 15) / 16 * 16;
    at::Tensor t = empty({r, pitch}, at::kFloat8_e4m3fn, x);
    return pitch == c ? t : t.narrow(1, 0, c);
  };
  at::Tensor q = codes(R, C), s = empty({sr, sc}, at::kFloat, x), qt, st;
  ForgeFp8QuantizeArgs a = {};
  a.x = x.const_data_ptr();
  a.rows = R; a.cols = C; a.ld_x = C;
  a.dtype = dtype_id(x);
  a.block_rows = static_cast<int32_t>(block_rows);
  a.codes = q.data_ptr();
  a.ld_codes = (C + 15) / 16 * 16;
  a.scales = static_cast<float*>(s.data_ptr());
  if (transposed) {
    qt = codes(C, R);
    st = empty({sc, sr}, at::kFloat, x);
    a.codes_t = qt.data_ptr();
    a.ld_codes_t = (R + 15) / 16 * 16;
    a.scales_t = static_cast<float*>(st.data_ptr());
  }
  check(forge_fp8_quantize(&a, stream_of(dev)), "forge_fp8_quantize");
  auto wrap = [](const at::Tensor& v) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(v)); };
  if (!transposed) return py::make_tuple(wrap(q), wrap(s));
  return py::make_tuple(wrap(q), wrap(s), wrap(qt), wrap(st));
}

}  // namespace

void bind_operators(pybind11::module_& m) {
  m.def("token_logprobs", &token_logprobs);
  m.def("multi_adamw", &multi_adamw);
  m.def("multi_norm", &multi_norm);
  m.def("fp8_linear", &fp8_linear);
  m.def("fp8_quantize", &quantize);
  m.def("set_status_word", [](int64_t device, int64_t ptr) {
    if (device >= 0 && device < 64) g_status[device] = reinterpret_cast<int32_t*>(ptr);
  });
}
