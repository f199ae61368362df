// Operators of a training step on the batches that the samplers deliver: layer norm, softmax cross entropy against a large
// vocabulary, AdamW.  Additions (no counterparts in the reference's src/pybind.cc); thin layers over the C ABI like the
// operators of ops.cc.
#pragma once
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "chunk_tensor.h"

namespace dgs {

inline int32_t training_dtype(const torch::Tensor& t, const char* op, const char* what) {
  switch (t.scalar_type()) {
    case torch::kFloat: return DGS_F32;
    case torch::kBFloat16: return DGS_BF16;
    case torch::kHalf: return DGS_F16;
    default: TORCH_CHECK(false, op, ": ", what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

inline void check_on(const torch::Tensor& t, const torch::Device& dev, const char* op, const char* what) {
  TORCH_CHECK(t.device() == dev, op, ": ", what, " must be on ", dev, ", is on ", t.device());
}

// `t` as rows of `D` elements: its own memory where the rows are whole and do not overlap, else a contiguous copy.
struct Rows {
  torch::Tensor t;
  int64_t stride;
};
inline Rows as_rows(const torch::Tensor& t, int64_t D) {
  if (t.is_contiguous()) return {t, D};
  if (t.dim() == 2 && (t.stride(1) == 1 || D == 1) && t.stride(0) >= D) return {t, t.stride(0)};
  return {t.contiguous(), D};
}

inline std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> LayerNormCUDA(torch::Tensor x, c10::optional<torch::Tensor> weight,
                                                                             c10::optional<torch::Tensor> bias, double eps) {
  const char* op = "_CAPI_layer_norm";
  CHECK_CUDA(x);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, op, ": x must have at least one dimension and rows of at least one element");
  const int32_t dtype = training_dtype(x, op, "x");
  const int64_t D = x.size(-1), n = x.numel() / D;
  int32_t pd = dtype;
  torch::Tensor w, b;
  TORCH_CHECK(weight.has_value() || !bias.has_value(), op, ": a bias needs a weight");
  if (weight.has_value()) {
    check_on(*weight, x.device(), op, "weight");
    TORCH_CHECK(weight->dim() == 1 && weight->size(0) == D, op, ": weight must have the ", D, " elements of a row");
    pd = training_dtype(*weight, op, "weight");
    w = weight->contiguous();
  }
  if (bias.has_value()) {
    check_on(*bias, x.device(), op, "bias");
    TORCH_CHECK(bias->sizes() == weight->sizes() && bias->scalar_type() == weight->scalar_type(), op,
                ": bias must have the weight's shape and type");
    b = bias->contiguous();
  }
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = as_rows(x, D);
  torch::Tensor y = device_empty(x.sizes(), x.scalar_type(), x.device());
  torch::Tensor mean = device_empty(x.sizes().slice(0, x.dim() - 1), torch::kFloat, x.device());
  torch::Tensor rstd = device_empty(x.sizes().slice(0, x.dim() - 1), torch::kFloat, x.device());
  DGS_CHECK_RC(dgs_layer_norm(r.t.data_ptr(), r.stride, dtype, w.defined() ? w.data_ptr() : nullptr,
                              b.defined() ? b.data_ptr() : nullptr, pd, n, D, static_cast<float>(eps), y.data_ptr(),
                              mean.data_ptr<float>(), rstd.data_ptr<float>(), current_stream()));
  return std::make_tuple(y, mean, rstd);
}

// (dx, dweight, dbias); what is not wanted comes back with no elements
inline std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> LayerNormBackwardCUDA(torch::Tensor grad, torch::Tensor x,
                                                                                     c10::optional<torch::Tensor> weight,
                                                                                     torch::Tensor mean, torch::Tensor rstd,
                                                                                     bool want_input, bool want_params) {
  const char* op = "_CAPI_layer_norm_backward";
  CHECK_CUDA(x);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, op, ": x must have at least one dimension and rows of at least one element");
  check_on(grad, x.device(), op, "grad");
  check_on(mean, x.device(), op, "mean");
  check_on(rstd, x.device(), op, "rstd");
  const int32_t dtype = training_dtype(x, op, "x");
  TORCH_CHECK(grad.sizes() == x.sizes() && grad.scalar_type() == x.scalar_type(), op, ": grad must have x's shape and type");
  const int64_t D = x.size(-1), n = x.numel() / D;
  TORCH_CHECK(mean.scalar_type() == torch::kFloat && rstd.scalar_type() == torch::kFloat && mean.numel() == n && rstd.numel() == n, op,
              ": mean and rstd must be the float32 values of ", n, " rows that _CAPI_layer_norm returned");
  TORCH_CHECK(weight.has_value() || !want_params, op, ": without a weight there are no gradients of the parameters");
  int32_t pd = dtype;
  torch::Tensor w;
  if (weight.has_value()) {
    check_on(*weight, x.device(), op, "weight");
    TORCH_CHECK(weight->dim() == 1 && weight->size(0) == D, op, ": weight must have the ", D, " elements of a row");
    pd = training_dtype(*weight, op, "weight");
    w = weight->contiguous();
  }
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = as_rows(x, D), g = as_rows(grad, D);
  mean = mean.contiguous();
  rstd = rstd.contiguous();
  const auto ptype = w.defined() ? w.scalar_type() : torch::kFloat;
  torch::Tensor dx = want_input ? device_empty(x.sizes(), x.scalar_type(), x.device()) : device_empty({0}, x.scalar_type(), x.device());
  torch::Tensor dw = device_empty({want_params ? D : 0}, ptype, x.device());
  torch::Tensor db = device_empty({want_params ? D : 0}, ptype, x.device());
  const size_t wb = want_params ? dgs_layer_norm_backward_workspace_bytes(n, D) : 0;
  torch::Tensor ws = byte_scratch(wb, x.device());
  DGS_CHECK_RC(dgs_layer_norm_backward(g.t.data_ptr(), g.stride, r.t.data_ptr(), r.stride, dtype, w.defined() ? w.data_ptr() : nullptr,
                                       pd, mean.data_ptr<float>(), rstd.data_ptr<float>(), n, D, want_input ? dx.data_ptr() : nullptr,
                                       want_params ? dw.data_ptr() : nullptr, want_params ? db.data_ptr() : nullptr, ws.data_ptr(), wb,
                                       current_stream()));
  return std::make_tuple(dx, dw, db);
}

namespace {
// what both directions of the cross entropy check
struct CrossEntropyInputs {
  int64_t n, D, V;
  int32_t dtype;
  bool ids64;
  Rows hidden, weight;
  torch::Tensor target;
};
inline CrossEntropyInputs cross_entropy_inputs(const char* op, const torch::Tensor& hidden, const torch::Tensor& weight,
                                               const torch::Tensor& target) {
  CHECK_CUDA(hidden);
  check_on(weight, hidden.device(), op, "weight");
  check_on(target, hidden.device(), op, "target");
  TORCH_CHECK(hidden.dim() == 2 && weight.dim() == 2 && hidden.size(1) == weight.size(1), op,
              ": hidden [n, D] and weight [V, D] must be matrices with rows of one length");
  TORCH_CHECK(weight.size(0) >= 1 && weight.size(1) >= 1, op, ": there must be at least one class and one element a row");
  TORCH_CHECK(target.dim() == 1 && target.size(0) == hidden.size(0), op, ": target must hold one id for each row of hidden");
  CrossEntropyInputs in;
  in.n = hidden.size(0);
  in.D = hidden.size(1);
  in.V = weight.size(0);
  in.dtype = training_dtype(hidden, op, "hidden");
  TORCH_CHECK(weight.scalar_type() == hidden.scalar_type(), op, ": hidden and weight must share one type");
  in.ids64 = is_id64(target, "target");
  return in;
}
inline void lay_out(CrossEntropyInputs& in, const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& target) {
  in.hidden = as_rows(hidden, in.D);
  in.weight = as_rows(weight, in.D);
  // 16-bit rows of a multiple of 8 elements are fetched where they lie, which needs 16-byte boundaries
  if (in.dtype != DGS_F32 && in.D % 8 == 0 && (in.weight.stride % 8 != 0 || reinterpret_cast<uintptr_t>(in.weight.t.data_ptr()) % 16 != 0)) {
    in.weight.t = device_empty({in.V, in.D}, weight.scalar_type(), weight.device());
    in.weight.t.copy_(weight);
    in.weight.stride = in.D;
  }
  in.target = target.contiguous();
}
}  // namespace

// (loss, lse), one float32 value for each row
inline std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyCUDA(torch::Tensor hidden, torch::Tensor weight, torch::Tensor target,
                                                                       int64_t ignore_index) {
  const char* op = "_CAPI_linear_cross_entropy";
  CrossEntropyInputs in = cross_entropy_inputs(op, hidden, weight, target);
  c10::cuda::CUDAGuard guard(hidden.device());
  lay_out(in, hidden, weight, target);
  torch::Tensor loss = device_empty({in.n}, torch::kFloat, hidden.device());
  torch::Tensor lse = device_empty({in.n}, torch::kFloat, hidden.device());
  const size_t wb = dgs_linear_cross_entropy_workspace_bytes(in.n, in.D, in.V, in.dtype);
  torch::Tensor ws = byte_scratch(wb, hidden.device());
  const Lease w(op, hidden.device().index(), current_stream());
  DGS_CHECK_RC(dgs_linear_cross_entropy(in.hidden.t.data_ptr(), in.hidden.stride, in.weight.t.data_ptr(), in.weight.stride, in.dtype,
                                        in.target.data_ptr(), in.ids64, in.n, in.D, in.V, ignore_index, loss.data_ptr<float>(),
                                        lse.data_ptr<float>(), ws.data_ptr(), wb, w.status(), current_stream()));
  w.finish();
  return std::make_tuple(loss, lse);
}

// (dhidden, dweight); what is not wanted comes back with no elements.  loss: may be undefined
inline std::tuple<torch::Tensor, torch::Tensor> cross_entropy_backward(torch::Tensor grad_loss, const torch::Tensor& hidden,
                                                                       const torch::Tensor& weight, const torch::Tensor& target,
                                                                       torch::Tensor lse, torch::Tensor loss, int64_t ignore_index,
                                                                       bool want_hidden, bool want_weight) {
  const char* op = "_CAPI_linear_cross_entropy_backward";
  CrossEntropyInputs in = cross_entropy_inputs(op, hidden, weight, target);
  check_on(grad_loss, hidden.device(), op, "grad_loss");
  check_on(lse, hidden.device(), op, "lse");
  TORCH_CHECK(grad_loss.scalar_type() == torch::kFloat && lse.scalar_type() == torch::kFloat && grad_loss.dim() == 1 && lse.dim() == 1 &&
                  grad_loss.size(0) == in.n && lse.size(0) == in.n,
              op, ": grad_loss and lse must be float32 with one value for each row of hidden");
  if (loss.defined()) {
    check_on(loss, hidden.device(), op, "loss");
    TORCH_CHECK(loss.scalar_type() == torch::kFloat && loss.dim() == 1 && loss.size(0) == in.n, op,
                ": loss must be float32 with one value for each row of hidden");
    loss = loss.contiguous();
  }
  c10::cuda::CUDAGuard guard(hidden.device());
  lay_out(in, hidden, weight, target);
  grad_loss = grad_loss.contiguous();
  lse = lse.contiguous();
  torch::Tensor dh = device_empty({want_hidden ? in.n : 0, in.D}, hidden.scalar_type(), hidden.device());
  torch::Tensor dw = device_empty({want_weight ? in.V : 0, in.D}, hidden.scalar_type(), hidden.device());
  const size_t wb = want_hidden || want_weight ? dgs_linear_cross_entropy_backward_workspace_bytes(in.n, in.D, in.V, in.dtype) : 0;
  torch::Tensor ws = byte_scratch(wb, hidden.device());
  const Lease w(op, hidden.device().index(), current_stream());
  DGS_CHECK_RC(dgs_linear_cross_entropy_backward_from_loss(
      grad_loss.data_ptr<float>(), in.hidden.t.data_ptr(), in.hidden.stride, in.weight.t.data_ptr(), in.weight.stride, in.dtype,
      in.target.data_ptr(), in.ids64, lse.data_ptr<float>(), loss.defined() ? loss.data_ptr<float>() : nullptr, in.n, in.D, in.V, ignore_index,
      want_hidden ? dh.data_ptr() : nullptr, want_weight ? dw.data_ptr() : nullptr, ws.data_ptr(), wb, w.status(), current_stream()));
  w.finish();
  return std::make_tuple(dh, dw);
}
inline std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyBackwardCUDA(torch::Tensor grad_loss, torch::Tensor hidden,
                                                                               torch::Tensor weight, torch::Tensor target,
                                                                               torch::Tensor lse, int64_t ignore_index,
                                                                               bool want_hidden, bool want_weight) {
  return cross_entropy_backward(grad_loss, hidden, weight, target, lse, {}, ignore_index, want_hidden, want_weight);
}
// ... with the loss that the forward call gave beside lse
inline std::tuple<torch::Tensor, torch::Tensor> LinearCrossEntropyBackwardFromLossCUDA(torch::Tensor grad_loss, torch::Tensor hidden,
                                                                                       torch::Tensor weight, torch::Tensor target,
                                                                                       torch::Tensor lse, torch::Tensor loss,
                                                                                       int64_t ignore_index, bool want_hidden,
                                                                                       bool want_weight) {
  return cross_entropy_backward(grad_loss, hidden, weight, target, lse, loss, ignore_index, want_hidden, want_weight);
}

namespace {
// The list of one step.  `keep` holds gradients that had to be made contiguous, `written` what the step writes.
struct AdamWList {
  std::vector<dgs_adamw_tensor> tensors;
  std::vector<torch::Tensor> keep;
  std::vector<const torch::Tensor*> written;
  int64_t slots = 0;  // elements of all slots
};
inline AdamWList adamw_list(const char* op, const std::vector<torch::Tensor>& params,
                            const c10::List<c10::optional<torch::Tensor>>& grads, const std::vector<torch::Tensor>& copies,
                            const torch::Device& dev) {
  TORCH_CHECK(grads.size() == params.size(), op, ": ", params.size(), " parameters and ", grads.size(), " gradients");
  TORCH_CHECK(copies.empty() || copies.size() == params.size(), op, ": ", params.size(), " parameters and ", copies.size(), " copies");
  AdamWList list;
  list.tensors.reserve(params.size());
  list.written.reserve(2 * params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    const torch::Tensor& p = params[i];
    check_on(p, dev, op, "every parameter");
    TORCH_CHECK(p.is_contiguous(), op, ": parameter ", i, " is written in place and must be contiguous");
    dgs_adamw_tensor t;
    std::memset(&t, 0, sizeof(t));
    t.n = p.numel();
    t.at = list.slots;
    list.slots += dgs_adamw_slot_elems(t.n);
    t.param_dtype = training_dtype(p, op, "every parameter");
    if (!copies.empty()) {
      const torch::Tensor& c = copies[i];
      check_on(c, dev, op, "every copy");
      TORCH_CHECK(c.numel() == t.n && c.is_contiguous(), op, ": copy ", i, " must be contiguous and have its parameter's elements");
      t.copy = t.n ? c.data_ptr() : nullptr;
      t.copy_dtype = training_dtype(c, op, "every copy");
    }
    const c10::optional<torch::Tensor> g = grads.get(i);
    if (!g.has_value() || !g->defined() || t.n == 0) continue;  // no gradient: the tensor and its slot stay as they are
    check_on(*g, dev, op, "every gradient");
    TORCH_CHECK(g->numel() == t.n, op, ": gradient ", i, " must have its parameter's elements");
    t.grad_dtype = training_dtype(*g, op, "every gradient");
    if (g->is_contiguous()) {
      t.grad = g->data_ptr();
    } else {
      list.keep.push_back(g->contiguous());
      t.grad = list.keep.back().data_ptr();
    }
    t.param = p.data_ptr();
    list.tensors.push_back(t);
    list.written.push_back(&p);
    if (!copies.empty()) list.written.push_back(&copies[i]);
  }
  return list;
}
// The tensors were written behind torch's back: what autograd saved of them is out of date.  (Of those without a gradient it is not.)
inline void mark_written(const std::vector<const torch::Tensor*>& ts) {
  for (const torch::Tensor* t : ts)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
// No element may have two writers: they would race.  (A copy that is its own parameter has one, which writes the same value twice.)
class Written {
 public:
  explicit Written(size_t most) { spans_.reserve(most); }
  void add(const void* p, int64_t bytes) {
    if (bytes > 0) spans_.emplace_back(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes);
  }
  void check(const char* op) {
    std::sort(spans_.begin(), spans_.end());
    for (size_t i = 1; i < spans_.size(); ++i)
      TORCH_CHECK(spans_[i - 1].second <= spans_[i].first, op, ": parameters, copies and moments are written in place and must not overlap");
  }

 private:
  std::vector<std::pair<uintptr_t, uintptr_t>> spans_;
};
// moments: with the number of elements of each that the slots take
inline void check_written(const char* op, const AdamWList& list, std::initializer_list<std::pair<const torch::Tensor*, int64_t>> moments) {
  Written w(2 * list.tensors.size() + moments.size());
  for (const dgs_adamw_tensor& t : list.tensors) {
    const auto bytes = [&](int32_t dtype) { return t.n * (dtype == DGS_F32 ? 4 : 2); };
    w.add(t.param, bytes(t.param_dtype));
    if (t.copy != nullptr && !(t.copy == t.param && t.copy_dtype == t.param_dtype)) w.add(t.copy, bytes(t.copy_dtype));
  }
  for (const auto& [m, elems] : moments) w.add(m->data_ptr(), elems * m->element_size());
  w.check(op);
}
inline void check_moment(const torch::Tensor& t, torch::ScalarType type, int64_t elems, const torch::Device& dev, const char* op,
                         const char* what) {
  check_on(t, dev, op, what);
  TORCH_CHECK(t.scalar_type() == type && t.is_contiguous() && t.numel() >= elems, op, ": ", what, " must be contiguous, of type ", type,
              " and have at least ", elems, " elements");
}
}  // namespace

inline void AdamWStepCUDA(std::vector<torch::Tensor> params, c10::List<c10::optional<torch::Tensor>> grads,
                          std::vector<torch::Tensor> copies, torch::Tensor exp_avg, torch::Tensor exp_avg_sq, double lr, double beta1,
                          double beta2, double eps, double weight_decay, int64_t step) {
  const char* op = "_CAPI_adamw_step";
  CHECK_CUDA(exp_avg);
  c10::cuda::CUDAGuard guard(exp_avg.device());
  const AdamWList list = adamw_list(op, params, grads, copies, exp_avg.device());
  check_moment(exp_avg, torch::kFloat, list.slots, exp_avg.device(), op, "exp_avg");
  check_moment(exp_avg_sq, torch::kFloat, list.slots, exp_avg.device(), op, "exp_avg_sq");
  check_written(op, list, {{&exp_avg, list.slots}, {&exp_avg_sq, list.slots}});
  DGS_CHECK_RC(dgs_adamw_step(list.tensors.data(), static_cast<int32_t>(list.tensors.size()), exp_avg.data_ptr<float>(),
                              exp_avg_sq.data_ptr<float>(), lr, beta1, beta2, eps, weight_decay, step, current_stream()));
  mark_written(list.written);
}

namespace {
// seed: of codes rounded at random; null: the nearest codes
inline void adamw_step_8bit(const char* op, const std::vector<torch::Tensor>& params, const c10::List<c10::optional<torch::Tensor>>& grads,
                            const std::vector<torch::Tensor>& copies, const torch::Tensor& exp_avg, const torch::Tensor& exp_avg_scale,
                            const torch::Tensor& exp_avg_sq, const torch::Tensor& exp_avg_sq_scale, double lr, double beta1, double beta2,
                            double eps, double weight_decay, int64_t step, const int64_t* seed) {
  CHECK_CUDA(exp_avg);
  c10::cuda::CUDAGuard guard(exp_avg.device());
  const torch::Device dev = exp_avg.device();
  const AdamWList list = adamw_list(op, params, grads, copies, dev);
  const int64_t blocks = list.slots / dgs_adamw_slot_elems(1);
  check_moment(exp_avg, torch::kChar, list.slots, dev, op, "exp_avg");
  check_moment(exp_avg_sq, torch::kByte, list.slots, dev, op, "exp_avg_sq");
  check_moment(exp_avg_scale, torch::kFloat, blocks, dev, op, "exp_avg_scale");
  check_moment(exp_avg_sq_scale, torch::kFloat, blocks, dev, op, "exp_avg_sq_scale");
  check_written(op, list, {{&exp_avg, list.slots}, {&exp_avg_scale, blocks}, {&exp_avg_sq, list.slots}, {&exp_avg_sq_scale, blocks}});
  const dgs_adamw_tensor* ts = list.tensors.data();
  const int32_t count = static_cast<int32_t>(list.tensors.size());
  int8_t* m = exp_avg.data_ptr<int8_t>();
  uint8_t* v = exp_avg_sq.data_ptr<uint8_t>();
  float *ms = exp_avg_scale.data_ptr<float>(), *vs = exp_avg_sq_scale.data_ptr<float>();
  if (seed == nullptr)
    DGS_CHECK_RC(dgs_adamw_step_8bit(ts, count, m, ms, v, vs, lr, beta1, beta2, eps, weight_decay, step, current_stream()));
  else
    DGS_CHECK_RC(dgs_adamw_step_8bit_unbiased(ts, count, m, ms, v, vs, lr, beta1, beta2, eps, weight_decay, step,
                                              static_cast<uint64_t>(*seed), current_stream()));
  mark_written(list.written);
}
}  // namespace

inline void AdamWStep8bitCUDA(std::vector<torch::Tensor> params, c10::List<c10::optional<torch::Tensor>> grads,
                              std::vector<torch::Tensor> copies, torch::Tensor exp_avg, torch::Tensor exp_avg_scale,
                              torch::Tensor exp_avg_sq, torch::Tensor exp_avg_sq_scale, double lr, double beta1, double beta2, double eps,
                              double weight_decay, int64_t step) {
  adamw_step_8bit("_CAPI_adamw_step_8bit", params, grads, copies, exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale, lr, beta1, beta2,
                  eps, weight_decay, step, nullptr);
}
inline void AdamWStep8bitUnbiasedCUDA(std::vector<torch::Tensor> params, c10::List<c10::optional<torch::Tensor>> grads,
                                      std::vector<torch::Tensor> copies, torch::Tensor exp_avg, torch::Tensor exp_avg_scale,
                                      torch::Tensor exp_avg_sq, torch::Tensor exp_avg_sq_scale, double lr, double beta1, double beta2,
                                      double eps, double weight_decay, int64_t step, int64_t seed) {
  adamw_step_8bit("_CAPI_adamw_step_8bit.unbiased", params, grads, copies, exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale, lr, beta1,
                  beta2, eps, weight_decay, step, &seed);
}

inline torch::Tensor AdamWStateValuesCUDA(torch::Tensor codes, torch::Tensor scales) {
  const char* op = "_CAPI_adamw_state_values";
  CHECK_CUDA(codes);
  check_on(scales, codes.device(), op, "scales");
  TORCH_CHECK(codes.scalar_type() == torch::kChar || codes.scalar_type() == torch::kByte, op,
              ": codes must be int8 (first moments) or uint8 (second moments)");
  const int64_t block = dgs_adamw_slot_elems(1);
  TORCH_CHECK(codes.numel() % block == 0 && scales.scalar_type() == torch::kFloat && scales.numel() >= codes.numel() / block, op,
              ": whole blocks of ", block, " codes with a float32 scale each");
  c10::cuda::CUDAGuard guard(codes.device());
  codes = codes.contiguous();
  scales = scales.contiguous();
  torch::Tensor out = device_empty(codes.sizes(), torch::kFloat, codes.device());
  DGS_CHECK_RC(dgs_adamw_state_values(codes.data_ptr(), codes.scalar_type() == torch::kByte, scales.data_ptr<float>(), codes.numel(),
                                      out.data_ptr<float>(), current_stream()));
  return out;
}

}  // namespace dgs
