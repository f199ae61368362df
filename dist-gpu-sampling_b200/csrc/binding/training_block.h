// Operators of the blocks of a model on the batches that the samplers deliver: attention over packed sequences, the end of a block
// (norm, gate, residual, norm), rows kept for the backward pass in 8 bits.  Additions like those of training.h.
#pragma once
#include <c10/cuda/CUDAGraphsC10Utils.h>

#include <memory>

#include "training.h"

namespace dgs {

namespace {
// A status word for the call, or none while the stream is recorded (a replay has nobody to report to).
class CallStatus {
 public:
  CallStatus(const char* op, int device, cudaStream_t stream) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &st) != cudaSuccess) (void)cudaGetLastError();
    if (st == cudaStreamCaptureStatusNone) lease_ = std::make_unique<Lease>(op, device, stream);
  }
  int32_t* status() const { return lease_ ? lease_->status() : nullptr; }
  void finish() const {
    if (lease_) lease_->finish();
  }

 private:
  std::unique_ptr<Lease> lease_;
};

// ---- attention ----------------------------------------------------------------------------------------------------
// [n, heads, d] where its heads begin at 16-byte boundaries, else a copy with heads filled up with zeros (which change no score)
struct Heads {
  torch::Tensor t;
  int64_t row, head;
};
inline Heads as_heads(const torch::Tensor& t, int64_t width) {
  const int64_t vec = 16 / t.element_size();
  const auto whole = [&](int64_t dim) { return t.size(dim) <= 1 || (t.stride(dim) > 0 && t.stride(dim) % vec == 0); };
  if (t.size(2) == width && (t.stride(2) == 1 || width == 1) && whole(0) && whole(1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return {t, t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
  torch::Tensor c = device_empty({t.size(0), t.size(1), width}, t.scalar_type(), t.device());
  if (width != t.size(2)) c.narrow(2, t.size(2), width - t.size(2)).zero_();
  c.narrow(2, 0, t.size(2)).copy_(t);
  return {c, c.size(1) * width, width};
}

struct AttentionInputs {
  dgs_attention p;
  int64_t d, width;  // elements of a head, and as the kernels take them
  Heads q, k, v;
  torch::Tensor q_offsets, k_offsets;
};
inline void check_attention(const char* op, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                            const torch::Tensor& q_offsets, const torch::Tensor& k_offsets, double scale) {
  CHECK_CUDA(q);
  check_on(k, q.device(), op, "k");
  check_on(v, q.device(), op, "v");
  check_on(q_offsets, q.device(), op, "q_offsets");
  check_on(k_offsets, q.device(), op, "k_offsets");
  training_dtype(q, op, "q");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), op, ": q, k and v must share one type");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, op, ": q must be [rows, heads, d], k and v [rows, key heads, d]");
  TORCH_CHECK(k.sizes() == v.sizes(), op, ": k and v must have one shape");
  TORCH_CHECK(q.size(2) == k.size(2) && q.size(2) >= 1 && q.size(2) <= 128, op,
              ": the heads of q, k and v must have the same number of elements, 1 to 128, have ", q.size(2), " and ", k.size(2));
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0, op, ": the query heads must be a multiple of the key heads, are ",
              q.size(1), " and ", k.size(1));
  TORCH_CHECK(q_offsets.dim() == 1 && k_offsets.dim() == 1 && q_offsets.size(0) >= 1 && q_offsets.size(0) == k_offsets.size(0), op,
              ": q_offsets and k_offsets must hold where each sequence begins and where the last one ends");
  TORCH_CHECK(q_offsets.scalar_type() == k_offsets.scalar_type(), op, ": q_offsets and k_offsets must share one type");
  is_id64(q_offsets, "q_offsets");
  TORCH_CHECK(std::isfinite(scale), op, ": scale must be a finite number");
  TORCH_CHECK(q_offsets.size(0) <= INT32_MAX, op, ": too many sequences");
}
inline AttentionInputs attention_inputs(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& q_offsets,
                                        const torch::Tensor& k_offsets, bool causal, double scale, const char* op) {
  AttentionInputs in;
  const int64_t vec = 16 / q.element_size();
  in.d = q.size(2);
  in.width = (in.d + vec - 1) / vec * vec;
  in.q = as_heads(q, in.width);
  in.k = as_heads(k, in.width);
  in.v = as_heads(v, in.width);
  in.q_offsets = q_offsets.contiguous();
  in.k_offsets = k_offsets.contiguous();
  std::memset(&in.p, 0, sizeof(in.p));
  in.p.q = in.q.t.data_ptr();
  in.p.k = in.k.t.data_ptr();
  in.p.v = in.v.t.data_ptr();
  in.p.q_row = in.q.row;
  in.p.q_head = in.q.head;
  in.p.k_row = in.k.row;
  in.p.k_head = in.k.head;
  in.p.v_row = in.v.row;
  in.p.v_head = in.v.head;
  in.p.q_offsets = in.q_offsets.data_ptr();
  in.p.k_offsets = in.k_offsets.data_ptr();
  in.p.n_q = q.size(0);
  in.p.n_k = k.size(0);
  in.p.seqs = static_cast<int32_t>(q_offsets.size(0) - 1);
  in.p.heads = static_cast<int32_t>(q.size(1));
  in.p.kv_heads = static_cast<int32_t>(k.size(1));
  in.p.d = static_cast<int32_t>(in.width);
  in.p.dtype = training_dtype(q, op, "q");
  in.p.ids64 = is_id64(q_offsets, "q_offsets");
  in.p.causal = causal;
  in.p.scale = static_cast<float>(scale);
  return in;
}
// the first d elements of every head
inline torch::Tensor cut(const torch::Tensor& t, int64_t d) { return t.size(2) == d ? t : t.narrow(2, 0, d).contiguous(); }
}  // namespace

// (out [n_q, heads, d], lse [heads, n_q])
inline std::tuple<torch::Tensor, torch::Tensor> AttentionCUDA(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor q_offsets,
                                                              torch::Tensor k_offsets, bool causal, double scale) {
  const char* op = "_CAPI_attention";
  check_attention(op, q, k, v, q_offsets, k_offsets, scale);
  c10::cuda::CUDAGuard guard(q.device());
  const AttentionInputs in = attention_inputs(q, k, v, q_offsets, k_offsets, causal, scale, op);
  torch::Tensor out = device_empty({q.size(0), q.size(1), in.width}, q.scalar_type(), q.device());
  torch::Tensor lse = device_empty({q.size(1), q.size(0)}, torch::kFloat, q.device());
  const size_t wb = dgs_attention_workspace_bytes(&in.p, 0);
  torch::Tensor ws = byte_scratch(wb, q.device());
  const CallStatus w(op, q.device().index(), current_stream());
  DGS_CHECK_RC(dgs_attention_forward(&in.p, out.data_ptr(), lse.data_ptr<float>(), ws.data_ptr(), wb, w.status(), current_stream()));
  w.finish();
  return std::make_tuple(cut(out, in.d), lse);
}

// (dq, dk, dv); what is not wanted comes back with no rows
inline std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> AttentionBackwardCUDA(torch::Tensor grad, torch::Tensor q, torch::Tensor k,
                                                                                     torch::Tensor v, torch::Tensor out, torch::Tensor lse,
                                                                                     torch::Tensor q_offsets, torch::Tensor k_offsets,
                                                                                     bool causal, double scale, bool want_q, bool want_kv) {
  const char* op = "_CAPI_attention_backward";
  check_attention(op, q, k, v, q_offsets, k_offsets, scale);
  check_on(grad, q.device(), op, "grad");
  check_on(out, q.device(), op, "out");
  check_on(lse, q.device(), op, "lse");
  TORCH_CHECK(grad.sizes() == q.sizes() && grad.scalar_type() == q.scalar_type(), op, ": grad must have q's shape and type");
  TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && lse.scalar_type() == torch::kFloat && lse.dim() == 2 &&
                  lse.size(0) == q.size(1) && lse.size(1) == q.size(0),
              op, ": out and lse must be what _CAPI_attention returned for these inputs");
  c10::cuda::CUDAGuard guard(q.device());
  const AttentionInputs in = attention_inputs(q, k, v, q_offsets, k_offsets, causal, scale, op);
  const Heads g = as_heads(grad, in.width);
  Heads o = as_heads(out, in.width);
  o.t = o.t.contiguous();
  lse = lse.contiguous();
  torch::Tensor dq = device_empty({want_q ? q.size(0) : 0, q.size(1), in.width}, q.scalar_type(), q.device());
  torch::Tensor dk = device_empty({want_kv ? k.size(0) : 0, k.size(1), in.width}, q.scalar_type(), q.device());
  torch::Tensor dv = device_empty({want_kv ? k.size(0) : 0, k.size(1), in.width}, q.scalar_type(), q.device());
  if (want_q || want_kv) {
    const size_t wb = dgs_attention_workspace_bytes(&in.p, 1);
    torch::Tensor ws = byte_scratch(wb, q.device());
    const CallStatus w(op, q.device().index(), current_stream());
    // (an empty tensor has no address: what is wanted of no rows needs none)
    DGS_CHECK_RC(dgs_attention_backward(&in.p, g.t.data_ptr(), g.row, g.head, o.t.data_ptr(), lse.data_ptr<float>(),
                                        want_q ? dq.data_ptr() : nullptr, want_kv ? dk.data_ptr() : nullptr,
                                        want_kv ? dv.data_ptr() : nullptr, ws.data_ptr(), wb, w.status(), current_stream()));
    w.finish();
  }
  return std::make_tuple(cut(dq, in.d), cut(dk, in.d), cut(dv, in.d));
}

// ---- residual norm --------------------------------------------------------------------------------------------------
namespace {
inline int32_t norm_kind(const std::string& name, const char* op, const char* what) {
  if (name == "none") return DGS_NORM_NONE;
  if (name == "rms") return DGS_NORM_RMS;
  if (name == "layer") return DGS_NORM_LAYER;
  TORCH_CHECK(false, op, ": ", what, " must be 'none', 'rms' or 'layer', got '", name, "'");
}

struct ResidualNorm {
  dgs_residual_norm p;
  int64_t n, D;
  torch::ScalarType ptype;
  std::vector<torch::Tensor> keep;
};
// what both directions check and lay out; like: gives shape and type of the rows
inline ResidualNorm residual_norm(const char* op, const torch::Tensor& like, const torch::Tensor& y, const c10::optional<torch::Tensor>& gate,
                                  const std::string& post, const c10::optional<torch::Tensor>& post_weight,
                                  const c10::optional<torch::Tensor>& post_bias, const std::string& pre,
                                  const c10::optional<torch::Tensor>& weight, const c10::optional<torch::Tensor>& bias, double x_scale,
                                  double y_scale, double eps) {
  CHECK_CUDA(like);
  check_on(y, like.device(), op, "y");
  TORCH_CHECK(like.dim() >= 1 && like.size(-1) >= 1, op, ": rows must have at least one element");
  TORCH_CHECK(y.sizes() == like.sizes() && y.scalar_type() == like.scalar_type(), op, ": x and y must have one shape and type");
  ResidualNorm r;
  std::memset(&r.p, 0, sizeof(r.p));
  r.D = like.size(-1);
  r.n = like.numel() / r.D;
  r.p.n = r.n;
  r.p.D = r.D;
  r.p.dtype = training_dtype(like, op, "x");
  TORCH_CHECK(r.D <= 8192, op, ": rows of at most 8192 elements, have ", r.D);
  r.p.post = norm_kind(post, op, "post");
  r.p.pre = norm_kind(pre, op, "pre");
  r.p.x_scale = static_cast<float>(x_scale);
  r.p.y_scale = static_cast<float>(y_scale);
  r.p.eps = static_cast<float>(eps);
  r.ptype = like.scalar_type();
  bool typed = false;
  const auto param = [&](const c10::optional<torch::Tensor>& t, const char* what, bool allowed) -> const void* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(allowed, op, ": ", what, " without its norm");
    check_on(*t, like.device(), op, what);
    training_dtype(*t, op, what);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == r.D, op, ": ", what, " must have the ", r.D, " elements of a row");
    TORCH_CHECK(!typed || t->scalar_type() == r.ptype, op, ": weights, biases and a gate of the columns must share one type");
    typed = true;
    r.ptype = t->scalar_type();
    r.keep.push_back(t->contiguous());
    return r.keep.back().data_ptr();
  };
  r.p.post_weight = param(post_weight, "post_weight", r.p.post != DGS_NORM_NONE);
  r.p.post_bias = param(post_bias, "post_bias", r.p.post != DGS_NORM_NONE);
  r.p.weight = param(weight, "weight", r.p.pre != DGS_NORM_NONE);
  r.p.bias = param(bias, "bias", r.p.pre != DGS_NORM_NONE);
  TORCH_CHECK(r.p.post_bias == nullptr || r.p.post_weight != nullptr, op, ": a bias needs a weight");
  TORCH_CHECK(r.p.bias == nullptr || r.p.weight != nullptr, op, ": a bias needs a weight");
  const Rows rows = as_rows(y, r.D);
  r.keep.push_back(rows.t);
  r.p.y = rows.t.data_ptr();
  r.p.y_stride = rows.stride;
  if (gate.has_value()) {
    check_on(*gate, like.device(), op, "gate");
    if (gate->sizes() == like.sizes() && like.dim() >= 2) {
      TORCH_CHECK(gate->scalar_type() == like.scalar_type(), op, ": a gate of each element must have the type of x");
      const Rows g = as_rows(*gate, r.D);
      r.keep.push_back(g.t);
      r.p.gate_kind = DGS_GATE_ELEMENT;
      r.p.gate = g.t.data_ptr();
      r.p.gate_stride = g.stride;
    } else if (gate->dim() == 1 && gate->size(0) == r.D) {
      r.p.gate = param(gate, "gate", true);
      r.p.gate_kind = DGS_GATE_COLUMN;
    } else {
      TORCH_CHECK(gate->dim() == like.dim() && gate->size(-1) == 1 && gate->numel() == r.n &&
                      gate->sizes().slice(0, like.dim() - 1) == like.sizes().slice(0, like.dim() - 1),
                  op, ": the gate must have a value for each column [", r.D, "], for each row [..., 1] or for each element");
      TORCH_CHECK(gate->scalar_type() == like.scalar_type(), op, ": a gate of each row must have the type of x");
      r.keep.push_back(gate->contiguous());
      r.p.gate_kind = DGS_GATE_ROW;
      r.p.gate = r.keep.back().data_ptr();
    }
  }
  r.p.param_dtype = r.ptype == torch::kFloat ? DGS_F32 : r.ptype == torch::kBFloat16 ? DGS_BF16 : DGS_F16;
  return r;
}
}  // namespace

// (sum, out, post_mean, post_rstd, mean, rstd); what is absent has no elements
inline std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> ResidualNormCUDA(
    torch::Tensor x, torch::Tensor y, c10::optional<torch::Tensor> gate, std::string post, c10::optional<torch::Tensor> post_weight,
    c10::optional<torch::Tensor> post_bias, std::string pre, c10::optional<torch::Tensor> weight, c10::optional<torch::Tensor> bias,
    double x_scale, double y_scale, double eps) {
  const char* op = "_CAPI_residual_norm";
  CHECK_CUDA(x);
  c10::cuda::CUDAGuard guard(x.device());
  const ResidualNorm r = residual_norm(op, x, y, gate, post, post_weight, post_bias, pre, weight, bias, x_scale, y_scale, eps);
  const Rows rows = as_rows(x, r.D);
  const auto stats = [&](bool there) { return device_empty({there ? r.n : 0}, torch::kFloat, x.device()); };
  torch::Tensor sum = device_empty(x.sizes(), x.scalar_type(), x.device());
  torch::Tensor out = r.p.pre != DGS_NORM_NONE ? device_empty(x.sizes(), x.scalar_type(), x.device())
                                               : device_empty({0}, x.scalar_type(), x.device());
  torch::Tensor pm = stats(r.p.post == DGS_NORM_LAYER), pr = stats(r.p.post != DGS_NORM_NONE);
  torch::Tensor m = stats(r.p.pre == DGS_NORM_LAYER), s = stats(r.p.pre != DGS_NORM_NONE);
  DGS_CHECK_RC(dgs_residual_norm_forward(&r.p, rows.t.data_ptr(), rows.stride, sum.data_ptr(), out.data_ptr(), pm.data_ptr<float>(),
                                         pr.data_ptr<float>(), m.data_ptr<float>(), s.data_ptr<float>(), current_stream()));
  return std::make_tuple(sum, out, pm, pr, m, s);
}

// (dx, dy, dgate, dpost_weight, dpost_bias, dweight, dbias); the gradient of what is absent has no elements.  post_bias is needed for the
// gate's gradient
inline std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
ResidualNormBackwardCUDA(c10::optional<torch::Tensor> grad_sum, c10::optional<torch::Tensor> grad_out, torch::Tensor sum, torch::Tensor y,
                         c10::optional<torch::Tensor> gate, std::string post, c10::optional<torch::Tensor> post_weight,
                         c10::optional<torch::Tensor> post_bias, std::string pre, c10::optional<torch::Tensor> weight,
                         torch::Tensor post_mean, torch::Tensor post_rstd, torch::Tensor mean, torch::Tensor rstd, double x_scale,
                         double y_scale) {
  const char* op = "_CAPI_residual_norm_backward";
  CHECK_CUDA(sum);
  c10::cuda::CUDAGuard guard(sum.device());
  const ResidualNorm r = residual_norm(op, sum, y, gate, post, post_weight, post_bias, pre, weight, {}, x_scale, y_scale, 0.0);
  const auto stats = [&](torch::Tensor& t, bool there, const char* what) {
    check_on(t, sum.device(), op, what);
    TORCH_CHECK(t.scalar_type() == torch::kFloat && t.numel() == (there ? r.n : 0), op, ": ", what, " must be what _CAPI_residual_norm returned");
    t = t.contiguous();
    return t.data_ptr<float>();
  };
  const float* pm = stats(post_mean, r.p.post == DGS_NORM_LAYER, "post_mean");
  const float* pr = stats(post_rstd, r.p.post != DGS_NORM_NONE, "post_rstd");
  const float* m = stats(mean, r.p.pre == DGS_NORM_LAYER, "mean");
  const float* s = stats(rstd, r.p.pre != DGS_NORM_NONE, "rstd");
  Rows ds{{}, 0}, dout{{}, 0};
  const auto grad = [&](const c10::optional<torch::Tensor>& t, const char* what) -> Rows {
    if (!t.has_value()) return {{}, 0};
    check_on(*t, sum.device(), op, what);
    TORCH_CHECK(t->sizes() == sum.sizes() && t->scalar_type() == sum.scalar_type(), op, ": ", what, " must have the shape and type of sum");
    return as_rows(*t, r.D);
  };
  TORCH_CHECK(!grad_out.has_value() || r.p.pre != DGS_NORM_NONE, op, ": a gradient of out without its norm");
  ds = grad(grad_sum, "grad_sum");
  dout = grad(grad_out, "grad_out");
  sum = sum.contiguous();
  const auto device = sum.device();
  const auto none = [&](torch::ScalarType t) { return device_empty({0}, t, device); };
  const auto like = [&](bool there) { return there ? device_empty({r.D}, r.ptype, device) : none(r.ptype); };
  torch::Tensor dx = device_empty(sum.sizes(), sum.scalar_type(), device), dy = device_empty(sum.sizes(), sum.scalar_type(), device);
  torch::Tensor dg = gate.has_value() ? device_empty(gate->sizes(), gate->scalar_type(), device) : none(sum.scalar_type());
  torch::Tensor dpw = like(r.p.post_weight != nullptr), dpb = like(r.p.post_weight != nullptr);
  torch::Tensor dw = like(r.p.weight != nullptr), db = like(r.p.weight != nullptr);
  const size_t wb = dgs_residual_norm_backward_workspace_bytes(r.n, r.D);
  torch::Tensor ws = byte_scratch(wb, device);
  DGS_CHECK_RC(dgs_residual_norm_backward(
      &r.p, sum.data_ptr(), ds.t.defined() ? ds.t.data_ptr() : nullptr, ds.stride, dout.t.defined() ? dout.t.data_ptr() : nullptr, dout.stride,
      pm, pr, m, s, dx.data_ptr(), dy.data_ptr(), gate.has_value() ? dg.data_ptr() : nullptr, r.p.post_weight ? dpw.data_ptr() : nullptr,
      r.p.post_weight ? dpb.data_ptr() : nullptr, r.p.weight ? dw.data_ptr() : nullptr, r.p.weight ? db.data_ptr() : nullptr, ws.data_ptr(), wb,
      current_stream()));
  return std::make_tuple(dx, dy, dg, dpw, dpb, dw, db);
}

// ---- rows kept in 8 bits --------------------------------------------------------------------------------------------
// (codes [n, D] int8, scales [n, ceil(D / 128)] float32)
inline std::tuple<torch::Tensor, torch::Tensor> Keep8bitCUDA(torch::Tensor x) {
  const char* op = "_CAPI_keep_8bit";
  CHECK_CUDA(x);
  TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, op, ": x must be rows of at least one element");
  const int32_t dtype = training_dtype(x, op, "x");
  const int64_t n = x.size(0), D = x.size(1);
  c10::cuda::CUDAGuard guard(x.device());
  const Rows r = as_rows(x, D);
  torch::Tensor codes = device_empty({n, D}, torch::kChar, x.device());
  torch::Tensor scales = device_empty({n, (D + 127) / 128}, torch::kFloat, x.device());
  DGS_CHECK_RC(dgs_keep_8bit(r.t.data_ptr(), r.stride, dtype, n, D, n ? codes.data_ptr<int8_t>() : nullptr,
                             n ? scales.data_ptr<float>() : nullptr, current_stream()));
  return std::make_tuple(codes, scales);
}

namespace {
inline Rows check_kept(const char* op, const torch::Tensor& codes, torch::Tensor& scales) {
  CHECK_CUDA(codes);
  check_on(scales, codes.device(), op, "scales");
  TORCH_CHECK(codes.dim() == 2 && codes.size(1) >= 1 && codes.scalar_type() == torch::kChar, op, ": codes must be int8 rows");
  TORCH_CHECK(scales.scalar_type() == torch::kFloat && scales.dim() == 2 && scales.size(0) == codes.size(0) &&
                  scales.size(1) == (codes.size(1) + 127) / 128,
              op, ": scales must be float32 with one for every 128 codes of a row");
  scales = scales.contiguous();
  return as_rows(codes, codes.size(1));
}
}  // namespace

inline torch::Tensor Kept8bitValuesCUDA(torch::Tensor codes, torch::Tensor scales, int64_t dtype) {
  const char* op = "_CAPI_kept_8bit_values";
  CHECK_CUDA(codes);
  c10::cuda::CUDAGuard guard(codes.device());
  const Rows c = check_kept(op, codes, scales);
  const auto type = static_cast<torch::ScalarType>(dtype);
  TORCH_CHECK(type == torch::kFloat || type == torch::kBFloat16 || type == torch::kHalf, op, ": the type must be float32, bfloat16 or float16");
  torch::Tensor out = device_empty(codes.sizes(), type, codes.device());
  DGS_CHECK_RC(dgs_kept_8bit_values(c.t.data_ptr<int8_t>(), c.stride, scales.data_ptr<float>(), codes.size(0), codes.size(1),
                                    training_dtype(out, op, "the result"), out.data_ptr(), current_stream()));
  return out;
}

// (dweight [O, D], dbias [O]); a bias that is not wanted has no elements
inline std::tuple<torch::Tensor, torch::Tensor> Kept8bitWeightGradCUDA(torch::Tensor grad, torch::Tensor codes, torch::Tensor scales,
                                                                       bool want_bias) {
  const char* op = "_CAPI_kept_8bit_weight_grad";
  CHECK_CUDA(codes);
  c10::cuda::CUDAGuard guard(codes.device());
  const Rows c = check_kept(op, codes, scales);
  check_on(grad, codes.device(), op, "grad");
  TORCH_CHECK(grad.dim() == 2 && grad.size(0) == codes.size(0) && grad.size(1) >= 1, op, ": grad must have one row for each row of codes");
  const int32_t dtype = training_dtype(grad, op, "grad");
  const int64_t n = codes.size(0), D = codes.size(1), O = grad.size(1);
  const Rows g = as_rows(grad, O);
  torch::Tensor dw = device_empty({O, D}, grad.scalar_type(), grad.device());
  torch::Tensor db = device_empty({want_bias ? O : 0}, grad.scalar_type(), grad.device());
  const size_t wb = dgs_kept_8bit_weight_grad_workspace_bytes(n, O, D, dtype);
  torch::Tensor ws = byte_scratch(wb, grad.device());
  const CallStatus w(op, grad.device().index(), current_stream());
  DGS_CHECK_RC(dgs_kept_8bit_weight_grad_reported(g.t.data_ptr(), g.stride, dtype, c.t.data_ptr<int8_t>(), c.stride, scales.data_ptr<float>(), n,
                                                  O, D, dw.data_ptr(), want_bias ? db.data_ptr() : nullptr, ws.data_ptr(), wb, w.status(),
                                                  current_stream()));
  w.finish();
  return std::make_tuple(dw, db);
}

}  // namespace dgs
