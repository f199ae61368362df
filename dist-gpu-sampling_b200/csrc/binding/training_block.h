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
  const auto whole = [&](int64_t dim) { return t.size(dim) <= 1 || (t.stride(dim) >= 0 && t.stride(dim) % vec == 0); };
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

}  // namespace dgs
