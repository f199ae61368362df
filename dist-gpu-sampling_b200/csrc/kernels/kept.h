// What the kernels of rows kept in 8 bits share (kept.cu: codes, values, entry points; kept_mma.cu: the weight's gradient on the tensor cores).  Not part of the C ABI.
#pragma once
#include "train_common.cuh"

namespace dgs {

constexpr int KEPT_GROUP = 128;  // elements of a row that share a scale

struct KeptGradArgs {
  const void* grad;
  int64_t grad_stride;
  const int8_t* codes;
  int64_t codes_stride;
  const float* scales;
  int64_t n;
  int32_t O, D, groups, splits;
  float *parts, *bias_parts;  // [splits][O][D], [splits][O]
  void *dweight, *dbias;
  int32_t* status;
  uint64_t wait_limit;  // of a wait, in nanoseconds
};

// kept_mma.cu: 16-bit gradients on the tensor cores; one share writes the results, several leave parts to be added
int64_t kept_mma_shares(int64_t n, int64_t O, int64_t D);
int kept_mma_weight_grad(const KeptGradArgs& a, int32_t dtype, cudaStream_t s);

}  // namespace dgs
