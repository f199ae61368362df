// What the two forms of the cross entropy share: 32-bit operands on the CUDA cores (cross_entropy.cu), 16-bit operands on the
// tensor cores (cross_entropy_mma.cu).
#pragma once
#include "train_common.cuh"

namespace dgs {

struct CeProblem {
  const void* hidden;
  int64_t hidden_stride;
  const void* weight;
  int64_t weight_stride;
  int32_t dtype;
  const void* target;
  bool ids64;
  int64_t n, D, V, ignore_index;
  char* ws;
  int32_t* status;
};

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline int64_t tiles(int64_t v, int64_t per) { return (v + per - 1) / per; }

// Parts of a workspace, 256-byte aligned
struct Layout {
  size_t bytes = 0;
  size_t take(int64_t count) {
    const size_t here = bytes;
    bytes += static_cast<size_t>(up(count, 256));
    return here;
  }
};

// Slices of `cols` column tiles for `rows` row blocks on `slots` CTAs that run at once: the cut with the fewest tiles in
// the busiest slot.
inline int64_t slices_for(int64_t rows, int64_t cols, int64_t slots) {
  int64_t best = 1, least = tiles(rows, slots) * cols;
  for (int64_t s = 2; s <= cols && s <= slots; ++s) {
    const int64_t cost = tiles(rows * s, slots) * tiles(cols, s);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// cross_entropy.cu: rows with a valid target, packed `pitch` elements apart (zero where there is none), the targets as 32-bit
// words (-1: none); target_logit (may be null) is cleared.
int ce_pack(const CeProblem& q, void* packed, int64_t pitch, int32_t* word, float* target_logit, cudaStream_t s);
// loss and lse from `parts` (maximum, sum) pairs a row: top, total [parts][n]
int ce_join(const CeProblem& q, const float* top, const float* total, int64_t parts, const int32_t* word, const float* target_logit,
            float* loss, float* lse, cudaStream_t s);
// out[n][D] of `dtype` = the sum of parts[splits][rows][pitch], rows >= n
int ce_sum(const float* parts, int64_t splits, int64_t n, int64_t D, int64_t rows, int64_t pitch, void* out, int32_t dtype, cudaStream_t s);

// cross_entropy_mma.cu
size_t ce_mma_forward_bytes(int64_t n, int64_t D, int64_t V);
size_t ce_mma_backward_bytes(int64_t n, int64_t D, int64_t V);
int ce_mma_forward(const CeProblem& q, float* loss, float* lse, cudaStream_t s);
int ce_mma_backward(const CeProblem& q, const float* dloss, const float* lse, void* dhidden, void* dweight, cudaStream_t s);

}  // namespace dgs
