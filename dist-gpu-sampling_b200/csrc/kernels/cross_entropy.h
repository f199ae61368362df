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
// the busiest slot.  More than one slice only while that gives a slot no more than kMostRounds of them, which also bounds what
// the slices' results take.
constexpr int64_t kMostRounds = 8;
inline int64_t slices_for(int64_t rows, int64_t cols, int64_t slots) {
  // (in 32 bits and with one division a candidate: this is worked out on every call)
  if (rows > kMostRounds * slots) return 1;
  const uint32_t r = static_cast<uint32_t>(rows), c = static_cast<uint32_t>(cols), most = static_cast<uint32_t>(cols < slots ? cols : slots);
  uint32_t best = 1, rounds = 0, room = 0;  // rounds = tiles(r * s, slots), room = rounds * slots - r * s
  uint64_t least = UINT64_MAX;
  for (uint32_t s = 1; s <= most && (s == 1 || r * s <= kMostRounds * slots); ++s) {
    while (room < r) {
      room += static_cast<uint32_t>(slots);
      ++rounds;
    }
    room -= r;
    const uint64_t cost = static_cast<uint64_t>(rounds) * ((c + s - 1) / s);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// The rows that count, as cross_entropy.cu packs them.  Packed row c holds what the products read: the hidden row, its target
// as a 32-bit word (-1: none), and for the backward pass dloss, lse and, where the loss is given, the target's entry p - 1.  Either row c is row c of the call (rows without a valid
// target: zeros, word -1), or (compact) the rows with a valid target alone, in their order; then slot[i] is row i's place among
// them (-1: none), live[0] their number, live[1] the slices for that many rows in blocks of block_rows, and the packed rows from
// there to the end of the block (the first one, where there is no row) are zeros.
struct CePacked {
  void* rows;
  int64_t pitch;
  int32_t* word;
  float *dloss, *lse;      // null in the forward pass
  float* hit;              // p - 1 at the target; null where the loss is not given
  float* largest;          // [ce_pack_ctas(n)] largest finite |dloss| among a CTA's rows; may be null
  bool compact;
  int32_t *slot, *live;
  int32_t block_rows, col_tiles, slots;  // what slices_for takes
  int32_t* counts;         // [tiles(n, CE_COUNT_ROWS)], scratch
};
constexpr int CE_PACK_ROWS = 16, CE_COUNT_ROWS = 1024;
inline int64_t ce_pack_ctas(int64_t n) { return tiles(n, CE_PACK_ROWS); }

// cross_entropy.cu
int ce_pack(const CeProblem& q, const CePacked& p, const float* dloss, const float* lse, const float* loss, cudaStream_t s);
// loss and lse from (maximum, sum) pairs of each packed row, [row][slices][groups].  live, slot: those of compact rows, or null.
// word: that of packed rows; null: rows are those of the call, and the targets are looked at here.
int ce_join(const CeProblem& q, const float* top, const float* total, int64_t groups, int64_t slices, const int32_t* live,
            const int32_t* word, const int32_t* slot, const float* target_logit, float* loss, float* lse, cudaStream_t s);
// out[n][D] = the sums of parts[splits][rows][pitch]; slot as above or null
int ce_sum(const float* parts, int64_t splits, int64_t n, int64_t D, int64_t rows, int64_t pitch, const int32_t* slot, void* out,
           int32_t dtype, cudaStream_t s);

// cross_entropy_mma.cu
size_t ce_mma_forward_bytes(int64_t n, int64_t D, int64_t V);
size_t ce_mma_backward_bytes(int64_t n, int64_t D, int64_t V);
int ce_mma_forward(const CeProblem& q, float* loss, float* lse, cudaStream_t s);
int ce_mma_backward(const CeProblem& q, const float* dloss, const float* lse, const float* loss, void* dhidden, void* dweight, cudaStream_t s);

#ifdef __CUDACC__
// a row's target as a word, -1 where it is ignored or no class
__device__ __forceinline__ int32_t target_word(const void* target, bool ids64, int64_t row, int64_t V, int64_t ignore_index, bool* wrong) {
  const int64_t t = ids64 ? static_cast<const int64_t*>(target)[row] : static_cast<int64_t>(static_cast<const int32_t*>(target)[row]);
  const bool in = t >= 0 && t < V;
  *wrong = !in && t != ignore_index;
  return in && t != ignore_index ? static_cast<int32_t>(t) : -1;
}
#endif

}  // namespace dgs
