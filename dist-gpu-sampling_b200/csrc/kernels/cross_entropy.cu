// Softmax cross entropy of hidden rows against a weight row per class, the logits never all held, with its gradients.
//
//   s_iv = h_i . W_v,  lse_i = log sum_v exp(s_iv),  loss_i = lse_i - s_i,t(i)
//   G_iv = dloss_i (exp(s_iv - lse_i) - [v = t(i)]),  dh = G W,  dW = G^T h
//
// At the target exp(s - lse) - 1 = expm1(-loss).  lse is a sum in 32 bits, off by 2^-25 of itself: of a row that is nearly right,
// with a loss of 1e-4 at logits of 100, the difference to one would be off by some percent, the loss is not.  Where it is given to
// the backward pass that entry comes from it.
//
// Forward: a block of rows meets the vocabulary tile by tile; each row carries a running maximum and a running sum of
// exponentials, so a tile of logits lives in registers only.  The vocabulary is cut into slices where there are fewer row
// blocks than SMs; a last launch joins the slices' (maximum, sum) pairs in their order (16-bit operands whose row blocks meet
// all classes at once join theirs on the spot).
// Backward: the vocabulary is taken in pieces.  Per piece the logits are computed again, leave as G into a buffer of 96 MB
// (256 MB in 16 bits), and two products read it: dh grows in 32 bits over the pieces, dW's rows of the piece are
// complete.  That is 8 n V D operations for a training step instead of 6 with the logits kept (n V values, 2.1 GB at
// 8 192 rows and 65 537 classes).
//
// This file: the entry points, the launches around the products, and the products of 32-bit operands on the CUDA cores (fused
// multiply-adds in 32 bits, which the tensor cores do not have): bound by their rate, 33 TFLOP/s forward and 26 backward at
// 4 096 rows of 256 against 30 000 classes (a library product of those sizes: 56).  16-bit operands: cross_entropy_mma.cu.
//
// A first launch copies the hidden rows into packed rows and the targets into 32-bit words: rows without a valid target
// become zero there, so that what stands in an ignored row (an infinity, say) reaches neither dh nor dW, and alignment
// and strides no longer matter.
#include "cross_entropy.h"

namespace dgs {
namespace {

constexpr int CE_ROWS = 128;            // rows of a tile
constexpr int CE_COLS = 128;            // classes of a tile
constexpr int CE_K = 16;
constexpr int CE_THREADS = 256;
constexpr int64_t CE_PIECE_BYTES = int64_t(96) << 20;  // of G: what L2 (126 MB) holds beside the operands

// ---- packing -----------------------------------------------------------------------------------------------------
struct PackArgs {
  const void* hidden;
  int64_t stride;
  const void* target;
  int32_t ids64, vectors;  // vectors: rows are moved 16 bytes at a time
  int64_t n, V, ignore_index;
  int32_t D, pitch;
  CePacked to;
  const float *dloss, *lse, *loss;
  int32_t* status;
};

// Rows with a valid target in each CE_COUNT_ROWS
__global__ void __launch_bounds__(CE_THREADS) ce_count_kernel(const __grid_constant__ PackArgs a) {
  pdl_enter();
  int mine = 0;
#pragma unroll
  for (int k = 0; k < CE_COUNT_ROWS / CE_THREADS; ++k) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * CE_COUNT_ROWS + k * CE_THREADS + threadIdx.x;
    bool wrong;
    if (row < a.n) mine += target_word(a.target, a.ids64, row, a.V, a.ignore_index, &wrong) >= 0;
  }
  __shared__ int sums[CE_THREADS / 32];
  mine = __reduce_add_sync(FULL_MASK, mine);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    int s = 0;
    for (int w = 0; w < CE_THREADS / 32; ++w) s += sums[w];
    a.to.counts[blockIdx.x] = s;
  }
}

__device__ __forceinline__ int cta_sum_int(int v, int* smem) {
  v = __reduce_add_sync(FULL_MASK, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < CE_THREADS / 32; ++w) s += smem[w];
  return s;
}

// A warp moves two rows.  Compact: a CTA's rows go behind all valid rows before them, counted from the chunks' numbers and the
// targets of its own chunk.
template <typename T>
__global__ void __launch_bounds__(CE_THREADS) ce_pack_kernel(const __grid_constant__ PackArgs a) {
  constexpr int VEC = 16 / sizeof(T), WARPS = CE_THREADS / 32;
  __shared__ int sums[WARPS];
  __shared__ int32_t words[CE_PACK_ROWS];
  __shared__ float peak[WARPS];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * CE_PACK_ROWS;
  if (threadIdx.x < CE_PACK_ROWS && row0 + threadIdx.x < a.n) {
    bool wrong;
    words[threadIdx.x] = target_word(a.target, a.ids64, row0 + threadIdx.x, a.V, a.ignore_index, &wrong);
    if (wrong) raise_status(a.status, DGS_ERR_RANGE);
  }
  int before = 0, live = 0;
  if (a.to.compact) {
    const int64_t chunk = row0 / CE_COUNT_ROWS, chunks = (a.n + CE_COUNT_ROWS - 1) / CE_COUNT_ROWS;
    for (int64_t c = threadIdx.x; c < chunks; c += CE_THREADS) {
      const int k = a.to.counts[c];
      live += k;
      if (c < chunk) before += k;
    }
    for (int64_t r = chunk * CE_COUNT_ROWS + threadIdx.x; r < row0; r += CE_THREADS) {
      bool wrong;
      before += target_word(a.target, a.ids64, r, a.V, a.ignore_index, &wrong) >= 0;
    }
    before = cta_sum_int(before, sums);
    live = cta_sum_int(live, sums);
  }
  __syncthreads();
  float most = 0.0f;
#pragma unroll
  for (int k = 0; k < CE_PACK_ROWS / WARPS; ++k) {
    const int i = warp * (CE_PACK_ROWS / WARPS) + k;
    const int64_t row = row0 + i;
    if (row >= a.n) break;
    const int32_t word = words[i];
    int64_t to = row;
    if (a.to.compact) {
      int ahead = 0;
      for (int j = 0; j < i; ++j) ahead += words[j] >= 0;
      to = word >= 0 ? before + ahead : -1;
      if (lane == 0) a.to.slot[row] = static_cast<int32_t>(to);
      if (to < 0) continue;
    }
    if (lane == 0) {
      a.to.word[to] = word;
      if (a.to.dloss != nullptr) {
        const float d = word >= 0 ? a.dloss[row] : 0.0f;
        a.to.dloss[to] = d;
        a.to.lse[to] = word >= 0 ? a.lse[row] : 0.0f;
        if (a.to.hit != nullptr) a.to.hit[to] = word >= 0 ? expm1f(-a.loss[row]) : 0.0f;
        if (fabsf(d) < INFINITY) most = fmaxf(most, fabsf(d));  // (an infinite one would leave nothing of the others)
      }
    }
    const T* from = static_cast<const T*>(a.hidden) + row * a.stride;
    T* dst = static_cast<T*>(a.to.rows) + to * a.pitch;
    if (a.vectors) {
      for (int j0 = lane * VEC; j0 < a.pitch; j0 += 4 * 32 * VEC) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + u * 32 * VEC;
          v[u] = word >= 0 && j < a.pitch ? *reinterpret_cast<const uint4*>(from + j) : uint4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + u * 32 * VEC;
          if (j < a.pitch) *reinterpret_cast<uint4*>(dst + j) = v[u];
        }
      }
    } else {
      for (int j0 = lane; j0 < a.pitch; j0 += 8 * 32) {
        T v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = word >= 0 && j0 + u * 32 < a.D ? from[j0 + u * 32] : from_float<T>(0.0f);
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (j0 + u * 32 < a.pitch) dst[j0 + u * 32] = v[u];
      }
    }
  }
  if (a.to.largest != nullptr) {
    if (lane == 0) peak[warp] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < WARPS; ++w) most = fmaxf(most, peak[w]);
      a.to.largest[blockIdx.x] = most;
    }
  }
  if (a.to.compact && blockIdx.x == gridDim.x - 1) {
    if (warp == 0) {  // slices_for, a lane for every 32nd number of slices: fewest tiles in the busiest slot, then fewest slices
      const int blocks = live > 0 ? (live + a.to.block_rows - 1) / a.to.block_rows : 1;
      unsigned long long best = ~0ull;
      for (int k = 1 + lane; k <= a.to.col_tiles && k <= a.to.slots && (k == 1 || int64_t(blocks) * k <= kMostRounds * a.to.slots); k += 32) {
        const unsigned long long rounds = (static_cast<unsigned long long>(blocks) * k + a.to.slots - 1) / a.to.slots;
        const unsigned long long cost = (rounds * ((a.to.col_tiles + k - 1) / k)) << 10 | k;
        best = cost < best ? cost : best;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(FULL_MASK, best, o);
        best = other < best ? other : best;
      }
      if (lane == 0) {
        a.to.live[0] = live;
        a.to.live[1] = static_cast<int32_t>(best & 1023);
      }
    }
  }
  if (a.to.compact) {  // zeros to the end of the last block, for the products' sake and because what lay there may be no numbers
    int64_t end = (static_cast<int64_t>(live) + a.to.block_rows - 1) / a.to.block_rows * a.to.block_rows;
    if (end == 0) end = a.to.block_rows;
    if (end > a.n) end = a.n;
    for (int64_t r = live + static_cast<int64_t>(blockIdx.x) * WARPS + warp; r < end; r += static_cast<int64_t>(gridDim.x) * WARPS) {
      T* dst = static_cast<T*>(a.to.rows) + r * a.pitch;
      for (int j = lane; j < a.pitch; j += 32) dst[j] = from_float<T>(0.0f);
    }
  }
}

// ---- products on the CUDA cores ------------------------------------------------------------------------------------
// A tile of CE_ROWS x CE_COLS, eight by eight values a thread, operands staged through shared memory CE_K at a time.
// KMAJOR: element (r, k) at p[r * stride + k]; else at p[k * stride + r].
template <bool KMAJOR>
struct Operand {
  const float* p;
  int64_t stride;
  int64_t rows;
  __device__ __forceinline__ float at(int64_t r, int64_t k, int64_t k_end) const {
    if (r >= rows || k >= k_end) return 0.0f;
    return KMAJOR ? p[r * stride + k] : p[k * stride + r];
  }
};

struct Stage {
  float a[CE_K][CE_ROWS + 4];
  float b[CE_K][CE_COLS + 4];
};

template <bool KMAJOR>
__device__ __forceinline__ void fetch(const Operand<KMAJOR>& o, int64_t r0, int64_t k0, int64_t k_end, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = threadIdx.x + i * CE_THREADS;
    const int r = KMAJOR ? e / CE_K : e % CE_ROWS, k = KMAJOR ? e % CE_K : e / CE_ROWS;
    v[i] = o.at(r0 + r, k0 + k, k_end);
  }
}
template <bool KMAJOR>
__device__ __forceinline__ void stage(float (*s)[CE_ROWS + 4], const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = threadIdx.x + i * CE_THREADS;
    const int r = KMAJOR ? e / CE_K : e % CE_ROWS, k = KMAJOR ? e % CE_K : e / CE_ROWS;
    s[k][r] = v[i];
  }
}
// rows (i < 4 ? i : 60 + i) + 4 * (thread / 16) of the tile, columns likewise with thread % 16
__device__ __forceinline__ int tile_at(int who, int i) { return who * 4 + (i < 4 ? i : 60 + i); }

template <bool AK, bool BK>
__device__ __forceinline__ void tile_product(const Operand<AK>& a, int64_t m0, const Operand<BK>& b, int64_t n0, int64_t k0,
                                             int64_t k_end, Stage& sm, float (&acc)[8][8]) {
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
  float va[8], vb[8];
  fetch(a, m0, k0, k_end, va);
  fetch(b, n0, k0, k_end, vb);
  for (int64_t k = k0; k < k_end; k += CE_K) {
    __syncthreads();
    stage<AK>(sm.a, va);
    stage<BK>(sm.b, vb);
    __syncthreads();
    if (k + CE_K < k_end) {
      fetch(a, m0, k + CE_K, k_end, va);
      fetch(b, n0, k + CE_K, k_end, vb);
    }
#pragma unroll
    for (int kk = 0; kk < CE_K; ++kk) {
      float ra[8], rb[8];
      *reinterpret_cast<float4*>(ra) = *reinterpret_cast<const float4*>(&sm.a[kk][ty * 4]);
      *reinterpret_cast<float4*>(ra + 4) = *reinterpret_cast<const float4*>(&sm.a[kk][ty * 4 + 64]);
      *reinterpret_cast<float4*>(rb) = *reinterpret_cast<const float4*>(&sm.b[kk][tx * 4]);
      *reinterpret_cast<float4*>(rb + 4) = *reinterpret_cast<const float4*>(&sm.b[kk][tx * 4 + 64]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] += ra[i] * rb[j];
    }
  }
}

struct StatsArgs {
  int64_t n, V;
  int D;
  int64_t row_blocks, col_tiles, slices;
  const int32_t* word;
  float* target_logit;
  float* top;    // [n][slices]
  float* total;  // [n][slices]
};

__global__ void __launch_bounds__(CE_THREADS, 2) ce_stats_kernel(const Operand<true> h, const Operand<true> w,
                                                                 const __grid_constant__ StatsArgs a) {
  __shared__ __align__(16) Stage sm;
  pdl_enter();
  const int64_t rb = blockIdx.x % a.row_blocks, slice = blockIdx.x / a.row_blocks;
  const int64_t t0 = a.col_tiles * slice / a.slices, t1 = a.col_tiles * (slice + 1) / a.slices;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t m0 = rb * CE_ROWS;
  float top[8], total[8];
  int32_t word[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + tile_at(ty, i);
    top[i] = -INFINITY;
    total[i] = 0.0f;
    word[i] = row < a.n ? a.word[row] : -1;
  }
  for (int64_t t = t0; t < t1; ++t) {
    float acc[8][8];
    const int64_t n0 = t * CE_COLS;
    tile_product(h, m0, w, n0, 0, a.D, sm, acc);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float m = top[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t v = n0 + tile_at(tx, j);
        if (v >= a.V) acc[i][j] = -INFINITY;
        if (v == word[i]) a.target_logit[m0 + tile_at(ty, i)] = acc[i][j];
        m = fmaxf(m, acc[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, o));
      // nothing but minus infinity so far: the exponential must not see their difference
      const float base = m == -INFINITY ? 0.0f : m;
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += expf(acc[i][j] - base);
      total[i] = total[i] * expf(top[i] - base) + s;  // each of the 16 threads keeps the sum of its own columns
      top[i] = m;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float s = total[i];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(FULL_MASK, s, o);
    const int64_t row = m0 + tile_at(ty, i);
    if (tx == 0 && row < a.n) {
      a.top[row * a.slices + slice] = top[i];
      a.total[row * a.slices + slice] = s;
    }
  }
}

struct JoinArgs {
  const float *top, *total;
  int64_t groups, slices, n, V, ignore_index;
  const void* target;
  int32_t ids64;
  const int32_t *live, *word, *slot;
  const float* target_logit;
  float *loss, *lse;
  int32_t* status;
};

// A warp joins one row's parts, in an order that depends on their number alone
__global__ void __launch_bounds__(CE_THREADS) ce_join_kernel(const __grid_constant__ JoinArgs a) {
  pdl_enter();
  const int64_t row = blockIdx.x * static_cast<int64_t>(CE_THREADS / 32) + (threadIdx.x >> 5);
  if (row >= a.n) return;
  const int lane = threadIdx.x & 31;
  int64_t c = row;  // its packed row
  bool live;
  if (a.slot != nullptr) {
    c = a.slot[row];
    live = c >= 0;
  } else if (a.word != nullptr) {
    live = a.word[row] >= 0;
  } else {
    bool wrong;
    live = target_word(a.target, a.ids64, row, a.V, a.ignore_index, &wrong) >= 0;
    if (wrong && lane == 0) raise_status(a.status, DGS_ERR_RANGE);
  }
  if (!live) {
    if (lane == 0) a.loss[row] = a.lse[row] = 0.0f;
    return;
  }
  const int64_t parts = a.groups * (a.live != nullptr ? a.live[1] : a.slices);
  const float *top = a.top + c * parts, *total = a.total + c * parts;
  float m = -INFINITY, s = 0.0f;
  constexpr int U = 8;  // parts under way a lane
  for (int64_t p0 = lane; p0 < parts; p0 += 32 * U) {
    float t[U], e[U], now = m;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const bool in = p0 + 32 * k < parts;
      t[k] = in ? top[p0 + 32 * k] : -INFINITY;
      e[k] = in ? total[p0 + 32 * k] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) now = fmaxf(now, t[k]);
    const float base = now == -INFINITY ? 0.0f : now;
    s *= expf(m - base);
#pragma unroll
    for (int k = 0; k < U; ++k) s += e[k] * expf(t[k] - base);
    m = now;
  }
  float all = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(FULL_MASK, all, o));
  const float base = all == -INFINITY ? 0.0f : all;
  s *= expf(m - base);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL_MASK, s, o);
  if (lane == 0) {
    const float l = logf(s);
    a.lse[row] = base + l;
    a.loss[row] = (base - a.target_logit[c]) + l;  // logits of one size meet first: exact, or nearly
  }
}

struct GradArgs {
  int64_t n, V, v0;  // first class of the piece
  int64_t pitch;     // of G
  int64_t row_blocks;
  int D;
  const int32_t* word;
  const float* dloss;
  const float* lse;
  const float* hit;
  float* g;  // [n][pitch]
};

__global__ void __launch_bounds__(CE_THREADS, 2) ce_grad_kernel(const Operand<true> h, const Operand<true> w,
                                                                const __grid_constant__ GradArgs a) {
  __shared__ __align__(16) Stage sm;
  pdl_enter();
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t m0 = blockIdx.x % a.row_blocks * CE_ROWS, n0 = blockIdx.x / a.row_blocks * CE_COLS;
  float acc[8][8];
  tile_product(h, m0, w, n0, 0, a.D, sm, acc);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + tile_at(ty, i);
    if (row >= a.n) continue;
    const int32_t word = a.word[row];
    const float scale = word >= 0 ? a.dloss[row] : 0.0f, lse = a.lse[row], hit = a.hit != nullptr ? a.hit[row] : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = n0 + tile_at(tx, j);
      if (a.v0 + c >= a.V || c >= a.pitch) continue;
      float p = expf(acc[i][j] - lse);
      if (a.v0 + c == word) p = a.hit != nullptr ? hit : p - 1.0f;
      a.g[row * a.pitch + c] = word >= 0 ? scale * p : 0.0f;
    }
  }
}

// out [splits][rows of a][rows of b]; grow: added to what is there
template <bool AK>
__global__ void __launch_bounds__(CE_THREADS, 2) ce_product_kernel(const Operand<AK> a, const Operand<false> b, const int64_t K,
                                                                   float* __restrict__ out, const bool grow) {
  __shared__ __align__(16) Stage sm;
  pdl_enter();
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * CE_ROWS, n0 = static_cast<int64_t>(blockIdx.y) * CE_COLS;
  const int64_t kt = (K + CE_K - 1) / CE_K;
  const int64_t k0 = kt * blockIdx.z / gridDim.z * CE_K, k1 = kt * (blockIdx.z + 1) / gridDim.z * CE_K;
  float acc[8][8];
  tile_product(a, m0, b, n0, k0, k1 < K ? k1 : K, sm, acc);
  float* to = out + static_cast<int64_t>(blockIdx.z) * a.rows * b.rows;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = m0 + tile_at(ty, i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = n0 + tile_at(tx, j);
      if (r < a.rows && c < b.rows) {
        float* at = to + r * b.rows + c;
        *at = grow ? *at + acc[i][j] : acc[i][j];
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(CE_THREADS) ce_sum_kernel(const float* __restrict__ parts, const int64_t splits, const int64_t split_elems,
                                                            const int64_t n, const int D, const int pitch,
                                                            const int32_t* __restrict__ slot, const bool vectors, const bool fours,
                                                            T* __restrict__ out) {
  pdl_enter();
  const int lane = threadIdx.x & 31, chunks = (D + 127) / 128;
  // a warp takes 128 columns of a row
  for (int64_t w = blockIdx.x * static_cast<int64_t>(CE_THREADS / 32) + (threadIdx.x >> 5); w < n * chunks;
       w += gridDim.x * static_cast<int64_t>(CE_THREADS / 32)) {
    const int64_t row = w / chunks;
    const int j = static_cast<int>(w - row * chunks) * 128 + lane * 4;
    if (j >= D) continue;
    const int64_t c = slot != nullptr ? slot[row] : row;
    const float* p = parts + c * pitch + j;
    T* to = out + row * D + j;
    float v[4] = {};
    if (c >= 0) {
#pragma unroll 8
      for (int64_t k = 0; k < splits; ++k) {
        float t[4];
        if (vectors) {
          load_vec<float, 4>(p + k * split_elems, t);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = j + i < D ? p[k * split_elems + i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
      }
    }
    if (fours) {
      store_vec<T, 4>(to, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i < D) to[i] = from_float<T>(v[i]);
    }
  }
}

// ---- host side -----------------------------------------------------------------------------------------------------
struct Plan {
  int64_t pitch;                       // of the packed rows, in elements
  int64_t row_blocks, col_tiles, slices;
  int64_t piece;                       // classes of a piece
  int64_t splits;                      // of a piece's classes in dh's product
  size_t packed, word, target_logit, top, total, dloss, lse, hit, g, dh;
  size_t forward_bytes, backward_bytes;
};

Plan make_plan(int64_t n, int64_t D, int64_t V) {
  Plan p{};
  const int64_t slots = static_cast<int64_t>(sm_count()) * 2;
  p.pitch = D;
  p.row_blocks = tiles(n, CE_ROWS);
  p.col_tiles = tiles(V, CE_COLS);
  p.slices = slices_for(p.row_blocks, p.col_tiles, slots);
  p.piece = CE_PIECE_BYTES / 4 / (n > 0 ? n : 1) / CE_COLS * CE_COLS;
  if (p.piece < 2 * CE_COLS) p.piece = 2 * CE_COLS;
  if (p.piece > p.col_tiles * CE_COLS) p.piece = p.col_tiles * CE_COLS;
  const int64_t dh_tiles = p.row_blocks * tiles(D, CE_COLS);
  p.splits = dh_tiles < slots ? slots / dh_tiles : 1;
  if (p.splits > tiles(p.piece, 512)) p.splits = tiles(p.piece, 512);
  Layout l;
  p.packed = l.take(n * p.pitch * 4);
  p.word = l.take(n * 4);
  const Layout common = l;
  p.target_logit = l.take(n * 4);
  p.top = l.take(p.slices * n * 4);
  p.total = l.take(p.slices * n * 4);
  p.forward_bytes = l.bytes;
  l = common;
  p.dloss = l.take(n * 4);
  p.lse = l.take(n * 4);
  p.hit = l.take(n * 4);
  p.g = l.take(n * p.piece * 4);
  p.dh = l.take(p.splits * n * D * 4);
  p.backward_bytes = l.bytes;
  return p;
}

int forward32(const CeProblem& q, float* loss, float* lse, cudaStream_t s) {
  const Plan p = make_plan(q.n, q.D, q.V);
  const float* packed = reinterpret_cast<const float*>(q.ws + p.packed);
  int32_t* word = reinterpret_cast<int32_t*>(q.ws + p.word);
  float* tl = reinterpret_cast<float*>(q.ws + p.target_logit);
  CePacked to{};
  to.rows = q.ws + p.packed;
  to.pitch = p.pitch;
  to.word = word;
  if (int rc = ce_pack(q, to, nullptr, nullptr, nullptr, s)) return rc;
  float *top = reinterpret_cast<float*>(q.ws + p.top), *total = reinterpret_cast<float*>(q.ws + p.total);
  const StatsArgs a{q.n, q.V, static_cast<int>(q.D), p.row_blocks, p.col_tiles, p.slices, word, tl, top, total};
  DGS_CUDA_TRY(launch_training(ce_stats_kernel, dim3(static_cast<unsigned>(p.row_blocks * p.slices)), CE_THREADS, 0, s,
                               Operand<true>{packed, p.pitch, q.n}, Operand<true>{static_cast<const float*>(q.weight), q.weight_stride, q.V}, a));
  return ce_join(q, top, total, 1, p.slices, nullptr, word, nullptr, tl, loss, lse, s);
}

int backward32(const CeProblem& q, const float* dloss, const float* lse, const float* loss, float* dhidden, float* dweight, cudaStream_t s) {
  const Plan p = make_plan(q.n, q.D, q.V);
  int32_t* word = reinterpret_cast<int32_t*>(q.ws + p.word);
  const float* packed = reinterpret_cast<const float*>(q.ws + p.packed);
  CePacked to{};
  to.rows = q.ws + p.packed;
  to.pitch = p.pitch;
  to.word = word;
  to.dloss = reinterpret_cast<float*>(q.ws + p.dloss);
  to.lse = reinterpret_cast<float*>(q.ws + p.lse);
  to.hit = loss != nullptr ? reinterpret_cast<float*>(q.ws + p.hit) : nullptr;
  if (int rc = ce_pack(q, to, dloss, lse, loss, s)) return rc;
  float *g = reinterpret_cast<float*>(q.ws + p.g), *dh = reinterpret_cast<float*>(q.ws + p.dh);
  const unsigned dtiles = static_cast<unsigned>(tiles(q.D, CE_COLS));
  for (int64_t v0 = 0; v0 < q.V; v0 += p.piece) {
    const int64_t width = q.V - v0 < p.piece ? q.V - v0 : p.piece;
    const float* wp = static_cast<const float*>(q.weight) + v0 * q.weight_stride;
    const GradArgs a{q.n, q.V, v0, p.piece, p.row_blocks, static_cast<int>(q.D), word, to.dloss, to.lse, to.hit, g};
    DGS_CUDA_TRY(launch_training(ce_grad_kernel, dim3(static_cast<unsigned>(p.row_blocks * tiles(width, CE_COLS))), CE_THREADS, 0, s,
                                 Operand<true>{packed, p.pitch, q.n}, Operand<true>{wp, q.weight_stride, width}, a));
    if (dhidden != nullptr)
      DGS_CUDA_TRY(launch_training(ce_product_kernel<true>, dim3(static_cast<unsigned>(p.row_blocks), dtiles, static_cast<unsigned>(p.splits)),
                                   CE_THREADS, 0, s, Operand<true>{g, p.piece, q.n}, Operand<false>{wp, q.weight_stride, q.D}, width, dh, v0 > 0));
    if (dweight != nullptr)
      DGS_CUDA_TRY(launch_training(ce_product_kernel<false>, dim3(static_cast<unsigned>(tiles(width, CE_ROWS)), dtiles), CE_THREADS, 0, s,
                                   Operand<false>{g, p.piece, width}, Operand<false>{packed, p.pitch, q.D}, q.n, dweight + v0 * q.D, false));
  }
  if (dhidden != nullptr) return ce_sum(dh, p.splits, q.n, q.D, q.n, q.D, nullptr, dhidden, DGS_F32, s);
  return DGS_OK;
}

int check(const char* who, const CeProblem& q) {
  DGS_REQUIRE(dtype_bytes(q.dtype) != 0, DGS_ERR_UNSUPPORTED, "%s: element type %d", who, q.dtype);
  DGS_REQUIRE(q.n >= 0 && q.D >= 1 && q.V >= 1, DGS_ERR_INVALID, "%s: %lld rows of %lld elements, %lld classes", who,
              static_cast<long long>(q.n), static_cast<long long>(q.D), static_cast<long long>(q.V));
  DGS_REQUIRE(q.n < (int64_t(1) << 30) && q.V < (int64_t(1) << 30) && q.D <= (int64_t(1) << 20), DGS_ERR_UNSUPPORTED,
              "%s: at most 2^30 rows and classes, and 2^20 elements a row", who);
  DGS_REQUIRE((q.hidden_stride >= q.D || q.n <= 1) && (q.weight_stride >= q.D || q.V == 1), DGS_ERR_INVALID,
              "%s: rows of %lld elements %lld and %lld apart", who, static_cast<long long>(q.D),
              static_cast<long long>(q.hidden_stride), static_cast<long long>(q.weight_stride));
  return DGS_OK;
}

}  // namespace

int ce_pack(const CeProblem& q, const CePacked& p, const float* dloss, const float* lse, const float* loss, cudaStream_t s) {
  const int64_t per16 = 16 / dtype_bytes(q.dtype);
  const bool vectors = q.D == p.pitch && p.pitch % per16 == 0 && q.hidden_stride % per16 == 0 && aligned_to(q.hidden, 16);
  const PackArgs a{q.hidden, q.hidden_stride, q.target, q.ids64,  vectors, q.n, q.V, q.ignore_index, static_cast<int32_t>(q.D),
                   static_cast<int32_t>(p.pitch), p, dloss, lse, loss, q.status};
  if (p.compact)
    DGS_CUDA_TRY(launch_training(ce_count_kernel, dim3(static_cast<unsigned>(tiles(q.n, CE_COUNT_ROWS))), CE_THREADS, 0, s, a));
  const dim3 grid(static_cast<unsigned>(ce_pack_ctas(q.n)));
  // (16-bit elements are moved as they are, whichever of the two types they have)
  if (q.dtype == DGS_F32) DGS_CUDA_TRY(launch_training(ce_pack_kernel<float>, grid, CE_THREADS, 0, s, a));
  else DGS_CUDA_TRY(launch_training(ce_pack_kernel<__half>, grid, CE_THREADS, 0, s, a));
  return DGS_OK;
}

int ce_join(const CeProblem& q, const float* top, const float* total, int64_t groups, int64_t slices, const int32_t* live,
            const int32_t* word, const int32_t* slot, const float* target_logit, float* loss, float* lse, cudaStream_t s) {
  const JoinArgs a{top, total, groups, slices, q.n, q.V, q.ignore_index, q.target, q.ids64, live, word, slot, target_logit, loss, lse, q.status};
  DGS_CUDA_TRY(launch_training(ce_join_kernel, dim3(static_cast<unsigned>(tiles(q.n, CE_THREADS / 32))), CE_THREADS, 0, s, a));
  return DGS_OK;
}

int ce_sum(const float* parts, int64_t splits, int64_t n, int64_t D, int64_t rows, int64_t pitch, const int32_t* slot, void* out,
           int32_t dtype, cudaStream_t s) {
  const int64_t need = tiles(n * tiles(D, 128), CE_THREADS / 32), most = static_cast<int64_t>(sm_count()) * 16;
  const dim3 grid(static_cast<unsigned>(need < most ? need : most));
  const int d = static_cast<int>(D), pt = static_cast<int>(pitch);
  const bool vectors = pitch % 4 == 0, fours = vectors && D % 4 == 0 && aligned_to(out, 16);
  if (dtype == DGS_F32)
    DGS_CUDA_TRY(launch_training(ce_sum_kernel<float>, grid, CE_THREADS, 0, s, parts, splits, rows * pitch, n, d, pt, slot, vectors, fours,
                                 static_cast<float*>(out)));
  else if (dtype == DGS_BF16)
    DGS_CUDA_TRY(launch_training(ce_sum_kernel<__nv_bfloat16>, grid, CE_THREADS, 0, s, parts, splits, rows * pitch, n, d, pt, slot, vectors, fours,
                                 static_cast<__nv_bfloat16*>(out)));
  else
    DGS_CUDA_TRY(launch_training(ce_sum_kernel<__half>, grid, CE_THREADS, 0, s, parts, splits, rows * pitch, n, d, pt, slot, vectors, fours,
                                 static_cast<__half*>(out)));
  return DGS_OK;
}

}  // namespace dgs

using namespace dgs;

extern "C" size_t dgs_linear_cross_entropy_workspace_bytes(int64_t n, int64_t D, int64_t V, int32_t dtype) {
  if (n <= 0 || D <= 0 || V <= 0 || dtype_bytes(dtype) == 0) return 0;
  return dtype == DGS_F32 ? make_plan(n, D, V).forward_bytes : ce_mma_forward_bytes(n, D, V);
}

extern "C" int dgs_linear_cross_entropy(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                                        int32_t dtype, const void* target, int32_t ids64, int64_t n, int64_t D, int64_t V,
                                        int64_t ignore_index, float* loss, float* lse, void* workspace, size_t workspace_bytes,
                                        int32_t* status, dgs_stream_t stream) {
  const CeProblem q{hidden, hidden_stride, weight, weight_stride, dtype, target, ids64 != 0, n, D, V, ignore_index, static_cast<char*>(workspace), status};
  if (int rc = check("linear_cross_entropy", q)) return rc;
  if (n == 0) return DGS_OK;
  DGS_REQUIRE(hidden != nullptr && weight != nullptr && target != nullptr && loss != nullptr && lse != nullptr, DGS_ERR_INVALID,
              "linear_cross_entropy: null argument");
  const size_t need = dgs_linear_cross_entropy_workspace_bytes(n, D, V, dtype);
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "linear_cross_entropy: workspace of %zu bytes, 256-byte aligned, is needed", need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == DGS_F32 ? forward32(q, loss, lse, s) : ce_mma_forward(q, loss, lse, s);
}

extern "C" size_t dgs_linear_cross_entropy_backward_workspace_bytes(int64_t n, int64_t D, int64_t V, int32_t dtype) {
  if (n <= 0 || D <= 0 || V <= 0 || dtype_bytes(dtype) == 0) return 0;
  return dtype == DGS_F32 ? make_plan(n, D, V).backward_bytes : ce_mma_backward_bytes(n, D, V);
}

extern "C" int dgs_linear_cross_entropy_backward_from_loss(const float* dloss, const void* hidden, int64_t hidden_stride, const void* weight,
                                                           int64_t weight_stride, int32_t dtype, const void* target, int32_t ids64,
                                                           const float* lse, const float* loss, int64_t n, int64_t D, int64_t V,
                                                           int64_t ignore_index, void* dhidden, void* dweight, void* workspace,
                                                           size_t workspace_bytes, int32_t* status, dgs_stream_t stream) {
  const CeProblem q{hidden, hidden_stride, weight, weight_stride, dtype, target, ids64 != 0, n, D, V, ignore_index, static_cast<char*>(workspace), status};
  if (int rc = check("linear_cross_entropy_backward", q)) return rc;
  if (dhidden == nullptr && dweight == nullptr) return DGS_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    if (dweight != nullptr) DGS_CUDA_TRY(cudaMemsetAsync(dweight, 0, static_cast<size_t>(V) * D * dtype_bytes(dtype), s));
    return DGS_OK;
  }
  DGS_REQUIRE(dloss != nullptr && hidden != nullptr && weight != nullptr && target != nullptr && lse != nullptr, DGS_ERR_INVALID,
              "linear_cross_entropy_backward: null argument");
  const size_t need = dgs_linear_cross_entropy_backward_workspace_bytes(n, D, V, dtype);
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "linear_cross_entropy_backward: workspace of %zu bytes, 256-byte aligned, is needed", need);
  return dtype == DGS_F32 ? backward32(q, dloss, lse, loss, static_cast<float*>(dhidden), static_cast<float*>(dweight), s)
                          : ce_mma_backward(q, dloss, lse, loss, dhidden, dweight, s);
}

extern "C" int dgs_linear_cross_entropy_backward(const float* dloss, const void* hidden, int64_t hidden_stride, const void* weight,
                                                 int64_t weight_stride, int32_t dtype, const void* target, int32_t ids64,
                                                 const float* lse, int64_t n, int64_t D, int64_t V, int64_t ignore_index, void* dhidden,
                                                 void* dweight, void* workspace, size_t workspace_bytes, int32_t* status,
                                                 dgs_stream_t stream) {
  return dgs_linear_cross_entropy_backward_from_loss(dloss, hidden, hidden_stride, weight, weight_stride, dtype, target, ids64, lse, nullptr, n, D,
                                                     V, ignore_index, dhidden, dweight, workspace, workspace_bytes, status, stream);
}
