// Softmax cross entropy of hidden rows against a weight row per class, the logits never all held, with its gradients.
//
//   s_iv = h_i . W_v,  lse_i = log sum_v exp(s_iv),  loss_i = lse_i - s_i,t(i)
//   G_iv = dloss_i (exp(s_iv - lse_i) - [v = t(i)]),  dh = G W,  dW = G^T h
//
// Forward: a row block of 128 meets the vocabulary tile by tile; each row carries a running maximum and a running sum of
// exponentials, so a tile of logits lives in registers only.  The vocabulary is cut into slices where there are fewer row
// blocks than SMs; a last launch joins the slices' (maximum, sum) pairs in their order.
// Backward: the vocabulary is taken in pieces.  Per piece the logits are computed again, leave as G into a buffer sized to
// stay in L2 for the most part, and two products read it: dh grows in 32 bits over the pieces, dW's rows of the piece are
// complete.  That is 8 n V D operations for a training step instead of 6 with the logits kept (n V values, 2.1 GB at
// 8 192 rows and 65 537 classes).
//
// A first launch copies the hidden rows into packed rows and the targets into 32-bit words: rows without a valid target
// become zero there, so that what stands in an ignored row (an infinity, say) reaches neither dh nor dW, and alignment
// and strides no longer matter.
#include "train_common.cuh"

namespace dgs {
namespace {

constexpr int CE_ROWS = 128;            // rows of a tile
constexpr int CE_COLS = 128;            // classes of a tile
constexpr int CE_K = 16;
constexpr int CE_THREADS = 256;
constexpr int64_t CE_PIECE_BYTES = int64_t(96) << 20;  // of G: what L2 (126 MB) holds beside the operands

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline int64_t tiles(int64_t v, int64_t per) { return (v + per - 1) / per; }

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

// ---- packing -----------------------------------------------------------------------------------------------------
template <typename T, typename IdT>
__global__ void __launch_bounds__(CE_THREADS) ce_pack_kernel(const T* __restrict__ hidden, const int64_t stride,
                                                             const IdT* __restrict__ target, const int64_t n, const int D,
                                                             const int pitch, const int64_t V, const int64_t ignore_index,
                                                             T* __restrict__ packed, int32_t* __restrict__ word,
                                                             float* __restrict__ target_logit, int32_t* status) {
  pdl_enter();
  const int64_t row = blockIdx.x * static_cast<int64_t>(CE_THREADS / 32) + (threadIdx.x >> 5);
  if (row >= n) return;
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(target[row]);
  const bool ignored = t == ignore_index;
  const bool live = !ignored && t >= 0 && t < V;
  if (lane == 0) {
    word[row] = live ? static_cast<int32_t>(t) : -1;
    if (target_logit != nullptr) target_logit[row] = 0.0f;
    if (!ignored && !live) raise_status(status, DGS_ERR_RANGE);
  }
  const T* from = hidden + row * stride;
  T* to = packed + row * pitch;
  for (int j = lane; j < pitch; j += 32) to[j] = live && j < D ? from[j] : from_float<T>(0.0f);
}

// ---- products on the CUDA cores ------------------------------------------------------------------------------------
// A tile of CE_ROWS x CE_COLS, eight by eight values a thread, operands staged through shared memory CE_K at a time.
// KMAJOR: element (r, k) at p[r * stride + k]; else at p[k * stride + r].
template <typename T, bool KMAJOR>
struct Operand {
  const T* p;
  int64_t stride;
  int64_t rows;
  __device__ __forceinline__ float at(int64_t r, int64_t k, int64_t k_end) const {
    if (r >= rows || k >= k_end) return 0.0f;
    return to_float<T>(KMAJOR ? p[r * stride + k] : p[k * stride + r]);
  }
};

struct Stage {
  float a[CE_K][CE_ROWS + 4];
  float b[CE_K][CE_COLS + 4];
};

template <typename T, bool KMAJOR>
__device__ __forceinline__ void fetch(const Operand<T, KMAJOR>& o, int64_t r0, int64_t k0, int64_t k_end, float (&v)[8]) {
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

template <typename TA, bool AK, typename TB, bool BK>
__device__ __forceinline__ void tile_product(const Operand<TA, AK>& a, int64_t m0, const Operand<TB, BK>& b, int64_t n0, int64_t k0,
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
  float* top;    // [slices][n]
  float* total;  // [slices][n]
};

template <typename T>
__global__ void __launch_bounds__(CE_THREADS, 2) ce_stats_kernel(const Operand<T, true> h, const Operand<T, true> w,
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
      const float base = m == -INFINITY ? 0.0f : m;  // nothing but minus infinity so far: exp must not see their difference
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
      a.top[slice * a.n + row] = top[i];
      a.total[slice * a.n + row] = s;
    }
  }
}

__global__ void __launch_bounds__(CE_THREADS) ce_join_kernel(const float* __restrict__ top, const float* __restrict__ total,
                                                             const int64_t parts, const int64_t n, const int32_t* __restrict__ word,
                                                             const float* __restrict__ target_logit, float* __restrict__ loss,
                                                             float* __restrict__ lse) {
  pdl_enter();
  const int64_t row = blockIdx.x * static_cast<int64_t>(CE_THREADS) + threadIdx.x;
  if (row >= n) return;
  float m = -INFINITY;
  for (int64_t p = 0; p < parts; ++p) m = fmaxf(m, top[p * n + row]);
  const float base = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
  for (int64_t p = 0; p < parts; ++p) s += total[p * n + row] * expf(top[p * n + row] - base);
  const float l = base + logf(s);
  const bool live = word[row] >= 0;
  lse[row] = live ? l : 0.0f;
  loss[row] = live ? l - target_logit[row] : 0.0f;
}

struct GradArgs {
  int64_t n, V, v0;  // first class of the piece
  int64_t pitch;     // of G
  int64_t row_blocks;
  int D;
  const int32_t* word;
  const float* dloss;
  const float* lse;
  float* g;  // [n][pitch]
};

template <typename T>
__global__ void __launch_bounds__(CE_THREADS, 2) ce_grad_kernel(const Operand<T, true> h, const Operand<T, true> w,
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
    const float scale = word >= 0 ? a.dloss[row] : 0.0f, lse = a.lse[row];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = n0 + tile_at(tx, j);
      if (a.v0 + c >= a.V || c >= a.pitch) continue;
      const float p = expf(acc[i][j] - lse) - (a.v0 + c == word ? 1.0f : 0.0f);
      a.g[row * a.pitch + c] = word >= 0 ? scale * p : 0.0f;
    }
  }
}

// out (32 bits, [splits][rows][cols], grown over the calls unless `first`) or, `last`-typed, T [rows][cols]
template <typename TA, bool AK, typename TB, bool BK, typename OUT>
__global__ void __launch_bounds__(CE_THREADS, 2) ce_product_kernel(const Operand<TA, AK> a, const Operand<TB, BK> b, const int64_t K,
                                                                   OUT* __restrict__ out, const bool grow) {
  __shared__ __align__(16) Stage sm;
  pdl_enter();
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * CE_ROWS, n0 = static_cast<int64_t>(blockIdx.y) * CE_COLS;
  const int64_t kt = (K + CE_K - 1) / CE_K;
  const int64_t k0 = kt * blockIdx.z / gridDim.z * CE_K, k1 = kt * (blockIdx.z + 1) / gridDim.z * CE_K;
  float acc[8][8];
  tile_product(a, m0, b, n0, k0, k1 < K ? k1 : K, sm, acc);
  OUT* to = out + static_cast<int64_t>(blockIdx.z) * a.rows * b.rows;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = m0 + tile_at(ty, i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t c = n0 + tile_at(tx, j);
      if (r < a.rows && c < b.rows) {
        float v = acc[i][j];
        if (grow) v += to_float<OUT>(to[r * b.rows + c]);
        to[r * b.rows + c] = from_float<OUT>(v);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(CE_THREADS) ce_sum_kernel(const float* __restrict__ parts, const int64_t splits, const int64_t n,
                                                            T* __restrict__ out) {
  pdl_enter();
  for (int64_t i = blockIdx.x * static_cast<int64_t>(CE_THREADS) + threadIdx.x; i < n; i += gridDim.x * static_cast<int64_t>(CE_THREADS)) {
    float s = 0.0f;
    for (int64_t p = 0; p < splits; ++p) s += parts[p * n + i];
    out[i] = from_float<T>(s);
  }
}

// ---- host side -----------------------------------------------------------------------------------------------------
struct Plan {
  int64_t pitch;                       // of the packed rows, in elements
  int64_t row_blocks, col_tiles, slices;
  int64_t piece;                       // classes of a piece
  int64_t splits;                      // of a piece's classes in dh's product
  // offsets in the workspace
  size_t packed, word, target_logit, top, total, g, dh;
  size_t forward_bytes, backward_bytes;
};

Plan make_plan(int64_t n, int64_t D, int64_t V, int32_t dtype) {
  Plan p{};
  const int64_t slots = static_cast<int64_t>(sm_count()) * 2;
  p.pitch = up(D, 8);
  p.row_blocks = tiles(n, CE_ROWS);
  p.col_tiles = tiles(V, CE_COLS);
  p.slices = slices_for(p.row_blocks, p.col_tiles, slots);
  p.piece = CE_PIECE_BYTES / 4 / (n > 0 ? n : 1) / CE_COLS * CE_COLS;
  if (p.piece < 2 * CE_COLS) p.piece = 2 * CE_COLS;
  if (p.piece > p.col_tiles * CE_COLS) p.piece = p.col_tiles * CE_COLS;
  const int64_t dh_tiles = p.row_blocks * tiles(D, CE_COLS);
  p.splits = dh_tiles < slots ? slots / dh_tiles : 1;
  if (p.splits > tiles(p.piece, 512)) p.splits = tiles(p.piece, 512);
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += static_cast<size_t>(up(bytes, 256));
    return here;
  };
  p.packed = take(n * p.pitch * dtype_bytes(dtype));
  p.word = take(n * 4);
  const size_t common = at;
  p.target_logit = take(n * 4);
  p.top = take(p.slices * n * 4);
  p.total = take(p.slices * n * 4);
  p.forward_bytes = at;
  at = common;
  p.g = take(n * p.piece * 4);
  p.dh = take(p.splits * n * D * 4);
  p.backward_bytes = at;
  return p;
}

struct Problem {
  const void* hidden;
  int64_t hidden_stride;
  const void* weight;
  int64_t weight_stride;
  const void* target;
  bool ids64;
  int64_t n, D, V, ignore_index;
  char* ws;
  int32_t* status;
};

template <typename T>
int pack(const Problem& q, const Plan& p, bool logits, cudaStream_t s) {
  T* packed = reinterpret_cast<T*>(q.ws + p.packed);
  int32_t* word = reinterpret_cast<int32_t*>(q.ws + p.word);
  float* tl = logits ? reinterpret_cast<float*>(q.ws + p.target_logit) : nullptr;
  const dim3 grid(static_cast<unsigned>(tiles(q.n, CE_THREADS / 32)));
  const T* h = static_cast<const T*>(q.hidden);
  if (q.ids64)
    DGS_CUDA_TRY(launch_training(ce_pack_kernel<T, int64_t>, grid, CE_THREADS, 0, s, h, q.hidden_stride, static_cast<const int64_t*>(q.target),
                                 q.n, static_cast<int>(q.D), static_cast<int>(p.pitch), q.V, q.ignore_index, packed, word, tl, q.status));
  else
    DGS_CUDA_TRY(launch_training(ce_pack_kernel<T, int32_t>, grid, CE_THREADS, 0, s, h, q.hidden_stride, static_cast<const int32_t*>(q.target),
                                 q.n, static_cast<int>(q.D), static_cast<int>(p.pitch), q.V, q.ignore_index, packed, word, tl, q.status));
  return DGS_OK;
}

template <typename T>
int forward(const Problem& q, const Plan& p, float* loss, float* lse, cudaStream_t s) {
  if (int rc = pack<T>(q, p, true, s)) return rc;
  const int32_t* word = reinterpret_cast<const int32_t*>(q.ws + p.word);
  float* tl = reinterpret_cast<float*>(q.ws + p.target_logit);
  float *top = reinterpret_cast<float*>(q.ws + p.top), *total = reinterpret_cast<float*>(q.ws + p.total);
  const Operand<T, true> h{reinterpret_cast<const T*>(q.ws + p.packed), p.pitch, q.n};
  const Operand<T, true> w{static_cast<const T*>(q.weight), q.weight_stride, q.V};
  const StatsArgs a{q.n, q.V, static_cast<int>(q.D), p.row_blocks, p.col_tiles, p.slices, word, tl, top, total};
  DGS_CUDA_TRY(launch_training(ce_stats_kernel<T>, dim3(static_cast<unsigned>(p.row_blocks * p.slices)), CE_THREADS, 0, s, h, w, a));
  DGS_CUDA_TRY(launch_training(ce_join_kernel, dim3(static_cast<unsigned>(tiles(q.n, CE_THREADS))), CE_THREADS, 0, s, top, total, p.slices,
                               q.n, word, tl, loss, lse));
  return DGS_OK;
}

template <typename T>
int backward(const Problem& q, const Plan& p, const float* dloss, const float* lse, T* dhidden, T* dweight, cudaStream_t s) {
  if (int rc = pack<T>(q, p, false, s)) return rc;
  const int32_t* word = reinterpret_cast<const int32_t*>(q.ws + p.word);
  const T* packed = reinterpret_cast<const T*>(q.ws + p.packed);
  float *g = reinterpret_cast<float*>(q.ws + p.g), *dh = reinterpret_cast<float*>(q.ws + p.dh);
  for (int64_t v0 = 0; v0 < q.V; v0 += p.piece) {
    const int64_t width = q.V - v0 < p.piece ? q.V - v0 : p.piece;
    const T* wp = static_cast<const T*>(q.weight) + v0 * q.weight_stride;
    const GradArgs a{q.n, q.V, v0, p.piece, p.row_blocks, static_cast<int>(q.D), word, dloss, lse, g};
    DGS_CUDA_TRY(launch_training(ce_grad_kernel<T>, dim3(static_cast<unsigned>(p.row_blocks * tiles(width, CE_COLS))), CE_THREADS, 0, s,
                                 Operand<T, true>{packed, p.pitch, q.n}, Operand<T, true>{wp, q.weight_stride, width}, a));
    const unsigned dtiles = static_cast<unsigned>(tiles(q.D, CE_COLS));
    if (dhidden != nullptr)
      DGS_CUDA_TRY(launch_training(ce_product_kernel<float, true, T, false, float>,
                                   dim3(static_cast<unsigned>(p.row_blocks), dtiles, static_cast<unsigned>(p.splits)), CE_THREADS, 0, s,
                                   Operand<float, true>{g, p.piece, q.n}, Operand<T, false>{wp, q.weight_stride, q.D}, width, dh, v0 > 0));
    if (dweight != nullptr)
      DGS_CUDA_TRY(launch_training(ce_product_kernel<float, false, T, false, T>,
                                   dim3(static_cast<unsigned>(tiles(width, CE_ROWS)), dtiles), CE_THREADS, 0, s,
                                   Operand<float, false>{g, p.piece, width}, Operand<T, false>{packed, p.pitch, q.D}, q.n,
                                   dweight + v0 * q.D, false));
  }
  if (dhidden != nullptr) {
    const int64_t count = q.n * q.D, need = tiles(count, CE_THREADS), most = static_cast<int64_t>(sm_count()) * 16;
    DGS_CUDA_TRY(launch_training(ce_sum_kernel<T>, dim3(static_cast<unsigned>(need < most ? need : most)), CE_THREADS, 0, s, dh, p.splits, count, dhidden));
  }
  return DGS_OK;
}

int check(const char* who, const Problem& q, int32_t dtype) {
  DGS_REQUIRE(dtype_bytes(dtype) != 0, DGS_ERR_UNSUPPORTED, "%s: element type %d", who, dtype);
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
}  // namespace dgs

using namespace dgs;

extern "C" size_t dgs_linear_cross_entropy_workspace_bytes(int64_t n, int64_t D, int64_t V, int32_t dtype) {
  if (n <= 0 || D <= 0 || V <= 0 || dtype_bytes(dtype) == 0) return 0;
  return make_plan(n, D, V, dtype).forward_bytes;
}

extern "C" int dgs_linear_cross_entropy(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                                        int32_t dtype, const void* target, int32_t ids64, int64_t n, int64_t D, int64_t V,
                                        int64_t ignore_index, float* loss, float* lse, void* workspace, size_t workspace_bytes,
                                        int32_t* status, dgs_stream_t stream) {
  const Problem q{hidden, hidden_stride, weight, weight_stride, target, ids64 != 0, n, D, V, ignore_index, static_cast<char*>(workspace), status};
  if (int rc = check("linear_cross_entropy", q, dtype)) return rc;
  if (n == 0) return DGS_OK;
  DGS_REQUIRE(hidden != nullptr && weight != nullptr && target != nullptr && loss != nullptr && lse != nullptr, DGS_ERR_INVALID,
              "linear_cross_entropy: null argument");
  const Plan p = make_plan(n, D, V, dtype);
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= p.forward_bytes && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "linear_cross_entropy: workspace of %zu bytes, 256-byte aligned, is needed", p.forward_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == DGS_F32    ? forward<float>(q, p, loss, lse, s)
         : dtype == DGS_BF16 ? forward<__nv_bfloat16>(q, p, loss, lse, s)
                             : forward<__half>(q, p, loss, lse, s);
}

extern "C" size_t dgs_linear_cross_entropy_backward_workspace_bytes(int64_t n, int64_t D, int64_t V, int32_t dtype) {
  if (n <= 0 || D <= 0 || V <= 0 || dtype_bytes(dtype) == 0) return 0;
  return make_plan(n, D, V, dtype).backward_bytes;
}

extern "C" int dgs_linear_cross_entropy_backward(const float* dloss, const void* hidden, int64_t hidden_stride, const void* weight,
                                                 int64_t weight_stride, int32_t dtype, const void* target, int32_t ids64,
                                                 const float* lse, int64_t n, int64_t D, int64_t V, int64_t ignore_index, void* dhidden,
                                                 void* dweight, void* workspace, size_t workspace_bytes, int32_t* status,
                                                 dgs_stream_t stream) {
  const Problem q{hidden, hidden_stride, weight, weight_stride, target, ids64 != 0, n, D, V, ignore_index, static_cast<char*>(workspace), status};
  if (int rc = check("linear_cross_entropy_backward", q, dtype)) return rc;
  if (dhidden == nullptr && dweight == nullptr) return DGS_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    if (dweight != nullptr) DGS_CUDA_TRY(cudaMemsetAsync(dweight, 0, static_cast<size_t>(V) * D * dtype_bytes(dtype), s));
    return DGS_OK;
  }
  DGS_REQUIRE(dloss != nullptr && hidden != nullptr && weight != nullptr && target != nullptr && lse != nullptr, DGS_ERR_INVALID,
              "linear_cross_entropy_backward: null argument");
  const Plan p = make_plan(n, D, V, dtype);
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= p.backward_bytes && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "linear_cross_entropy_backward: workspace of %zu bytes, 256-byte aligned, is needed", p.backward_bytes);
  return dtype == DGS_F32 ? backward<float>(q, p, dloss, lse, static_cast<float*>(dhidden), static_cast<float*>(dweight), s)
         : dtype == DGS_BF16
             ? backward<__nv_bfloat16>(q, p, dloss, lse, static_cast<__nv_bfloat16*>(dhidden), static_cast<__nv_bfloat16*>(dweight), s)
             : backward<__half>(q, p, dloss, lse, static_cast<__half*>(dhidden), static_cast<__half*>(dweight), s);
}
