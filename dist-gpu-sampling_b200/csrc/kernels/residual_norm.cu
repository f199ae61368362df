// The end of a block and the norm in front of the next one, forward and backward:
//
//   z = post(y),  s = xs x + ys gate z  (stored in x's type),  out = pre(s)
//   norm(v) = (v - mean) rstd w + b with mean = 0 for the root-mean-square form; either norm, the gate, biases may be absent
//
//   g = ds + pre'(dout),  dx = xs g,  dgate = ys g z,  dz = ys g gate,  dy = post'(dz)
//   norm'(d) = rstd (d w - avg(d w) - h avg(d w h)), h the normed values (the plain average is left out in the root-mean-square form)
//   dw = sum over rows of d h, db = sum of d, the gate's gradient summed over what it was spread over
//
// Bound by HBM: every row is read and written once in each direction.  TPR threads share a row, eight elements each, which stay in
// registers from the first sum to the result; sums are in 32 bits and of centred values.  A thread keeps its columns for all rows of
// its CTA, so column sums grow in registers; each CTA leaves one partial row and a second launch adds the partial rows in their
// order (no atomics: the same inputs give the same bits).
#include <initializer_list>

#include "train_common.cuh"

namespace dgs {
namespace {

constexpr int RN_ELEMS = 8;  // of a row, a thread
constexpr int RN_MAX_D = 8192;
constexpr int RN_SUMS = 5;   // column sums: dweight, dbias, dpost_weight, dpost_bias, dgate
constexpr int RN_MAX_CTAS_PER_SM = 4;
constexpr int RN_MAX_STAGES = 4;
constexpr int RN_JOIN_THREADS = 1024;
constexpr int RN_MAX_SMEM = 200 * 1024;
constexpr int RN_MAX_DEVICES = 64;

struct Source {
  const void* p;  // nullptr: absent
  int64_t stride;
};

struct NormArgs {
  Source in[5];  // forward: x, y, gate of each element; backward: s, y, dout, ds, gate of each element
  const void *row_gate, *column_gate, *post_weight, *post_bias, *weight, *bias;
  int64_t n;
  int32_t D, param_dtype, post, pre;  // DGS_NORM_*
  float xs, ys, eps;
  // forward
  void *sum, *out;
  float *post_mean, *post_rstd, *mean, *rstd;
  // backward
  void *dx, *dy, *dgate;  // dgate: of each element, or of each row
  float* partial;         // [CTAs][RN_SUMS][D]
  int32_t stages, stage_bytes;
};

template <int TPR>
constexpr int threads_of() {
  return TPR > 32 ? TPR : 256;
}

// COUNT sums over the threads of a row, returned to all of them.  Every thread of the CTA calls it; `red` alternates between two.
template <int TPR, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], float (*red)[4]) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int q = 0; q < COUNT; ++q) v[q] += __shfl_xor_sync(FULL_MASK, v[q], o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int q = 0; q < COUNT; ++q) red[threadIdx.x >> 5][q] = v[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < COUNT; ++q) v[q] = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w)
#pragma unroll
      for (int q = 0; q < COUNT; ++q) v[q] += red[w][q];
  }
}

// The rows of up to COUNT arrays.  16-byte vectors travel by cp.async through a ring in shared memory, so the next rows are on
// their way while one is summed; a thread fetches what it will read itself, so its own wait is all the synchronisation.  Narrower
// vectors (rows off the 16-byte grid) are loaded where they are used.
template <typename T, int VEC, int TPR, int COUNT>
struct Feed {
  static constexpr int NV = RN_ELEMS / VEC, THREADS = threads_of<TPR>();
  static constexpr bool kRing = sizeof(T) * VEC == 16;
  const NormArgs& a;
  uint32_t ring;
  int t, stage;
  int64_t step, ahead;

  __device__ __forceinline__ bool in(int k) const { return (k * TPR + t) * VEC < a.D; }
  __device__ __forceinline__ int column(int k) const { return (k * TPR + t) * VEC; }
  __device__ __forceinline__ void issue(int64_t row, int st) {
    if constexpr (kRing) {
      if (row < a.n) {
        uint32_t at = ring + st * a.stage_bytes + threadIdx.x * 16;
#pragma unroll
        for (int q = 0; q < COUNT; ++q) {
          if (a.in[q].p == nullptr) continue;
          const T* p = static_cast<const T*>(a.in[q].p) + row * a.in[q].stride;
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            if (in(k)) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(p + column(k)) : "memory");
            at += THREADS * 16;
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ void begin(int64_t row, int64_t apart, unsigned char* smem) {
    t = threadIdx.x % TPR;
    stage = 0;
    step = apart;
    if constexpr (kRing) {
      ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
      for (int s = 0; s < a.stages - 1; ++s) issue(row + s * step, s);
    }
    ahead = (a.stages - 1) * step;
  }
  // the rows `row` of this stage: asks for those `stages - 1` steps on, waits for these
  __device__ __forceinline__ void next(int64_t row) {
    if constexpr (kRing) {
      const int last = stage == 0 ? a.stages - 1 : stage - 1;
      issue(row + ahead, last);
      if (a.stages == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else if (a.stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else if (a.stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else asm volatile("cp.async.wait_group 3;" ::: "memory");
    }
  }
  __device__ __forceinline__ void done() {
    if constexpr (kRing) stage = stage + 1 == a.stages ? 0 : stage + 1;
  }
  // array q's elements of the row (zeros outside); `slot`: how many arrays are there before it
  __device__ __forceinline__ void get(int q, int slot, int64_t row, bool there, float (&v)[RN_ELEMS], const unsigned char* smem) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[VEC];
      if (there && in(k)) {
        const T* p = kRing ? reinterpret_cast<const T*>(smem + stage * a.stage_bytes + (slot * NV + k) * THREADS * 16 + threadIdx.x * 16)
                           : static_cast<const T*>(a.in[q].p) + row * a.in[q].stride + column(k);
        load_vec<T, VEC>(p, x);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k * VEC + e] = x[e];
    }
  }
  __device__ __forceinline__ void put(void* base, int64_t row, bool there, const float (&v)[RN_ELEMS]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!(there && in(k))) continue;
      float x[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = v[k * VEC + e];
      store_vec<T, VEC>(static_cast<T*>(base) + row * a.D + column(k), x);
    }
  }
  __device__ __forceinline__ void param(const void* p, float absent, float (&v)[RN_ELEMS]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[VEC];
      if (p != nullptr && in(k)) {
        if constexpr (VEC == 1) x[0] = load_as_float(p, a.param_dtype, column(k));
        else load_vec_as_float<VEC>(p, a.param_dtype, column(k), x);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = absent;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k * VEC + e] = x[e];
    }
  }
};

// normed values of v in place; every thread of the CTA calls it
template <int TPR, int VEC, typename FeedT>
__device__ __forceinline__ void normalise(const FeedT& f, bool layer, int D, float eps, float (&v)[RN_ELEMS], float* mean, float* rstd,
                                          float (*red)[32][4]) {
  const float inv = 1.0f / static_cast<float>(D);
  *mean = 0.0f;
  if (layer) {
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < RN_ELEMS; ++i) s[0] += v[i];
    row_sums<TPR, 1>(s, red[0]);
    *mean = s[0] * inv;
  }
  float s[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < RN_ELEMS; ++i) {
    if (f.in(i / VEC)) {
      v[i] -= *mean;
      s[0] = fmaf(v[i], v[i], s[0]);
    }
  }
  row_sums<TPR, 1>(s, red[1]);
  *rstd = 1.0f / sqrtf(fmaf(s[0], inv, eps));
#pragma unroll
  for (int i = 0; i < RN_ELEMS; ++i) v[i] *= *rstd;
}

template <typename T, int VEC, int TPR>
__global__ __launch_bounds__(threads_of<TPR>()) void residual_norm_kernel(const __grid_constant__ NormArgs a) {
  constexpr int ROWS = threads_of<TPR>() / TPR;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[4][32][4];
  pdl_enter();
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  Feed<T, VEC, TPR, 3> f{a};
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR;
  f.begin(mine, step, smem);
  for (int64_t row = mine; row - threadIdx.x / TPR < a.n; row += step) {
    f.next(row);
    const bool there = row < a.n;
    float y[RN_ELEMS], p[RN_ELEMS], m, r;
    f.get(1, 1, row, there, y, smem);
    if (a.post != DGS_NORM_NONE) {
      normalise<TPR, VEC>(f, a.post == DGS_NORM_LAYER, a.D, a.eps, y, &m, &r, red);
      if (there && f.t == 0) {
        if (a.post == DGS_NORM_LAYER) a.post_mean[row] = m;
        a.post_rstd[row] = r;
      }
      f.param(a.post_weight, 1.0f, p);
      if (a.post_bias != nullptr) {
        float b[RN_ELEMS];
        f.param(a.post_bias, 0.0f, b);
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) y[i] = fmaf(y[i], p[i], b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) y[i] *= p[i];
      }
    }
    if (a.in[2].p != nullptr) {
      f.get(2, 2, row, there, p, smem);
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) y[i] *= p[i];
    } else if (a.column_gate != nullptr) {
      f.param(a.column_gate, 1.0f, p);
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) y[i] *= p[i];
    } else if (a.row_gate != nullptr) {
      const float by = there ? to_float<T>(static_cast<const T*>(a.row_gate)[row]) : 0.0f;
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) y[i] *= by;
    }
    f.get(0, 0, row, there, p, smem);
#pragma unroll
    for (int i = 0; i < RN_ELEMS; ++i) {
      // (the next norm is of the row as it is stored, so that the backward pass finds the same)
      y[i] = to_float<T>(from_float<T>(fmaf(a.ys, y[i], a.xs * p[i])));
    }
    f.done();
    f.put(a.sum, row, there, y);
    if (a.pre != DGS_NORM_NONE) {
      normalise<TPR, VEC>(f, a.pre == DGS_NORM_LAYER, a.D, a.eps, y, &m, &r, red + 2);
      if (there && f.t == 0) {
        if (a.pre == DGS_NORM_LAYER) a.mean[row] = m;
        a.rstd[row] = r;
      }
      f.param(a.weight, 1.0f, p);
      if (a.bias != nullptr) {
        float b[RN_ELEMS];
        f.param(a.bias, 0.0f, b);
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) y[i] = fmaf(y[i], p[i], b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) y[i] *= p[i];
      }
      f.put(a.out, row, there, y);
    }
    if constexpr (TPR > 32) {
      // (a row with one sum alone: `red` must not be written before all have read it)
      if ((a.post != DGS_NORM_NONE) + (a.post == DGS_NORM_LAYER) + (a.pre != DGS_NORM_NONE) + (a.pre == DGS_NORM_LAYER) == 1) __syncthreads();
    }
  }
}

// norm' of d (the gradient of the normed and weighted values) in place, zeros outside of the row; h the normed values; `also` is summed
// over the row too
template <int TPR, int VEC, typename FeedT>
__device__ __forceinline__ void norm_back(const FeedT& f, bool layer, int D, float rstd, const float (&w)[RN_ELEMS], const float (&h)[RN_ELEMS],
                                          float (&d)[RN_ELEMS], float* also, float (*red)[4]) {
  float s[3] = {0.0f, 0.0f, *also};
#pragma unroll
  for (int i = 0; i < RN_ELEMS; ++i) {
    d[i] *= w[i];
    s[0] += d[i];
    s[1] = fmaf(d[i], h[i], s[1]);
  }
  row_sums<TPR, 3>(s, red);
  const float inv = 1.0f / static_cast<float>(D), avg = layer ? s[0] * inv : 0.0f, dot = s[1] * inv;
  *also = s[2];
#pragma unroll
  for (int i = 0; i < RN_ELEMS; ++i) d[i] = f.in(i / VEC) ? rstd * (d[i] - avg - h[i] * dot) : 0.0f;
}

template <typename T, int VEC, int TPR>
__global__ __launch_bounds__(threads_of<TPR>()) void residual_norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int THREADS = threads_of<TPR>(), ROWS = THREADS / TPR;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float red[2][32][4];
  pdl_enter();
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  Feed<T, VEC, TPR, 5> f{a};
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR;
  f.begin(mine, step, smem);
  int slot[5], slots = 0;
#pragma unroll
  for (int q = 0; q < 5; ++q) {
    slot[q] = slots;
    slots += a.in[q].p != nullptr;
  }
  float sums[RN_SUMS][RN_ELEMS];
#pragma unroll
  for (int q = 0; q < RN_SUMS; ++q)
#pragma unroll
    for (int i = 0; i < RN_ELEMS; ++i) sums[q][i] = 0.0f;
  for (int64_t row = mine; row - threadIdx.x / TPR < a.n; row += step) {
    f.next(row);
    const bool there = row < a.n;
    float g[RN_ELEMS], h[RN_ELEMS], w[RN_ELEMS], none = 0.0f;
    if (a.pre != DGS_NORM_NONE && a.in[2].p != nullptr) {
      const float m = there && a.pre == DGS_NORM_LAYER ? a.mean[row] : 0.0f, r = there ? a.rstd[row] : 0.0f;
      f.get(0, slot[0], row, there, h, smem);
      f.get(2, slot[2], row, there, g, smem);
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) {
        h[i] = f.in(i / VEC) ? (h[i] - m) * r : 0.0f;
        sums[0][i] = fmaf(g[i], h[i], sums[0][i]);
        sums[1][i] += g[i];
      }
      f.param(a.weight, 1.0f, w);
      norm_back<TPR, VEC>(f, a.pre == DGS_NORM_LAYER, a.D, r, w, h, g, &none, red[0]);
    } else {
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) g[i] = 0.0f;
    }
    if (a.in[3].p != nullptr) {
      f.get(3, slot[3], row, there, w, smem);
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) g[i] += w[i];
    }
    if (a.dx != nullptr) {
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) w[i] = a.xs * g[i];
      f.put(a.dx, row, there, w);
    }
    float r = 0.0f;
    f.get(1, slot[1], row, there, h, smem);
    if (a.post != DGS_NORM_NONE) {
      const float m = there && a.post == DGS_NORM_LAYER ? a.post_mean[row] : 0.0f;
      r = there ? a.post_rstd[row] : 0.0f;
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) h[i] = f.in(i / VEC) ? (h[i] - m) * r : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < RN_ELEMS; ++i) g[i] *= a.ys;
    float of_row = 0.0f;
    if (a.dgate != nullptr || a.column_gate != nullptr) {
      // the gate's gradient: g times post(y)
      float z[RN_ELEMS];
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) z[i] = h[i];
      if (a.post != DGS_NORM_NONE) {
        f.param(a.post_weight, 1.0f, w);
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) z[i] *= w[i];
        if (a.post_bias != nullptr) {
          f.param(a.post_bias, 0.0f, w);
#pragma unroll
          for (int i = 0; i < RN_ELEMS; ++i) z[i] += w[i];
        }
      }
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) z[i] *= g[i];
      if (a.column_gate != nullptr) {
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) sums[4][i] += z[i];
      } else if (a.row_gate != nullptr) {
#pragma unroll
        for (int i = 0; i < RN_ELEMS; ++i) of_row += z[i];
      } else {
        f.put(a.dgate, row, there, z);
      }
    }
    if (a.in[4].p != nullptr) {
      f.get(4, slot[4], row, there, w, smem);
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) g[i] *= w[i];
    } else if (a.column_gate != nullptr) {
      f.param(a.column_gate, 1.0f, w);
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) g[i] *= w[i];
    } else if (a.row_gate != nullptr) {
      const float by = there ? to_float<T>(static_cast<const T*>(a.row_gate)[row]) : 0.0f;
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) g[i] *= by;
    }
    f.done();
    if (a.post != DGS_NORM_NONE) {
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) {
        sums[2][i] = fmaf(g[i], h[i], sums[2][i]);
        sums[3][i] += g[i];
      }
      f.param(a.post_weight, 1.0f, w);
      norm_back<TPR, VEC>(f, a.post == DGS_NORM_LAYER, a.D, r, w, h, g, &of_row, red[1]);
    } else if (a.row_gate != nullptr) {
      float s[1] = {of_row};
      row_sums<TPR, 1>(s, red[1]);
      of_row = s[0];
    }
    if (a.dy != nullptr) f.put(a.dy, row, there, g);
    if (a.row_gate != nullptr && a.dgate != nullptr && there && f.t == 0) static_cast<T*>(a.dgate)[row] = from_float<T>(of_row);
    if constexpr (TPR > 32) {
      // (a row with one sum alone: `red` must not be written before all have read it)
      if (a.pre == DGS_NORM_NONE || a.in[2].p == nullptr || (a.post == DGS_NORM_NONE && a.row_gate == nullptr)) __syncthreads();
    }
  }
  if (a.partial == nullptr) return;
  float* to = a.partial + static_cast<int64_t>(blockIdx.x) * RN_SUMS * a.D;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int q = 0; q < RN_SUMS; ++q)
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i)
        if (f.in(i / VEC)) to[q * a.D + f.column(i / VEC) + i % VEC] = sums[q][i];
  } else {
    // the CTA's groups, in their order
    constexpr int WIDTH = TPR * RN_ELEMS;
    float* all = reinterpret_cast<float*>(smem);  // [ROWS][WIDTH]
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int q = 0; q < RN_SUMS; ++q) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < RN_ELEMS; ++i) all[(threadIdx.x / TPR) * WIDTH + f.column(i / VEC) + i % VEC] = sums[q][i];
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += THREADS) {
        float s = 0.0f;
        for (int r = 0; r < ROWS; ++r) s += all[r * WIDTH + c];
        to[q * a.D + c] = s;
      }
    }
  }
}

struct JoinArgs {
  const float* partial;
  int32_t partials, D, param_dtype;
  void* to[RN_SUMS];
};
// partial rows added in their order: 32 columns a CTA, a warp for every 32nd row
__global__ __launch_bounds__(RN_JOIN_THREADS) void residual_norm_join_kernel(const __grid_constant__ JoinArgs a) {
  __shared__ float part[32][33];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = blockIdx.y, c = blockIdx.x * 32 + lane;
  if (a.to[q] == nullptr) return;
  float s = 0.0f;
  if (c < a.D)
    for (int r = warp; r < a.partials; r += 32) s += a.partial[(static_cast<int64_t>(r) * RN_SUMS + q) * a.D + c];
  part[warp][lane] = s;
  __syncthreads();
  s = part[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL_MASK, s, o);
  const int column = blockIdx.x * 32 + warp;
  if (lane == 0 && column < a.D) store_from_float(a.to[q], a.param_dtype, column, s);
}

// ---- host ------------------------------------------------------------------------------------------------------------
int64_t partial_rows(int64_t n) {
  const int64_t most = static_cast<int64_t>(sm_count()) * RN_MAX_CTAS_PER_SM;
  return n < most ? n : most;
}

template <typename T, int VEC, int TPR, bool BACK>
int launch_rows(NormArgs a, int arrays, int* ctas, cudaStream_t s) {
  constexpr int THREADS = threads_of<TPR>(), ROWS = THREADS / TPR, NV = RN_ELEMS / VEC;
  constexpr bool ring = sizeof(T) * VEC == 16;
  void (*kernel)(NormArgs);
  if constexpr (BACK) kernel = residual_norm_backward_kernel<T, VEC, TPR>;
  else kernel = residual_norm_kernel<T, VEC, TPR>;
  // two CTAs of up to 256 threads or one larger one fill the SM's registers; what they have under way, its shared memory
  constexpr int room = THREADS <= 256 ? RN_MAX_SMEM / 2 : RN_MAX_SMEM;
  a.stage_bytes = ring ? arrays * NV * THREADS * 16 : 0;
  a.stages = !ring ? 1 : a.stage_bytes * RN_MAX_STAGES <= room ? RN_MAX_STAGES : room / a.stage_bytes;
  size_t smem = static_cast<size_t>(a.stages) * a.stage_bytes;
  const size_t joined = BACK && ROWS > 1 ? static_cast<size_t>(THREADS) * RN_ELEMS * sizeof(float) : 0;
  if (smem < joined) smem = joined;
  // CTAs that an SM holds of it, known for the size that was asked for last (two host calls less)
  static std::atomic<int64_t> known[RN_MAX_DEVICES] = {};
  int dev = 0;
  DGS_CUDA_TRY(cudaGetDevice(&dev));
  std::atomic<int64_t>& last = known[dev < RN_MAX_DEVICES ? dev : 0];
  const int64_t seen = last.load(std::memory_order_relaxed);
  int held = static_cast<int>(seen & 15);
  if (held == 0 || seen >> 4 != static_cast<int64_t>(smem) || dev >= RN_MAX_DEVICES) {
    DGS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RN_MAX_SMEM));
    DGS_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, THREADS, smem));
    if (held < 1) held = 1;
    if (held > RN_MAX_CTAS_PER_SM) held = RN_MAX_CTAS_PER_SM;
    last.store(static_cast<int64_t>(smem) << 4 | held, std::memory_order_relaxed);
  }
  const int64_t most = static_cast<int64_t>(sm_count()) * held, need = (a.n + ROWS - 1) / ROWS;
  *ctas = static_cast<int>(need < most ? need : most);
  DGS_CUDA_TRY(launch_training(kernel, dim3(static_cast<unsigned>(*ctas)), THREADS, smem, s, a));
  return DGS_OK;
}

template <typename T, int VEC, bool BACK>
int with_row(const NormArgs& a, int arrays, int* ctas, cudaStream_t s) {
  // eight elements a thread; the next wider form holds the rest
  const int threads = (a.D + RN_ELEMS - 1) / RN_ELEMS;
  if (threads <= 4) return launch_rows<T, VEC, 4, BACK>(a, arrays, ctas, s);
  if (threads <= 16) return launch_rows<T, VEC, 16, BACK>(a, arrays, ctas, s);
  if (threads <= 32) return launch_rows<T, VEC, 32, BACK>(a, arrays, ctas, s);
  if (threads <= 128) return launch_rows<T, VEC, 128, BACK>(a, arrays, ctas, s);
  if (threads <= 512) return launch_rows<T, VEC, 512, BACK>(a, arrays, ctas, s);
  return launch_rows<T, VEC, 1024, BACK>(a, arrays, ctas, s);
}

template <bool BACK>
int run_rows(const NormArgs& a, int32_t dtype, bool vectors, int arrays, int* ctas, cudaStream_t s) {
  if (dtype == DGS_F32)
    return vectors ? with_row<float, 4, BACK>(a, arrays, ctas, s) : with_row<float, 1, BACK>(a, arrays, ctas, s);
  if (dtype == DGS_BF16)
    return vectors ? with_row<__nv_bfloat16, 8, BACK>(a, arrays, ctas, s) : with_row<__nv_bfloat16, 1, BACK>(a, arrays, ctas, s);
  return vectors ? with_row<__half, 8, BACK>(a, arrays, ctas, s) : with_row<__half, 1, BACK>(a, arrays, ctas, s);
}

int check(const char* who, const dgs_residual_norm* p) {
  DGS_REQUIRE(p != nullptr, DGS_ERR_INVALID, "%s: null argument", who);
  DGS_REQUIRE(dtype_bytes(p->dtype) != 0 && dtype_bytes(p->param_dtype) != 0, DGS_ERR_UNSUPPORTED, "%s: element types %d and %d", who, p->dtype,
              p->param_dtype);
  DGS_REQUIRE(p->n >= 0 && p->D >= 1, DGS_ERR_INVALID, "%s: %lld rows of %lld elements", who, static_cast<long long>(p->n),
              static_cast<long long>(p->D));
  DGS_REQUIRE(p->D <= RN_MAX_D, DGS_ERR_UNSUPPORTED, "%s: rows of %lld elements (at most %d)", who, static_cast<long long>(p->D), RN_MAX_D);
  const auto norm = [](int32_t k) { return k == DGS_NORM_NONE || k == DGS_NORM_RMS || k == DGS_NORM_LAYER; };
  const auto gate = [](int32_t k) { return k == DGS_GATE_NONE || k == DGS_GATE_ROW || k == DGS_GATE_COLUMN || k == DGS_GATE_ELEMENT; };
  DGS_REQUIRE(norm(p->post) && norm(p->pre) && gate(p->gate_kind), DGS_ERR_INVALID, "%s: norms %d and %d, gate %d", who, p->post, p->pre,
              p->gate_kind);
  DGS_REQUIRE((p->gate_kind == DGS_GATE_NONE) == (p->gate == nullptr) || p->n == 0, DGS_ERR_INVALID, "%s: the gate and its kind", who);
  DGS_REQUIRE((p->post != DGS_NORM_NONE || (p->post_weight == nullptr && p->post_bias == nullptr)) &&
                  (p->pre != DGS_NORM_NONE || (p->weight == nullptr && p->bias == nullptr)),
              DGS_ERR_INVALID, "%s: a weight or bias without its norm", who);
  DGS_REQUIRE((p->post_weight != nullptr || p->post_bias == nullptr) && (p->weight != nullptr || p->bias == nullptr), DGS_ERR_INVALID,
              "%s: a bias without a weight", who);
  DGS_REQUIRE(p->y_stride >= p->D || p->n <= 1, DGS_ERR_INVALID, "%s: rows that overlap", who);
  DGS_REQUIRE(p->gate_kind != DGS_GATE_ELEMENT || p->gate_stride >= p->D || p->n <= 1, DGS_ERR_INVALID, "%s: rows that overlap", who);
  DGS_REQUIRE(p->eps >= 0.0f && p->x_scale - p->x_scale == 0.0f && p->y_scale - p->y_scale == 0.0f, DGS_ERR_INVALID,
              "%s: eps must be >= 0, the scales finite numbers", who);
  return DGS_OK;
}

NormArgs arguments(const dgs_residual_norm& p) {
  NormArgs a{};
  a.row_gate = p.gate_kind == DGS_GATE_ROW ? p.gate : nullptr;
  a.column_gate = p.gate_kind == DGS_GATE_COLUMN ? p.gate : nullptr;
  a.post_weight = p.post_weight;
  a.post_bias = p.post_bias;
  a.weight = p.weight;
  a.bias = p.bias;
  a.n = p.n;
  a.D = static_cast<int32_t>(p.D);
  a.param_dtype = p.param_dtype;
  a.post = p.post;
  a.pre = p.pre;
  a.xs = p.x_scale;
  a.ys = p.y_scale;
  a.eps = p.eps;
  return a;
}

// whether every row of every array can be moved in 16-byte vectors
bool in_vectors(const dgs_residual_norm& p, const NormArgs& a, int count, std::initializer_list<const void*> results) {
  const int64_t vec = 16 / dtype_bytes(p.dtype);
  if (p.D % vec != 0) return false;
  for (int q = 0; q < count; ++q)
    if (a.in[q].p != nullptr && (!aligned_to(a.in[q].p, 16) || (a.in[q].stride % vec != 0 && p.n > 1))) return false;
  for (const void* r : results)
    if (!aligned_to(r, 16)) return false;
  for (const void* w : {a.post_weight, a.post_bias, a.weight, a.bias, a.column_gate})
    if (!aligned_to(w, 16)) return false;
  return true;
}

}  // namespace
}  // namespace dgs

using namespace dgs;

extern "C" int dgs_residual_norm_forward(const dgs_residual_norm* p, const void* x, int64_t x_stride, void* sum, void* out, float* post_mean,
                                         float* post_rstd, float* mean, float* rstd, dgs_stream_t stream) {
  if (int rc = check("residual_norm", p)) return rc;
  if (p->n == 0) return DGS_OK;
  DGS_REQUIRE(x_stride >= p->D || p->n <= 1, DGS_ERR_INVALID, "residual_norm: rows that overlap");
  DGS_REQUIRE(x != nullptr && p->y != nullptr && sum != nullptr && (p->pre == DGS_NORM_NONE || (out != nullptr && rstd != nullptr)) &&
                  (p->pre != DGS_NORM_LAYER || mean != nullptr) && (p->post == DGS_NORM_NONE || post_rstd != nullptr) &&
                  (p->post != DGS_NORM_LAYER || post_mean != nullptr),
              DGS_ERR_INVALID, "residual_norm: null argument");
  NormArgs a = arguments(*p);
  a.in[0] = {x, x_stride};
  a.in[1] = {p->y, p->y_stride};
  if (p->gate_kind == DGS_GATE_ELEMENT) a.in[2] = {p->gate, p->gate_stride};
  a.sum = sum;
  a.out = out;
  a.post_mean = post_mean;
  a.post_rstd = post_rstd;
  a.mean = mean;
  a.rstd = rstd;
  int ctas = 0;
  return run_rows<false>(a, p->dtype, in_vectors(*p, a, 3, {sum, out}), a.in[2].p != nullptr ? 3 : 2, &ctas, static_cast<cudaStream_t>(stream));
}

extern "C" size_t dgs_residual_norm_backward_workspace_bytes(int64_t n, int64_t D) {
  if (n <= 0 || D <= 0) return 0;
  return static_cast<size_t>(partial_rows(n)) * RN_SUMS * static_cast<size_t>(D) * sizeof(float);
}

extern "C" int dgs_residual_norm_backward(const dgs_residual_norm* p, const void* sum, const void* dsum, int64_t dsum_stride, const void* dout,
                                          int64_t dout_stride, const float* post_mean, const float* post_rstd, const float* mean,
                                          const float* rstd, void* dx, void* dy, void* dgate, void* dpost_weight, void* dpost_bias,
                                          void* dweight, void* dbias, void* workspace, size_t workspace_bytes, dgs_stream_t stream) {
  if (int rc = check("residual_norm_backward", p)) return rc;
  DGS_REQUIRE(p->n <= 1 || ((dsum == nullptr || dsum_stride >= p->D) && (dout == nullptr || dout_stride >= p->D)), DGS_ERR_INVALID,
              "residual_norm_backward: rows that overlap");
  DGS_REQUIRE((p->post != DGS_NORM_NONE || (dpost_weight == nullptr && dpost_bias == nullptr)) &&
                  (p->pre != DGS_NORM_NONE || (dweight == nullptr && dbias == nullptr && dout == nullptr)) &&
                  (p->gate_kind != DGS_GATE_NONE || dgate == nullptr),
              DGS_ERR_INVALID, "residual_norm_backward: a gradient of what is absent");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool column = p->gate_kind == DGS_GATE_COLUMN;
  void* to[RN_SUMS] = {dweight, dbias, dpost_weight, dpost_bias, column ? dgate : nullptr};
  bool any = false;
  for (void* t : to) any |= t != nullptr;
  if (p->n == 0) {
    for (void* t : to)
      if (t != nullptr) DGS_CUDA_TRY(cudaMemsetAsync(t, 0, static_cast<size_t>(p->D) * dtype_bytes(p->param_dtype), s));
    return DGS_OK;
  }
  if (!any && dx == nullptr && dy == nullptr && dgate == nullptr) return DGS_OK;
  DGS_REQUIRE(p->y != nullptr && (p->pre == DGS_NORM_NONE || (sum != nullptr && rstd != nullptr)) &&
                  (p->pre != DGS_NORM_LAYER || mean != nullptr) && (p->post == DGS_NORM_NONE || post_rstd != nullptr) &&
                  (p->post != DGS_NORM_LAYER || post_mean != nullptr),
              DGS_ERR_INVALID, "residual_norm_backward: null argument");
  const size_t need = any ? dgs_residual_norm_backward_workspace_bytes(p->n, p->D) : 0;
  DGS_REQUIRE(!any || (workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 16)), DGS_ERR_INVALID,
              "residual_norm_backward: workspace of %zu bytes, 16-byte aligned, is needed", need);
  NormArgs a = arguments(*p);
  if (p->pre != DGS_NORM_NONE && dout != nullptr) a.in[0] = {sum, p->D};
  a.in[1] = {p->y, p->y_stride};
  a.in[2] = {dout, dout_stride};
  a.in[3] = {dsum, dsum_stride};
  if (p->gate_kind == DGS_GATE_ELEMENT) a.in[4] = {p->gate, p->gate_stride};
  a.post_mean = const_cast<float*>(post_mean);
  a.post_rstd = const_cast<float*>(post_rstd);
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dx = dx;
  a.dy = dy;
  a.dgate = column ? nullptr : dgate;
  a.partial = any ? static_cast<float*>(workspace) : nullptr;
  int arrays = 0, ctas = 0;
  for (const Source& in : a.in) arrays += in.p != nullptr;
  if (int rc = run_rows<true>(a, p->dtype, in_vectors(*p, a, 5, {dx, dy, a.dgate}), arrays, &ctas, s)) return rc;
  if (!any) return DGS_OK;
  JoinArgs j{a.partial, ctas, a.D, p->param_dtype, {}};
  for (int q = 0; q < RN_SUMS; ++q) j.to[q] = to[q];
  DGS_CUDA_TRY(launch_training(residual_norm_join_kernel, dim3(static_cast<unsigned>((p->D + 31) / 32), RN_SUMS), RN_JOIN_THREADS, 0, s, j));
  return DGS_OK;
}
