// Layer norm: forward, and backward with the reduction of the weight's and the bias's gradient.
//
//   mean_i = avg_j x_ij,  rstd_i = 1 / sqrt(avg_j (x_ij - mean_i)^2 + eps),  h_ij = (x_ij - mean_i) rstd_i,  y = h w + b
//   g = dy w,  dx_ij = rstd_i (g_ij - avg_j g_ij - h_ij avg_j (g_ij h_ij)),  dw_j = sum_i dy_ij h_ij,  db_j = sum_i dy_ij
//
// Both directions read every element once and are bound by HBM.  A row stays in the registers of the threads that share
// it between its passes (mean, centred squares, result), so the variance is that of the centred values and does not
// cancel.  All sums are in 32 bits.
//   - TPR threads share a row, NV vectors of VEC elements each: 4 to 32 threads of a warp (shuffles alone), or a whole
//     CTA for rows beyond a warp's registers; rows that no variant holds go through kernels that read them again.
//   - Backward: a thread keeps the same columns for all rows of its CTA, so the column sums grow in its registers; each
//     CTA writes one partial row and a second launch adds the partial rows in their order.  No atomics: the same inputs
//     give the same bits.
#include "train_common.cuh"

namespace dgs {
namespace {

constexpr int LN_THREADS = 256;

struct NormArgs {
  const void* x;
  int64_t x_stride;
  const void* weight;
  const void* bias;
  int32_t param_dtype;
  int64_t n;
  int D;
  float eps;
  void* y;
  float* mean;
  float* rstd;
};

// Sum over the TPR threads that share a row, returned to all of them.  Every thread of the CTA calls it.  `red` (TPR ==
// LN_THREADS): one float per warp, not written again before every thread has passed another CTA-wide sum.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  if constexpr (TPR > 32) {
    constexpr int NW = LN_THREADS / 32;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += red[w];
  }
  return v;
}

template <int VEC>
__device__ __forceinline__ void load_param(const void* p, int32_t dtype, int64_t i, float absent, float (&out)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) out[k] = absent;
  } else if constexpr (VEC == 1) {
    out[0] = load_as_float(p, dtype, i);
  } else {
    load_vec_as_float<VEC>(p, dtype, i, out);
  }
}

template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(LN_THREADS) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int ROWS = LN_THREADS / TPR;
  constexpr bool KEEP = VEC * NV <= 16;  // the parameters of a thread's columns stay in its registers
  __shared__ float red[2][LN_THREADS / 32];
  pdl_enter();
  const int t = threadIdx.x % TPR;
  const int nvec = a.D / VEC;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  float w[KEEP ? NV : 1][VEC], b[KEEP ? NV : 1][VEC];
  if constexpr (KEEP) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = t + k * TPR;
      if (c < nvec) {
        load_param<VEC>(a.weight, a.param_dtype, c * VEC, 1.0f, w[k]);
        load_param<VEC>(a.bias, a.param_dtype, c * VEC, 0.0f, b[k]);
      }
    }
  }
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS; row0 < a.n; row0 += static_cast<int64_t>(gridDim.x) * ROWS) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.n;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float v[NV][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = t + k * TPR;
      if (live && c < nvec) {
        load_vec<T, VEC>(x + c * VEC, v[k]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k][i] = 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += v[k][i];
    const float mean = row_sum<TPR>(sum, red[0]) * inv_d;
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (t + k * TPR < nvec) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[k][i] -= mean;
          sq += v[k][i] * v[k][i];
        }
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, red[1]) * inv_d + a.eps);
    if (live) {
      T* y = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = t + k * TPR;
        if (c < nvec) {
          float wk[VEC], bk[VEC];
          if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) wk[i] = w[k][i], bk[i] = b[k][i];
          } else {
            load_param<VEC>(a.weight, a.param_dtype, c * VEC, 1.0f, wk);
            load_param<VEC>(a.bias, a.param_dtype, c * VEC, 0.0f, bk);
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[k][i] = v[k][i] * rstd * wk[i] + bk[i];
          store_vec<T, VEC>(y + c * VEC, v[k]);
        }
      }
      if (t == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
  }
}

// Sum over the CTA, for kernels whose rows are read again (`red`: one float per warp)
__device__ __forceinline__ float cta_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  __syncthreads();  // the sum before this one has been read
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < LN_THREADS / 32; ++w) v += red[w];
  return v;
}

// Rows wider than any register variant holds: three passes, the second and third of them out of L2
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) norm_forward_wide_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[LN_THREADS / 32];
  pdl_enter();
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* y = static_cast<T*>(a.y) + row * a.D;
    float sum = 0.0f, sq = 0.0f;
    for (int j = threadIdx.x; j < a.D; j += LN_THREADS) sum += to_float<T>(x[j]);
    const float mean = cta_sum(sum, red) / static_cast<float>(a.D);
    for (int j = threadIdx.x; j < a.D; j += LN_THREADS) {
      const float c = to_float<T>(x[j]) - mean;
      sq += c * c;
    }
    const float rstd = 1.0f / sqrtf(cta_sum(sq, red) / static_cast<float>(a.D) + a.eps);
    for (int j = threadIdx.x; j < a.D; j += LN_THREADS) {
      float w[1], b[1];
      load_param<1>(a.weight, a.param_dtype, j, 1.0f, w);
      load_param<1>(a.bias, a.param_dtype, j, 0.0f, b);
      y[j] = from_float<T>((to_float<T>(x[j]) - mean) * rstd * w[0] + b[0]);
    }
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

struct NormBackArgs {
  const void* dy;
  int64_t dy_stride;
  const void* x;
  int64_t x_stride;
  const void* weight;
  int32_t param_dtype;
  const float* mean;
  const float* rstd;
  int64_t n;
  int D;
  void* dx;        // may be null
  float* partial;  // [CTAs][2][D], or null when the parameters' gradients are not wanted
};

template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(LN_THREADS) norm_backward_kernel(const __grid_constant__ NormBackArgs a) {
  constexpr int ROWS = LN_THREADS / TPR;
  constexpr bool KEEP = VEC * NV <= 16;
  __shared__ float red[4][LN_THREADS / 32];
  __shared__ float merge[ROWS > 1 ? LN_THREADS * VEC : 1];
  pdl_enter();
  const int t = threadIdx.x % TPR;
  const int nvec = a.D / VEC;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  float w[KEEP ? NV : 1][VEC];
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0.0f;
    const int c = t + k * TPR;
    if constexpr (KEEP) {
      if (c < nvec) load_param<VEC>(a.weight, a.param_dtype, c * VEC, 1.0f, w[k]);
    }
  }
  int parity = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS; row0 < a.n; row0 += static_cast<int64_t>(gridDim.x) * ROWS) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const bool live = row < a.n;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    float h[NV][VEC], g[NV][VEC];
    const float mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = t + k * TPR;
      if (live && c < nvec) {
        load_vec<T, VEC>(x + c * VEC, h[k]);
        load_vec<T, VEC>(dy + c * VEC, g[k]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[k][i] = g[k][i] = 0.0f;
      }
    }
    float sg = 0.0f, sgh = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = t + k * TPR;
      if (live && c < nvec) {
        float wk[VEC];
        if constexpr (KEEP) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) wk[i] = w[k][i];
        } else {
          load_param<VEC>(a.weight, a.param_dtype, c * VEC, 1.0f, wk);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          h[k][i] = (h[k][i] - mean) * rstd;
          dw[k][i] += g[k][i] * h[k][i];
          db[k][i] += g[k][i];
          g[k][i] *= wk[i];
          sg += g[k][i];
          sgh += g[k][i] * h[k][i];
        }
      }
    }
    if (a.dx != nullptr) {
      // two buffers in turn: a CTA-wide sum of the next row may begin while another thread still reads this one's
      sg = row_sum<TPR>(sg, red[parity]) * inv_d;
      sgh = row_sum<TPR>(sgh, red[2 + parity]) * inv_d;
      parity ^= 1;
      if (live) {
        T* dx = static_cast<T*>(a.dx) + row * a.D;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = t + k * TPR;
          if (c < nvec) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) g[k][i] = rstd * (g[k][i] - sg - h[k][i] * sgh);
            store_vec<T, VEC>(dx + c * VEC, g[k]);
          }
        }
      }
    }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.D;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = t + k * TPR;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float* mine = half == 0 ? dw[k] : db[k];
      if constexpr (ROWS > 1) {  // the CTA's row groups, added in their order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) merge[threadIdx.x * VEC + i] = mine[i];
        __syncthreads();
        if (threadIdx.x < TPR) {
#pragma unroll
          for (int r = 1; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < VEC; ++i) mine[i] += merge[(r * TPR + t) * VEC + i];
        }
      }
      if (threadIdx.x < TPR && c < nvec) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[half * a.D + c * VEC + i] = mine[i];
      }
    }
  }
}

// dx of rows wider than the register variants hold
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) norm_backward_wide_kernel(const __grid_constant__ NormBackArgs a) {
  __shared__ float red[LN_THREADS / 32];
  pdl_enter();
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    T* dx = static_cast<T*>(a.dx) + row * a.D;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.0f, sgh = 0.0f, w[1];
    for (int j = threadIdx.x; j < a.D; j += LN_THREADS) {
      load_param<1>(a.weight, a.param_dtype, j, 1.0f, w);
      const float g = to_float<T>(dy[j]) * w[0];
      sg += g;
      sgh += g * (to_float<T>(x[j]) - mean) * rstd;
    }
    sg = cta_sum(sg, red) / static_cast<float>(a.D);
    sgh = cta_sum(sgh, red) / static_cast<float>(a.D);
    for (int j = threadIdx.x; j < a.D; j += LN_THREADS) {
      load_param<1>(a.weight, a.param_dtype, j, 1.0f, w);
      const float g = to_float<T>(dy[j]) * w[0];
      dx[j] = from_float<T>(rstd * (g - sg - (to_float<T>(x[j]) - mean) * rstd * sgh));
    }
  }
}

// Column sums for the same rows: a CTA takes LN_THREADS columns and every gridDim.y-th row
template <typename T>
__global__ void __launch_bounds__(LN_THREADS) norm_columns_wide_kernel(const __grid_constant__ NormBackArgs a) {
  pdl_enter();
  const int j = blockIdx.x * LN_THREADS + threadIdx.x;
  if (j >= a.D) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.n; row += gridDim.y) {
    const float g = to_float<T>(static_cast<const T*>(a.dy)[row * a.dy_stride + j]);
    const float h = (to_float<T>(static_cast<const T*>(a.x)[row * a.x_stride + j]) - a.mean[row]) * a.rstd[row];
    dw += g * h;
    db += g;
  }
  float* out = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.D;
  out[j] = dw;
  out[a.D + j] = db;
}

// Adds `count` partial rows [2][D]: 32 columns a CTA, 8 warps that take every eighth partial row each
__global__ void __launch_bounds__(LN_THREADS) norm_join_kernel(const float* __restrict__ partial, int count, int D,
                                                               void* dweight, void* dbias, int32_t dtype) {
  __shared__ float part[LN_THREADS / 32][33];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;  // of 2 D columns: the weight's, then the bias's
  float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
  if (j < 2 * D) {
    const float* p = partial + j;
    const int64_t step = 2 * static_cast<int64_t>(D);
    int r = warp;
    for (; r + 24 < count; r += 32) {
      s0 += p[r * step];
      s1 += p[(r + 8) * step];
      s2 += p[(r + 16) * step];
      s3 += p[(r + 24) * step];
    }
    for (; r < count; r += 8) s0 += p[r * step];
  }
  part[warp][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (warp == 0 && j < 2 * D) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < LN_THREADS / 32; ++w) s += part[w][lane];
    if (j < D) store_from_float(dweight, dtype, j, s);
    else store_from_float(dbias, dtype, j - D, s);
  }
}

// Threads per row and vectors per thread that hold `nvec` vectors; TPR == 0: none does.
struct Shape {
  int tpr, nv;
};
inline Shape shape_for(int64_t nvec, int vec, int most_values) {
  for (int tpr = 4; tpr <= 32; tpr *= 2)
    if (nvec <= tpr) return {tpr, 1};
  for (int tpr = 32; tpr <= LN_THREADS; tpr *= LN_THREADS / 32)
    for (int nv = tpr == 32 ? 2 : 1; nv * vec <= (tpr == 32 ? 32 : most_values); nv *= 2)
      if (nvec <= static_cast<int64_t>(tpr) * nv) return {tpr, nv};
  return {0, 0};
}

constexpr int LN_FORWARD_VALUES = 64, LN_BACKWARD_VALUES = 32;  // values of a row that one thread holds
constexpr int LN_WIDE_SPLITS = 64;

template <typename T>
constexpr int full_vec() {
  return 16 / static_cast<int>(sizeof(T));
}

inline int64_t ctas_for(int64_t n, int rows, int per_sm) {
  const int64_t need = (n + rows - 1) / rows, most = static_cast<int64_t>(sm_count()) * per_sm;
  return need < most ? need : most;
}

// f.template run<VEC, TPR, NV>() for a shape, f.run_wide() where no variant holds the row
template <int VEC, typename F>
int with_shape(const Shape& s, const F& f) {
  constexpr int MOST = F::kMostValues;
  switch (s.tpr) {
    case 4: return f.template run<VEC, 4, 1>();
    case 8: return f.template run<VEC, 8, 1>();
    case 16: return f.template run<VEC, 16, 1>();
    case 32:
      if (s.nv == 1) return f.template run<VEC, 32, 1>();
      if (s.nv == 2) return f.template run<VEC, 32, 2>();
      if (s.nv == 4) return f.template run<VEC, 32, 4>();
      if constexpr (VEC <= 4)
        if (s.nv == 8) return f.template run<VEC, 32, 8>();
      if constexpr (VEC == 1) {
        if (s.nv == 16) return f.template run<VEC, 32, 16>();
        if (s.nv == 32) return f.template run<VEC, 32, 32>();
      }
      break;
    case LN_THREADS:
      if (s.nv == 1) return f.template run<VEC, LN_THREADS, 1>();
      if (s.nv == 2) return f.template run<VEC, LN_THREADS, 2>();
      if (s.nv == 4) return f.template run<VEC, LN_THREADS, 4>();
      if constexpr (VEC * 8 <= MOST)
        if (s.nv == 8) return f.template run<VEC, LN_THREADS, 8>();
      if constexpr (VEC * 16 <= MOST)
        if (s.nv == 16) return f.template run<VEC, LN_THREADS, 16>();
      if constexpr (VEC * 32 <= MOST)
        if (s.nv == 32) return f.template run<VEC, LN_THREADS, 32>();
      if constexpr (VEC * 64 <= MOST)
        if (s.nv == 64) return f.template run<VEC, LN_THREADS, 64>();
      break;
    default: break;
  }
  return f.run_wide();
}

template <typename T>
struct Forward {
  static constexpr int kMostValues = LN_FORWARD_VALUES;
  const NormArgs& a;
  cudaStream_t s;
  template <int VEC, int TPR, int NV>
  int run() const {
    DGS_CUDA_TRY(launch_training(norm_forward_kernel<T, VEC, TPR, NV>, dim3(static_cast<unsigned>(ctas_for(a.n, LN_THREADS / TPR, 8))),
                                 LN_THREADS, 0, s, a));
    return DGS_OK;
  }
  int run_wide() const {
    DGS_CUDA_TRY(launch_training(norm_forward_wide_kernel<T>, dim3(static_cast<unsigned>(ctas_for(a.n, 1, 8))), LN_THREADS, 0, s, a));
    return DGS_OK;
  }
};

template <typename T>
int forward(const NormArgs& a, cudaStream_t s) {
  constexpr int VEC = full_vec<T>();
  const bool whole = a.D % VEC == 0 && a.x_stride % VEC == 0 && aligned_to(a.x, 16) && aligned_to(a.y, 16) &&
                     aligned_to(a.weight, 16) && aligned_to(a.bias, 16);
  const Forward<T> f{a, s};
  if (whole) return with_shape<VEC>(shape_for(a.D / VEC, VEC, LN_FORWARD_VALUES), f);
  return with_shape<1>(shape_for(a.D, 1, LN_FORWARD_VALUES), f);
}

// CTAs of the backward launch, each of which writes a partial row
inline int64_t backward_ctas(int64_t n, int tpr) { return ctas_for(n, LN_THREADS / tpr, 4); }

template <typename T>
struct Backward {
  static constexpr int kMostValues = LN_BACKWARD_VALUES;
  const NormBackArgs& a;
  cudaStream_t s;
  int64_t* partials;
  template <int VEC, int TPR, int NV>
  int run() const {
    *partials = backward_ctas(a.n, TPR);
    DGS_CUDA_TRY(launch_training(norm_backward_kernel<T, VEC, TPR, NV>, dim3(static_cast<unsigned>(*partials)), LN_THREADS, 0, s, a));
    return DGS_OK;
  }
  int run_wide() const {
    if (a.dx != nullptr)
      DGS_CUDA_TRY(launch_training(norm_backward_wide_kernel<T>, dim3(static_cast<unsigned>(ctas_for(a.n, 1, 8))), LN_THREADS, 0, s, a));
    *partials = a.n < LN_WIDE_SPLITS ? a.n : LN_WIDE_SPLITS;
    if (a.partial != nullptr)
      DGS_CUDA_TRY(launch_training(norm_columns_wide_kernel<T>,
                                   dim3(static_cast<unsigned>((a.D + LN_THREADS - 1) / LN_THREADS), static_cast<unsigned>(*partials)),
                                   LN_THREADS, 0, s, a));
    return DGS_OK;
  }
};

template <typename T>
int backward(const NormBackArgs& a, int64_t* partials, cudaStream_t s) {
  constexpr int VEC = full_vec<T>();
  const bool whole = a.D % VEC == 0 && a.x_stride % VEC == 0 && a.dy_stride % VEC == 0 && aligned_to(a.x, 16) &&
                     aligned_to(a.dy, 16) && aligned_to(a.dx, 16) && aligned_to(a.weight, 16);
  const Backward<T> f{a, s, partials};
  if (whole) return with_shape<VEC>(shape_for(a.D / VEC, VEC, LN_BACKWARD_VALUES), f);
  return with_shape<1>(shape_for(a.D, 1, LN_BACKWARD_VALUES), f);
}

int check_sizes(const char* who, int64_t n, int64_t D, int32_t dtype, int32_t param_dtype) {
  DGS_REQUIRE(n >= 0 && D >= 1 && D <= (int64_t(1) << 29), DGS_ERR_INVALID, "%s: %lld rows of %lld elements", who,
              static_cast<long long>(n), static_cast<long long>(D));
  DGS_REQUIRE(dtype_bytes(dtype) != 0, DGS_ERR_UNSUPPORTED, "%s: element type %d", who, dtype);
  DGS_REQUIRE(dtype_bytes(param_dtype) != 0, DGS_ERR_UNSUPPORTED, "%s: element type %d of the parameters", who, param_dtype);
  return DGS_OK;
}

}  // namespace
}  // namespace dgs

using namespace dgs;

extern "C" int dgs_layer_norm(const void* x, int64_t x_stride, int32_t dtype, const void* weight, const void* bias,
                              int32_t param_dtype, int64_t n, int64_t D, float eps, void* y, float* mean, float* rstd,
                              dgs_stream_t stream) {
  if (int rc = check_sizes("layer_norm", n, D, dtype, param_dtype)) return rc;
  DGS_REQUIRE(x_stride >= D || n <= 1, DGS_ERR_INVALID, "layer_norm: rows of %lld elements %lld apart", static_cast<long long>(D),
              static_cast<long long>(x_stride));
  DGS_REQUIRE(eps >= 0.0f, DGS_ERR_INVALID, "layer_norm: eps must be >= 0");
  DGS_REQUIRE(weight != nullptr || bias == nullptr, DGS_ERR_INVALID, "layer_norm: a bias without a weight");
  if (n == 0) return DGS_OK;
  DGS_REQUIRE(x != nullptr && y != nullptr && mean != nullptr && rstd != nullptr, DGS_ERR_INVALID, "layer_norm: null argument");
  const NormArgs a{x, x_stride, weight, bias, param_dtype, n, static_cast<int>(D), eps, y, mean, rstd};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == DGS_F32 ? forward<float>(a, s) : dtype == DGS_BF16 ? forward<__nv_bfloat16>(a, s) : forward<__half>(a, s);
}

extern "C" size_t dgs_layer_norm_backward_workspace_bytes(int64_t n, int64_t D) {
  if (n <= 0 || D <= 0) return 0;
  // an upper bound over all variants: one partial row for each CTA, of which no variant launches more than rows
  const int64_t most = static_cast<int64_t>(sm_count()) * 4;
  int64_t partials = most > LN_WIDE_SPLITS ? most : LN_WIDE_SPLITS;
  if (n < partials) partials = n;
  return static_cast<size_t>(partials) * 2 * static_cast<size_t>(D) * sizeof(float);
}

extern "C" int dgs_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int32_t dtype,
                                       const void* weight, int32_t param_dtype, const float* mean, const float* rstd, int64_t n,
                                       int64_t D, void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                                       dgs_stream_t stream) {
  if (int rc = check_sizes("layer_norm_backward", n, D, dtype, param_dtype)) return rc;
  DGS_REQUIRE((x_stride >= D && dy_stride >= D) || n <= 1, DGS_ERR_INVALID,
              "layer_norm_backward: rows of %lld elements %lld and %lld apart", static_cast<long long>(D),
              static_cast<long long>(x_stride), static_cast<long long>(dy_stride));
  DGS_REQUIRE((dweight == nullptr) == (dbias == nullptr), DGS_ERR_INVALID,
              "layer_norm_backward: the gradients of weight and bias come together");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    if (dweight != nullptr) {
      DGS_CUDA_TRY(cudaMemsetAsync(dweight, 0, D * dtype_bytes(param_dtype), s));
      DGS_CUDA_TRY(cudaMemsetAsync(dbias, 0, D * dtype_bytes(param_dtype), s));
    }
    return DGS_OK;
  }
  if (dx == nullptr && dweight == nullptr) return DGS_OK;
  DGS_REQUIRE(dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr, DGS_ERR_INVALID,
              "layer_norm_backward: null argument");
  const size_t need = dgs_layer_norm_backward_workspace_bytes(n, D);
  DGS_REQUIRE(dweight == nullptr || (workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 16)), DGS_ERR_INVALID,
              "layer_norm_backward: workspace of %zu bytes, 16-byte aligned, is needed", need);
  const NormBackArgs a{dy,   dy_stride, x, x_stride,            weight, param_dtype,
                       mean, rstd,      n, static_cast<int>(D), dx,     dweight != nullptr ? static_cast<float*>(workspace) : nullptr};
  int64_t partials = 0;
  const int rc = dtype == DGS_F32    ? backward<float>(a, &partials, s)
                 : dtype == DGS_BF16 ? backward<__nv_bfloat16>(a, &partials, s)
                                     : backward<__half>(a, &partials, s);
  if (rc != DGS_OK || dweight == nullptr) return rc;
  DGS_CUDA_TRY(launch_training(norm_join_kernel, dim3(static_cast<unsigned>((2 * D + 31) / 32)), LN_THREADS, 0, s, a.partial,
                               static_cast<int>(partials), a.D, dweight, dbias, param_dtype));
  return DGS_OK;
}
