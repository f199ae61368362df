// Layer norm: forward, and backward with the reduction of the weight's and the bias's gradient.
//
//   mean_i = avg_j x_ij,  rstd_i = 1 / sqrt(avg_j (x_ij - mean_i)^2 + eps),  h_ij = (x_ij - mean_i) rstd_i,  y = h w + b
//   g = dy w,  dx_ij = rstd_i (g_ij - avg_j g_ij - h_ij avg_j (g_ij h_ij)),  dw_j = sum_i dy_ij h_ij,  db_j = sum_i dy_ij
//
// Both directions read every element once and are bound by HBM: 430 000 x 100 float32 57 us forward and 80 us backward (6.0 and
// 6.4 TB/s), 16 384 x 4 096 bfloat16 46 and 78 us (5.8 and 5.2 TB/s; two sums over the CTA stand between a row's loads and
// stores).  A row stays in the registers of the threads that share it between its passes (mean, centred squares, result), so
// the variance is that of the centred values and does not cancel.  All sums are in 32 bits.
//   - TPR threads share a row, NV vectors of VEC elements each: 4 to 32 threads of a warp (shuffles alone), or a CTA of 256
//     or 512 for rows beyond a warp's registers; rows that no variant holds go through kernels that read them again.
//   - Backward: a thread keeps the same columns for all rows of its CTA, so the column sums grow in its registers; each
//     CTA writes one partial row and a second launch adds the partial rows in their order; rows that one cluster takes at
//     once are added out of its CTAs' shared memory instead.  No atomics: the same inputs give the same bits.
#include "train_common.cuh"

namespace dgs {
namespace {

constexpr int LN_THREADS = 256;
// threads of a CTA whose threads share rows TPR at a time
template <int TPR>
constexpr int threads_of() {
  return TPR > LN_THREADS ? TPR : LN_THREADS;
}

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

// Sums over the TPR threads that share a row, returned to all of them: COUNT of them together.  Every thread of the CTA calls
// it.  `red` (TPR > 32): not written again before every thread has passed another CTA-wide sum.
template <int TPR, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], float (*red)[COUNT]) {
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

// Rows that a thread group works on at a time: R, whose sums run through the shuffles side by side.
template <int VEC, int TPR, int NV>
constexpr int rows_at_once() {
  return TPR <= 32 && VEC * NV <= 8 ? 2 : 1;
}

// The next rows are on their way while these are summed: HBM needs some 40 KB under way per SM, and a row of 100 floats is 400
// bytes.  Vectors of 16 bytes travel by cp.async into a ring of S stages in shared memory; a thread fetches what it will read
// itself, so its own wait is all the synchronisation there is, and what is under way costs no registers.  Narrower vectors
// (rows that do not begin at 16-byte boundaries) are fetched into registers, one stage ahead.
template <typename T, int VEC, int TPR, int NV, int R, int S, int COUNT>  // COUNT arrays
struct Rows {
  static constexpr bool kRing = sizeof(T) * VEC == 16;
  static constexpr uint32_t kStageBytes = COUNT * R * NV * threads_of<TPR>() * 16;
  Vec<T, VEC> raw[COUNT][R][NV];
  const T* base[COUNT];
  int64_t stride[COUNT];
  int64_t n, step;
  int t, nvec, stage;
  uint32_t ring;

  __device__ __forceinline__ void issue(int64_t row0, int st) {
#pragma unroll
    for (int q = 0; q < COUNT; ++q)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const T* p = base[q] + (row0 + r) * stride[q];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = t + k * TPR;
          if (row0 + r < n && c < nvec) {
            if constexpr (kRing)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + st * kStageBytes +
                                                                             (((q * R + r) * NV + k) * threads_of<TPR>() + threadIdx.x) * 16),
                           "l"(p + c * VEC)
                           : "memory");
            else
              raw[q][r][k] = *reinterpret_cast<const Vec<T, VEC>*>(p + c * VEC);
          }
        }
      }
    if constexpr (kRing) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // first rows of this thread's group
  __device__ __forceinline__ void begin(int64_t row0, unsigned char* smem) {
    stage = 0;
    if constexpr (kRing) {
      ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
#pragma unroll
      for (int s = 0; s < S - 1; ++s) issue(row0 + s * step, s);
    } else {
      issue(row0, 0);
    }
  }
  // raw = the rows at row0 (in the order of begin); then
  __device__ __forceinline__ void take() {
    if constexpr (kRing) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
#pragma unroll
      for (int q = 0; q < COUNT; ++q)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            uint4 v;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(ring + stage * kStageBytes + (((q * R + r) * NV + k) * threads_of<TPR>() + threadIdx.x) * 16)
                         : "memory");
            raw[q][r][k] = *reinterpret_cast<const Vec<T, VEC>*>(&v);
          }
    }
  }
  // ... once raw has been used, the rows that come S - 1 rounds (registers: one) after row0
  __device__ __forceinline__ void next(int64_t row0) {
    if constexpr (kRing) {
      issue(row0 + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);
      if (++stage == S) stage = 0;
    } else {
      issue(row0 + step, 0);
    }
  }
};
// Stages that keep a CTA's ring within 64 KB
template <typename T, int VEC, int TPR, int NV, int R, int COUNT>
constexpr int ring_stages() {
  constexpr int fit = 65536 / (COUNT * R * NV * threads_of<TPR>() * 16);
  return sizeof(T) * VEC != 16 ? 2 : fit > 6 ? 6 : fit < 2 ? 2 : fit;
}
template <typename T, int VEC, int TPR, int NV, int R, int COUNT>
constexpr size_t ring_bytes() {
  return sizeof(T) * VEC != 16 ? 0 : size_t(ring_stages<T, VEC, TPR, NV, R, COUNT>()) * COUNT * R * NV * threads_of<TPR>() * 16;
}

template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(threads_of<TPR>()) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int R = rows_at_once<VEC, TPR, NV>(), ROWS = threads_of<TPR>() / TPR * R, S = ring_stages<T, VEC, TPR, NV, R, 1>();
  constexpr bool KEEP = VEC * NV <= 16;  // the parameters of a thread's columns stay in its registers
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[2][threads_of<TPR>() / 32][R];
  pdl_enter();
  const int t = threadIdx.x % TPR;
  const int nvec = a.D / VEC;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR * R;
  Rows<T, VEC, TPR, NV, R, S, 1> rows;
  rows.base[0] = static_cast<const T*>(a.x);
  rows.stride[0] = a.x_stride;
  rows.n = a.n;
  rows.step = step;
  rows.t = t;
  rows.nvec = nvec;
  rows.begin(row0, ring);
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
  // (all groups of a CTA go round together: their first rows differ, not the number of rounds)
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.n; first += step, row0 += step) {
    float v[R][NV][VEC], mean[R], rstd[R];
    rows.take();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          v[r][k][i] = row0 + r < a.n && t + k * TPR < nvec ? to_float<T>(rows.raw[0][r][k].v[i]) : 0.0f;
    rows.next(row0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum += v[r][k][i];
      mean[r] = sum;
    }
    row_sums<TPR>(mean, red[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inv_d;
      float sq = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (t + k * TPR < nvec) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            v[r][k][i] -= mean[r];
            sq += v[r][k][i] * v[r][k][i];
          }
        }
      }
      rstd[r] = sq;
    }
    row_sums<TPR>(rstd, red[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) rstd[r] = 1.0f / sqrtf(rstd[r] * inv_d + a.eps);
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
        for (int r = 0; r < R; ++r) {
          if (row0 + r < a.n) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[r][k][i] = v[r][k][i] * rstd[r] * wk[i] + bk[i];
            store_vec<T, VEC>(static_cast<T*>(a.y) + (row0 + r) * a.D + c * VEC, v[r][k]);
          }
        }
      }
    }
    if (t == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row0 + r < a.n) {
          a.mean[row0 + r] = mean[r];
          a.rstd[row0 + r] = rstd[r];
        }
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
  float* partial;  // [CTAs][2][D], or null when the parameters' gradients are not wanted or are made here
  // few CTAs: one cluster, whose CTAs add their column sums out of one another's shared memory
  void *dweight, *dbias;
  int32_t ctas;
};

__device__ __forceinline__ float shared_of(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(threads_of<TPR>(), VEC * NV <= 16 ? 512 / threads_of<TPR>() : 1) norm_backward_kernel(const __grid_constant__ NormBackArgs a) {
  constexpr int R = rows_at_once<VEC, TPR, NV>(), GROUPS = threads_of<TPR>() / TPR, ROWS = GROUPS * R;
  constexpr int S = ring_stages<T, VEC, TPR, NV, R, 2>();
  constexpr bool KEEP = VEC * NV <= 16;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[2][threads_of<TPR>() / 32][2 * R];
  __shared__ float merge[GROUPS > 1 ? threads_of<TPR>() * VEC : 1];
  pdl_enter();
  const int t = threadIdx.x % TPR;
  const int nvec = a.D / VEC;
  const float inv_d = 1.0f / static_cast<float>(a.D);
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  int64_t row0 = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR * R;
  Rows<T, VEC, TPR, NV, R, S, 2> rows;
  rows.base[0] = static_cast<const T*>(a.x);
  rows.base[1] = static_cast<const T*>(a.dy);
  rows.stride[0] = a.x_stride;
  rows.stride[1] = a.dy_stride;
  rows.n = a.n;
  rows.step = step;
  rows.t = t;
  rows.nvec = nvec;
  float next_mean[R], next_rstd[R];
  auto statistics = [&](int64_t at) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      next_mean[r] = at + r < a.n ? a.mean[at + r] : 0.0f;
      next_rstd[r] = at + r < a.n ? a.rstd[at + r] : 0.0f;
    }
  };
  rows.begin(row0, ring);
  statistics(row0);
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
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.n; first += step, row0 += step) {
    float h[R][NV][VEC], g[R][NV][VEC], rstd[R], sums[2 * R];
    rows.take();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = next_rstd[r];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const bool live = row0 + r < a.n && t + k * TPR < nvec;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          h[r][k][i] = live ? (to_float<T>(rows.raw[0][r][k].v[i]) - next_mean[r]) * rstd[r] : 0.0f;
          g[r][k][i] = live ? to_float<T>(rows.raw[1][r][k].v[i]) : 0.0f;
        }
      }
    }
    rows.next(row0);
    statistics(row0 + step);
#pragma unroll
    for (int r = 0; r < 2 * R; ++r) sums[r] = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = t + k * TPR;
      float wk[VEC];
      if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) wk[i] = w[k][i];
      } else if (c < nvec) {
        load_param<VEC>(a.weight, a.param_dtype, c * VEC, 1.0f, wk);
      }
      if (c < nvec) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            dw[k][i] += g[r][k][i] * h[r][k][i];
            db[k][i] += g[r][k][i];
            g[r][k][i] *= wk[i];
            sums[2 * r] += g[r][k][i];
            sums[2 * r + 1] += g[r][k][i] * h[r][k][i];
          }
        }
      }
    }
    if (a.dx != nullptr) {
      // two buffers in turn: a CTA-wide sum of the next row may begin while another thread still reads this one's
      row_sums<TPR>(sums, red[parity]);
      parity ^= 1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float sg = sums[2 * r] * inv_d, sgh = sums[2 * r + 1] * inv_d;
        if (row0 + r < a.n) {
          T* dx = static_cast<T*>(a.dx) + (row0 + r) * a.D;
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            const int c = t + k * TPR;
            if (c < nvec) {
#pragma unroll
              for (int i = 0; i < VEC; ++i) g[r][k][i] = rstd[r] * (g[r][k][i] - sg - h[r][k][i] * sgh);
              store_vec<T, VEC>(dx + c * VEC, g[r][k]);
            }
          }
        }
      }
    }
  }
  const bool together = a.dweight != nullptr;
  if (a.partial == nullptr && !together) return;
  if (together) {  // the ring becomes this CTA's column sums
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
  }
  float* out = together ? reinterpret_cast<float*>(ring) : a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.D;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = t + k * TPR;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float* mine = half == 0 ? dw[k] : db[k];
      if constexpr (GROUPS > 1) {  // the CTA's row groups, added in their order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) merge[threadIdx.x * VEC + i] = mine[i];
        __syncthreads();
        if (threadIdx.x < TPR) {
#pragma unroll
          for (int r = 1; r < GROUPS; ++r)
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
  if (together) {
    cluster_barrier();
    const uint32_t sums = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    for (int j = blockIdx.x * threads_of<TPR>() + threadIdx.x; j < 2 * a.D; j += a.ctas * threads_of<TPR>()) {
      float v = 0.0f;
      for (int c = 0; c < a.ctas; ++c) v += shared_of(sums + j * 4, c);
      if (j < a.D) store_from_float(a.dweight, a.param_dtype, j, v);
      else store_from_float(a.dbias, a.param_dtype, j - a.D, v);
    }
    cluster_barrier();  // nobody leaves while its sums are read
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

// Adds `count` partial rows [2][D]: a CTA takes 32 columns, each of its 32 warps every 32nd partial row, eight loads under
// way at a time (what there is to read is small; the launch is as long as its loads are late).
constexpr int LN_JOIN_THREADS = 1024;
__global__ void __launch_bounds__(LN_JOIN_THREADS) norm_join_kernel(const float* __restrict__ partial, int count, int D,
                                                                    void* dweight, void* dbias, int32_t dtype) {
  constexpr int NW = LN_JOIN_THREADS / 32;
  __shared__ float part[NW][33];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;  // of 2 D columns: the weight's, then the bias's
  float s[8] = {};
  if (j < 2 * D) {
    const float* p = partial + j;
    const int64_t step = 2 * static_cast<int64_t>(D);
    for (int r0 = warp; r0 < count; r0 += 8 * NW) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r0 + u * NW < count) s[u] += p[(r0 + u * NW) * step];
    }
  }
  part[warp][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (warp == 0 && j < 2 * D) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += part[w][lane];
    if (j < D) store_from_float(dweight, dtype, j, sum);
    else store_from_float(dbias, dtype, j - D, sum);
  }
}

// Threads per row and vectors per thread that hold `nvec` vectors; TPR == 0: none does.  Rows in vectors of 16 bytes: the
// fewest threads that hold the row with 16 values each, as a row then needs the fewest shuffles (430 000 rows of 100 floats,
// backward: 8 threads 80 us, 32 threads 91 us).  Element by element, 32 threads, whose loads lie side by side.
// Vectors that a thread of a CTA-wide row holds at most: what two stages of the ring, or the registers, have room for
template <int VEC, bool BACKWARD>
constexpr int most_vectors() {
  return VEC == 1 ? (BACKWARD ? 16 : 32) : BACKWARD ? 4 : 8;
}
struct Shape {
  int tpr, nv;
};
// (with_shape has a kernel for each shape that is returned here, and for no other)
inline Shape shape_for(int64_t nvec, int vec, int most_nv) {
  const int nv16 = 16 / vec;
  if (vec > 1) {
    for (int nv = 1; nv <= nv16; nv *= 2)
      if (nvec <= 4 * nv) return {4, nv};
    for (int tpr = 8; tpr <= 32; tpr *= 2)
      if (nvec <= tpr * nv16) return {tpr, nv16};
    if (nvec <= 32 * 2 * nv16) return {32, 2 * nv16};
  } else {
    for (int tpr = 4; tpr <= 32; tpr *= 2)
      if (nvec <= tpr) return {tpr, 1};
    for (int nv = 2; nv <= 32; nv *= 2)
      if (nvec <= 32 * nv) return {32, nv};
  }
  if (vec > 1) {
    for (int nv = vec == 8 ? 1 : 2; nv <= 2; nv *= 2)
      if (nvec <= 256 * nv) return {256, nv};
  }
  for (int nv = vec > 1 ? 2 : 4; nv <= most_nv; nv *= 2)
    if (nvec <= static_cast<int64_t>(512) * nv) return {512, nv};
  return {0, 0};
}

constexpr int LN_WIDE_SPLITS = 64;

template <typename T>
constexpr int full_vec() {
  return 16 / static_cast<int>(sizeof(T));
}

inline int64_t ctas_for(int64_t n, int rows, int per_sm) {
  const int64_t need = (n + rows - 1) / rows, most = static_cast<int64_t>(sm_count()) * per_sm;
  return need < most ? need : most;
}

constexpr int LN_CTAS_PER_SM = 4;  // backward, at most: each CTA writes a partial row of its own

// Backward, rows that a cluster of eight CTAs takes at once: one launch and no partial sums in memory, 11.4 -> 9.1 us a call and
// in a graph 4.7 -> 4.4 (64 rows of 256 floats), 7.2 -> 6.9 (64 of 1 024 bf16). Rows for four such rounds are slower there
// (473 rows of 236 bf16 6.1 -> 9.1 us, 512 of 256 floats 4.9 -> 6.3): they keep the grid and the second launch.
constexpr int LN_CLUSTER = 8;
constexpr int64_t LN_CLUSTER_COLUMNS = 4096;  // whose sums, 32 KB, need no leave beside the static arrays

// CTAs of a kernel that an SM holds at once, asked for once per kernel and device, and its leave to use `smem` bytes
constexpr int LN_MAX_DEVICES = 64;
template <typename K>
int resident(K kernel, int threads, size_t smem, std::atomic<int> (&known)[LN_MAX_DEVICES], int* held) {
  int dev = 0;
  DGS_CUDA_TRY(cudaGetDevice(&dev));
  DGS_REQUIRE(dev >= 0 && dev < LN_MAX_DEVICES, DGS_ERR_UNSUPPORTED, "layer_norm: device ordinal %d", dev);
  *held = known[dev].load(std::memory_order_acquire);
  if (*held == 0) {
    // (what every kernel may have holds for the rest, and for the column sums of a cluster)
    if (smem > LN_CLUSTER_COLUMNS * 2 * sizeof(float))
      DGS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    DGS_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(held, kernel, threads, smem));
    if (*held < 1) *held = 1;
    known[dev].store(*held, std::memory_order_release);
  }
  return DGS_OK;
}

// f.template run<VEC, TPR, NV>() for a shape, f.run_wide() where no variant holds the row
template <int VEC, typename F>
int with_shape(const Shape& s, const F& f) {
  constexpr int NV16 = 16 / VEC, MOST = most_vectors<VEC, F::kBackward>();
  switch (s.tpr) {
    case 4:
      if (s.nv == 1) return f.template run<VEC, 4, 1>();
      if constexpr (VEC > 1) {
        if (s.nv == 2) return f.template run<VEC, 4, 2>();
        if constexpr (NV16 >= 4)
          if (s.nv == 4) return f.template run<VEC, 4, 4>();
      }
      break;
    case 8: return f.template run<VEC, 8, VEC == 1 ? 1 : NV16>();
    case 16: return f.template run<VEC, 16, VEC == 1 ? 1 : NV16>();
    case 32:
      if constexpr (VEC > 1) {
        return s.nv == NV16 ? f.template run<VEC, 32, NV16>() : f.template run<VEC, 32, 2 * NV16>();
      } else {
        switch (s.nv) {
          case 1: return f.template run<1, 32, 1>();
          case 2: return f.template run<1, 32, 2>();
          case 4: return f.template run<1, 32, 4>();
          case 8: return f.template run<1, 32, 8>();
          case 16: return f.template run<1, 32, 16>();
          default: return f.template run<1, 32, 32>();
        }
      }
    case 256:
      if constexpr (VEC == 8)
        if (s.nv == 1) return f.template run<VEC, 256, 1>();
      if constexpr (VEC > 1)
        if (s.nv == 2) return f.template run<VEC, 256, 2>();
      break;
    case 512:
      if constexpr (VEC > 1)
        if (s.nv == 2) return f.template run<VEC, 512, 2>();
      if constexpr (MOST >= 4)
        if (s.nv == 4) return f.template run<VEC, 512, 4>();
      if constexpr (MOST >= 8)
        if (s.nv == 8) return f.template run<VEC, 512, 8>();
      if constexpr (MOST >= 16)
        if (s.nv == 16) return f.template run<VEC, 512, 16>();
      if constexpr (MOST >= 32)
        if (s.nv == 32) return f.template run<VEC, 512, 32>();
      break;
    default: break;
  }
  return f.run_wide();
}

template <typename T>
struct Forward {
  static constexpr bool kBackward = false;
  const NormArgs& a;
  cudaStream_t s;
  template <int VEC, int TPR, int NV>
  int run() const {
    static std::atomic<int> known[LN_MAX_DEVICES] = {};
    constexpr int R = rows_at_once<VEC, TPR, NV>();
    constexpr size_t smem = ring_bytes<T, VEC, TPR, NV, R, 1>();
    constexpr int threads = threads_of<TPR>();
    auto kernel = norm_forward_kernel<T, VEC, TPR, NV>;
    int held = 0;
    if (int rc = resident(kernel, threads, smem, known, &held)) return rc;
    DGS_CUDA_TRY(launch_training(kernel, dim3(static_cast<unsigned>(ctas_for(a.n, threads / TPR * R, held))), threads, smem, s, a));
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
  if (whole) return with_shape<VEC>(shape_for(a.D / VEC, VEC, most_vectors<VEC, false>()), f);
  return with_shape<1>(shape_for(a.D, 1, most_vectors<1, false>()), f);
}

template <typename T>
struct Backward {
  static constexpr bool kBackward = true;
  NormBackArgs a;
  cudaStream_t s;
  int64_t* partials;
  void *dweight, *dbias;
  template <int VEC, int TPR, int NV>
  int run() const {
    static std::atomic<int> known[LN_MAX_DEVICES] = {};
    constexpr int R = rows_at_once<VEC, TPR, NV>();
    constexpr size_t smem = ring_bytes<T, VEC, TPR, NV, R, 2>();
    constexpr int threads = threads_of<TPR>();
    auto kernel = norm_backward_kernel<T, VEC, TPR, NV>;
    constexpr int64_t rows = threads / TPR * R;
    if (dweight != nullptr && a.n <= rows * LN_CLUSTER && a.D <= LN_CLUSTER_COLUMNS) {
      NormBackArgs b = a;
      b.partial = nullptr;
      b.dweight = dweight;
      b.dbias = dbias;
      b.ctas = static_cast<int32_t>((a.n + rows - 1) / rows);
      const size_t sums = 2 * static_cast<size_t>(a.D) * sizeof(float), bytes = smem > sums ? smem : sums;
      int held = 0;
      if (int rc = resident(kernel, threads, smem, known, &held)) return rc;
      *partials = 0;
      DGS_CUDA_TRY(launch_clusters(kernel, dim3(static_cast<unsigned>(b.ctas)), threads, bytes, s, static_cast<unsigned>(b.ctas), b));
      return DGS_OK;
    }
    int held = 0;
    if (int rc = resident(kernel, threads, smem, known, &held)) return rc;
    *partials = ctas_for(a.n, threads / TPR * R, held < LN_CTAS_PER_SM ? held : LN_CTAS_PER_SM);
    DGS_CUDA_TRY(launch_training(kernel, dim3(static_cast<unsigned>(*partials)), threads, smem, s, a));
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
int backward(const NormBackArgs& a, int64_t* partials, void* dweight, void* dbias, cudaStream_t s) {
  constexpr int VEC = full_vec<T>();
  const bool whole = a.D % VEC == 0 && a.x_stride % VEC == 0 && a.dy_stride % VEC == 0 && aligned_to(a.x, 16) &&
                     aligned_to(a.dy, 16) && aligned_to(a.dx, 16) && aligned_to(a.weight, 16);
  const Backward<T> f{a, s, partials, dweight, dbias};
  if (whole) return with_shape<VEC>(shape_for(a.D / VEC, VEC, most_vectors<VEC, true>()), f);
  return with_shape<1>(shape_for(a.D, 1, most_vectors<1, true>()), f);
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
  const int64_t most = static_cast<int64_t>(sm_count()) * LN_CTAS_PER_SM;
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
  NormBackArgs a{};
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.param_dtype = param_dtype;
  a.mean = mean;
  a.rstd = rstd;
  a.n = n;
  a.D = static_cast<int>(D);
  a.dx = dx;
  a.partial = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  int64_t partials = 0;
  const int rc = dtype == DGS_F32    ? backward<float>(a, &partials, dweight, dbias, s)
                 : dtype == DGS_BF16 ? backward<__nv_bfloat16>(a, &partials, dweight, dbias, s)
                                     : backward<__half>(a, &partials, dweight, dbias, s);
  if (rc != DGS_OK || dweight == nullptr || partials == 0) return rc;  // (no partial sums: the gradients are there)
  DGS_CUDA_TRY(launch_training(norm_join_kernel, dim3(static_cast<unsigned>((2 * D + 31) / 32)), LN_JOIN_THREADS, 0, s, a.partial,
                               static_cast<int>(partials), a.D, dweight, dbias, param_dtype));
  return DGS_OK;
}
