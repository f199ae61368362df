// The end of a block and the norm in front of the next one, forward and backward:
//
//   z = post(y),  s = xs x + ys gate z  (stored in x's type),  out = pre(s)
//   norm(v) = (v - mean) rstd w + b with mean = 0 for the root-mean-square form; either norm, the gate, biases may be absent
//
//   g = ds + pre'(dout),  dx = xs g,  dgate = ys g z,  dz = ys g gate,  dy = post'(dz)
//   norm'(d) = rstd (d w - avg(d w) - h avg(d w h)), h the normed values (the plain average is left out in the root-mean-square form)
//   dw = sum over rows of d h, db = sum of d, the gate's gradient summed over what it was spread over
//
// Bound by HBM: every row is read and written once in each direction.  TPR threads share a row, E elements each, which stay in
// registers from the first sum to the result; sums are in 32 bits and of centred values.  A thread keeps its columns for all rows of
// its CTA, so column sums grow in registers; each CTA leaves one partial row and a second launch adds the partial rows in their
// order (no atomics: the same inputs give the same bits).  A gate of the columns is the same factor in every row, so its gradient and
// those of the post norm's parameters come out of two sums: with S2 = sum g ys y^, S3 = sum g ys
//   dpost_weight = gate S2,  dpost_bias = gate S3,  dgate = post_weight S2 + post_bias S3
// At 12 bytes an element the issue slots allow some 60 instructions: weights lie in shared memory in 32 bits (a quarter of a load each, no
// conversion), arithmetic is two elements an instruction, and with 16 elements a thread a row's sums over the CTA cost a twentieth.
// Measured, 16 384 x 4 096 bfloat16, both norms and a gate of the columns: forward 131 us (3.5 TB/s of DRAM, 62 % of the issue slots), backward
// 244 us (3.2 TB/s).
#include <initializer_list>

#include "train_common.cuh"

namespace dgs {
namespace {

constexpr int RN_MAX_D = 8192;
constexpr int RN_SUMS = 4;     // column sums: dout h, dout, S2, S3
constexpr int RN_GRADS = 5;    // dweight, dbias, dpost_weight, dpost_bias, dgate
constexpr int RN_PARAMS = 5;   // post_weight, post_bias, the columns' gate, weight, bias
constexpr int RN_MAX_CTAS_PER_SM = 4;
constexpr int RN_MAX_STAGES = 4;
constexpr int RN_JOIN_THREADS = 1024;
constexpr int RN_MAX_SMEM = 220 * 1024;
constexpr int RN_MAX_DEVICES = 64;

struct Source {
  const void* p;  // nullptr: absent
  int64_t stride;
};

struct NormArgs {
  Source in[5];  // forward: x, y, gate of each element; backward: s, y, dout, ds, gate of each element
  const void* param[RN_PARAMS];
  const void* row_gate;
  int64_t n;
  int32_t D, param_dtype, post, pre;  // DGS_NORM_*
  float xs, ys, eps;
  // forward
  void *sum, *out;
  float *post_mean, *post_rstd, *mean, *rstd;
  // backward
  void *dx, *dy, *dgate;  // dgate: of each element, or of each row
  float* partial;         // [CTAs][RN_SUMS][D]
  int32_t stages, stage_bytes, ring_at, param_at[RN_PARAMS];  // shared memory: the weights that are there, in 32 bits, then the ring
};
enum { POST_WEIGHT, POST_BIAS, GATE, WEIGHT, BIAS };

// Threads of a CTA: as many as registers allow (64 a thread forward, 128 backward), so that several rows are under way beside one another
// over one copy of the weights; rows narrower than a warp need few of them and take smaller CTAs.
template <int TPR, bool BACK>
constexpr int threads_of() {
  return BACK ? 512 : TPR > 32 ? 1024 : 256;
}

// all threads of a row that several warps share
template <int TPR>
__device__ __forceinline__ void row_barrier() {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / TPR), "n"(TPR) : "memory");
}

// COUNT (up to 3) sums over the threads of a row, returned to all of them, who all call it; `red` is not written again before every one of
// them has passed another such sum, or a barrier.
template <int TPR, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], float4* red) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int q = 0; q < COUNT; ++q) v[q] += __shfl_xor_sync(FULL_MASK, v[q], o);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    float* mine = reinterpret_cast<float*>(red + (threadIdx.x >> 5));
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int q = 0; q < COUNT; ++q) mine[q] = v[q];
    }
    row_barrier<TPR>();
    const float* other = reinterpret_cast<const float*>(red + (threadIdx.x >> 5 & ~(WARPS - 1)) + (threadIdx.x & (WARPS - 1)));
#pragma unroll
    for (int q = 0; q < COUNT; ++q) v[q] = other[q];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1)
#pragma unroll
      for (int q = 0; q < COUNT; ++q) v[q] += __shfl_xor_sync(FULL_MASK, v[q], o);
  }
}

// two elements an instruction
__device__ __forceinline__ void add_to(float* v, float lo, float hi) {
  split2(add2(two(v[0], v[1]), two(lo, hi)), &v[0], &v[1]);
}
__device__ __forceinline__ void mul_to(float* v, float lo, float hi) {
  split2(mul2(two(v[0], v[1]), two(lo, hi)), &v[0], &v[1]);
}
// v += a b
__device__ __forceinline__ void fma_to(float* v, const float* a, const float* b) {
  split2(fma2(two(a[0], a[1]), two(b[0], b[1]), two(v[0], v[1])), &v[0], &v[1]);
}

// Rows of up to COUNT arrays.  Vectors of 4, 8 or 16 bytes travel by cp.async through a ring in shared memory, so the next rows are on
// their way while one is summed; a thread fetches what it will read itself, so its own wait is all the synchronisation.  Single
// elements of two bytes are loaded where they are used.
template <typename T, int VEC, int TPR, int E, int COUNT, bool BACK>
struct Feed {
  static constexpr int NV = E / VEC, THREADS = threads_of<TPR, BACK>(), BYTES = VEC * static_cast<int>(sizeof(T));
  static constexpr bool kRing = BYTES >= 4;
  const NormArgs& a;
  const unsigned char* ring;
  int t, stage;
  int64_t step, ahead;

  __device__ __forceinline__ bool in(int k) const { return (k * TPR + t) * VEC < a.D; }
  __device__ __forceinline__ int column(int k) const { return (k * TPR + t) * VEC; }
  __device__ __forceinline__ void issue(int64_t row, int st) {
    if constexpr (kRing) {
      if (row < a.n) {
        uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + st * a.stage_bytes + threadIdx.x * BYTES;
#pragma unroll
        for (int q = 0; q < COUNT; ++q) {
          if (a.in[q].p == nullptr) continue;
          const T* p = static_cast<const T*>(a.in[q].p) + row * a.in[q].stride;
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            if (in(k)) {
              if constexpr (BYTES == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(p + column(k)) : "memory");
              else
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(p + column(k)), "n"(BYTES) : "memory");
            }
            at += THREADS * BYTES;
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
    ring = smem;
    if constexpr (kRing) {
      // what lies behind a row's end is never fetched: zeros, once
      if (TPR * E != a.D)
        for (int at = threadIdx.x * 4; at < a.stages * a.stage_bytes; at += THREADS * 4) *reinterpret_cast<uint32_t*>(smem + at) = 0;
      __syncthreads();
      for (int s = 0; s < a.stages - 1; ++s) issue(row + s * step, s);
    }
    ahead = (a.stages - 1) * step;
  }
  // the rows `row` of this stage: asks for those `stages - 1` steps on, waits for these
  __device__ __forceinline__ void next(int64_t row) {
    if constexpr (kRing) {
      issue(row + ahead, stage == 0 ? a.stages - 1 : stage - 1);
      if (a.stages == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else if (a.stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else if (a.stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else asm volatile("cp.async.wait_group 3;" ::: "memory");
    }
  }
  __device__ __forceinline__ void done() {
    if constexpr (kRing) stage = stage + 1 == a.stages ? 0 : stage + 1;
  }
  // Array q's elements of the row, zeros behind its end; `slot`: how many arrays are there before it.  (A row that is not there: anything.)
  __device__ __forceinline__ void get(int q, int slot, int64_t row, bool there, float (&v)[E]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[VEC];
      if constexpr (kRing) {
        load_vec<T, VEC>(reinterpret_cast<const T*>(ring + stage * a.stage_bytes + ((slot * NV + k) * THREADS + threadIdx.x) * BYTES), x);
      } else {
        x[0] = there && in(k) ? to_float<T>((static_cast<const T*>(a.in[q].p) + row * a.in[q].stride)[column(k)]) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k * VEC + e] = x[e];
    }
  }
  __device__ __forceinline__ void put(void* base, int64_t row, bool there, const float (&v)[E]) const {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!(there && in(k))) continue;
      float x[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = v[k * VEC + e];
      store_vec<T, VEC>(static_cast<T*>(base) + row * a.D + column(k), x);
    }
  }
  __device__ __forceinline__ void zero_outside(float (&v)[E]) const {
    if (TPR * E == a.D) return;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (!in(k)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k * VEC + e] = 0.0f;
      }
  }
  // Weights: all TPR * E columns (beyond D: zeros), the fours of a vector of eight apart, so that neighbouring threads' 16 bytes lie
  // side by side.
  static __device__ __forceinline__ int place(int c) {
    if constexpr (VEC == 8) return (c % 8 / 4) * (TPR * E / 2) + c / 8 * 4 + c % 4;
    return c;
  }
  __device__ __forceinline__ void lay_out(unsigned char* smem) const {
#pragma unroll 1
    for (int q = 0; q < RN_PARAMS; ++q) {
      if (a.param[q] == nullptr || a.param_at[q] < 0) continue;
      float* to = reinterpret_cast<float*>(smem + a.param_at[q]);
      for (int c = threadIdx.x; c < TPR * E; c += THREADS) to[place(c)] = c < a.D ? load_as_float(a.param[q], a.param_dtype, c) : 0.0f;
    }
    __syncthreads();
  }
  __device__ __forceinline__ void param(int q, const unsigned char* smem, float (&v)[E]) const {
    if (a.param_at[q] < 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = in(i / VEC) ? load_as_float(a.param[q], a.param_dtype, column(i / VEC) + i % VEC) : 0.0f;
      return;
    }
    const float* p = reinterpret_cast<const float*>(smem + a.param_at[q]);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = column(k);
      if constexpr (VEC >= 4) {
#pragma unroll
        for (int f = 0; f < VEC / 4; ++f) {
          const float4 x = *reinterpret_cast<const float4*>(p + place(c + f * 4));
          v[k * VEC + f * 4] = x.x, v[k * VEC + f * 4 + 1] = x.y, v[k * VEC + f * 4 + 2] = x.z, v[k * VEC + f * 4 + 3] = x.w;
        }
      } else {
        v[k] = p[c];
      }
    }
  }
};

// 1 / sqrt(v): the approximation and one step of Newton's method, r + r (1 - v r r) / 2, within two units in the last place
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v), e = fmaf(-v * r, r, 1.0f);
  return v > 0.0f && v < INFINITY ? fmaf(0.5f * r, e, r) : r;
}

// normed values of v in place (zeros outside of the row); every thread of the CTA calls it
template <int TPR, int E, typename FeedT>
__device__ __forceinline__ void normalise(const FeedT& f, bool layer, int D, float eps, float (&v)[E], float* mean, float* rstd, float4 (*red)[32]) {
  const float inv = 1.0f / static_cast<float>(D);
  *mean = 0.0f;
  if (layer) {
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < E; i += 2) add_to(s, v[i], v[i + 1]);
    float t[1] = {s[0] + s[1]};
    row_sums<TPR, 1>(t, red[0]);
    *mean = t[0] * inv;
#pragma unroll
    for (int i = 0; i < E; i += 2) add_to(v + i, -*mean, -*mean);
    f.zero_outside(v);
  }
  float s[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < E; i += 2) fma_to(s, v + i, v + i);
  float t[1] = {s[0] + s[1]};
  row_sums<TPR, 1>(t, red[1]);
  *rstd = inverse_root(fmaf(t[0], inv, eps));
#pragma unroll
  for (int i = 0; i < E; i += 2) mul_to(v + i, *rstd, *rstd);
}

// v = v weight + bias, each where it is there
template <int E, typename FeedT>
__device__ __forceinline__ void weigh(const FeedT& f, int weight, int bias, const unsigned char* smem, float (&v)[E]) {
  float p[E];
  if (f.a.param[weight] != nullptr) {
    f.param(weight, smem, p);
#pragma unroll
    for (int i = 0; i < E; i += 2) mul_to(v + i, p[i], p[i + 1]);
  }
  if (f.a.param[bias] != nullptr) {
    f.param(bias, smem, p);
#pragma unroll
    for (int i = 0; i < E; i += 2) add_to(v + i, p[i], p[i + 1]);
  }
}

template <typename T, int VEC, int TPR, int E>
__global__ __launch_bounds__(threads_of<TPR, false>()) void residual_norm_kernel(const __grid_constant__ NormArgs a) {
  constexpr int ROWS = threads_of<TPR, false>() / TPR;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float4 red[4][32];
  pdl_enter();
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  Feed<T, VEC, TPR, E, 3, false> f{a};
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR;
  f.begin(mine, step, smem + a.ring_at);
  f.lay_out(smem);
  for (int64_t row = mine; row - threadIdx.x / TPR < a.n; row += step) {
    f.next(row);
    const bool there = row < a.n;
    float y[E], p[E], m, r;
    f.get(1, 1, row, there, y);
    if (a.post != DGS_NORM_NONE) {
      normalise<TPR, E>(f, a.post == DGS_NORM_LAYER, a.D, a.eps, y, &m, &r, red);
      if (there && f.t == 0) {
        if (a.post == DGS_NORM_LAYER) a.post_mean[row] = m;
        a.post_rstd[row] = r;
      }
      weigh(f, POST_WEIGHT, POST_BIAS, smem, y);
    }
    if (a.in[2].p != nullptr) {
      f.get(2, 2, row, there, p);
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(y + i, p[i], p[i + 1]);
    } else if (a.param[GATE] != nullptr) {
      f.param(GATE, smem, p);
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(y + i, p[i], p[i + 1]);
    } else if (a.row_gate != nullptr) {
      const float by = there ? to_float<T>(static_cast<const T*>(a.row_gate)[row]) : 0.0f;
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(y + i, by, by);
    }
    f.get(0, 0, row, there, p);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      mul_to(p + i, a.xs, a.xs);
      const float ys[2] = {a.ys, a.ys};
      fma_to(p + i, ys, y + i);
      // (the next norm is of the row as it is stored, so that the backward pass finds the same)
      y[i] = to_float<T>(from_float<T>(p[i]));
      y[i + 1] = to_float<T>(from_float<T>(p[i + 1]));
    }
    f.done();
    f.put(a.sum, row, there, y);
    if (a.pre != DGS_NORM_NONE) {
      f.zero_outside(y);
      normalise<TPR, E>(f, a.pre == DGS_NORM_LAYER, a.D, a.eps, y, &m, &r, red + 2);
      if (there && f.t == 0) {
        if (a.pre == DGS_NORM_LAYER) a.mean[row] = m;
        a.rstd[row] = r;
      }
      weigh(f, WEIGHT, BIAS, smem, y);
      f.put(a.out, row, there, y);
    }
    if constexpr (TPR > 32) {
      // (a row with one sum alone: `red` must not be written before all have read it)
      if ((a.post != DGS_NORM_NONE) + (a.post == DGS_NORM_LAYER) + (a.pre != DGS_NORM_NONE) + (a.pre == DGS_NORM_LAYER) == 1) row_barrier<TPR>();
    }
  }
}

// norm' of d (the gradient of the normed values) in place, zeros outside of the row; h the normed values; `also` is summed over the row too
template <int TPR, int E, typename FeedT>
__device__ __forceinline__ void norm_back(const FeedT& f, bool layer, int D, float rstd, const float (&h)[E], float (&d)[E], float* also,
                                          float4* red) {
  float p[2] = {0.0f, 0.0f}, q[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    add_to(p, d[i], d[i + 1]);
    fma_to(q, d + i, h + i);
  }
  float s[3] = {p[0] + p[1], q[0] + q[1], *also};
  row_sums<TPR, 3>(s, red);
  const float inv = 1.0f / static_cast<float>(D), avg = layer ? s[0] * inv * rstd : 0.0f, dot = s[1] * inv * rstd;
  *also = s[2];
  const float minus[2] = {-dot, -dot}, by[2] = {rstd, rstd};
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    // d rstd - avg - h dot
    float x[2] = {-avg, -avg};
    fma_to(x, h + i, minus);
    fma_to(x, d + i, by);
    d[i] = x[0];
    d[i + 1] = x[1];
  }
  f.zero_outside(d);
}

template <typename T, int VEC, int TPR, int E>
__global__ __launch_bounds__(threads_of<TPR, true>()) void residual_norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int THREADS = threads_of<TPR, true>(), ROWS = THREADS / TPR;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float4 red[2][32];
  pdl_enter();
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  Feed<T, VEC, TPR, E, 5, true> f{a};
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR;
  f.begin(mine, step, smem + a.ring_at);
  f.lay_out(smem);
  int slot[5], slots = 0;
#pragma unroll
  for (int q = 0; q < 5; ++q) {
    slot[q] = slots;
    slots += a.in[q].p != nullptr;
  }
  float sums[RN_SUMS][E];
#pragma unroll
  for (int q = 0; q < RN_SUMS; ++q)
#pragma unroll
    for (int i = 0; i < E; ++i) sums[q][i] = 0.0f;
  const bool pre = a.pre != DGS_NORM_NONE && a.in[2].p != nullptr, post = a.post != DGS_NORM_NONE, layer = a.pre == DGS_NORM_LAYER;
  const bool columns = a.param[GATE] != nullptr, post_layer = a.post == DGS_NORM_LAYER;
  // a row's statistics, asked for a row ahead
  float next[4] = {};
  const auto ask = [&](int64_t row) {
    if (row >= a.n) return;
    if (pre) next[1] = a.rstd[row];
    if (pre && layer) next[0] = a.mean[row];
    if (post) next[3] = a.post_rstd[row];
    if (post_layer) next[2] = a.post_mean[row];
  };
  ask(mine);
  for (int64_t row = mine; row - threadIdx.x / TPR < a.n; row += step) {
    f.next(row);
    const bool there = row < a.n;
    float g[E], h[E], w[E], none = 0.0f;
    const float m = next[0], r = next[1], post_m = next[2], post_r = next[3];
    ask(row + step);
    if (pre) {
      f.get(0, slot[0], row, there, h);
      f.get(2, slot[2], row, there, g);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        if (layer) add_to(h + i, -m, -m);
        mul_to(h + i, r, r);
      }
      f.zero_outside(h);
      if (there) {
#pragma unroll
        for (int i = 0; i < E; i += 2) {
          fma_to(sums[0] + i, g + i, h + i);
          add_to(sums[1] + i, g[i], g[i + 1]);
        }
      }
      if (a.param[WEIGHT] != nullptr) {
        f.param(WEIGHT, smem, w);
#pragma unroll
        for (int i = 0; i < E; i += 2) mul_to(g + i, w[i], w[i + 1]);
      }
      norm_back<TPR, E>(f, layer, a.D, r, h, g, &none, red[0]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) g[i] = 0.0f;
    }
    if (a.in[3].p != nullptr) {
      f.get(3, slot[3], row, there, w);
#pragma unroll
      for (int i = 0; i < E; i += 2) add_to(g + i, w[i], w[i + 1]);
    }
    if (a.dx != nullptr) {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        w[i] = g[i], w[i + 1] = g[i + 1];
        mul_to(w + i, a.xs, a.xs);
      }
      f.put(a.dx, row, there, w);
    }
    f.get(1, slot[1], row, there, h);
    if (post) {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        if (post_layer) add_to(h + i, -post_m, -post_m);
        mul_to(h + i, post_r, post_r);
      }
      f.zero_outside(h);
    }
#pragma unroll
    for (int i = 0; i < E; i += 2) mul_to(g + i, a.ys, a.ys);
    float of_row = 0.0f;
    if (a.dgate != nullptr) {  // of each row or element: g times post(y)
      float z[E];
#pragma unroll
      for (int i = 0; i < E; ++i) z[i] = h[i];
      if (post) weigh(f, POST_WEIGHT, POST_BIAS, smem, z);
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(z + i, g[i], g[i + 1]);
      if (a.row_gate != nullptr) {
        f.zero_outside(z);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < E; i += 2) add_to(s, z[i], z[i + 1]);
        of_row = s[0] + s[1];
      } else {
        f.put(a.dgate, row, there, z);
      }
    }
    if (a.in[4].p != nullptr) {
      f.get(4, slot[4], row, there, w);
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(g + i, w[i], w[i + 1]);
    } else if (a.row_gate != nullptr) {
      const float by = there ? to_float<T>(static_cast<const T*>(a.row_gate)[row]) : 0.0f;
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(g + i, by, by);
    }
    f.done();
    if (there && (post || columns)) {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        fma_to(sums[2] + i, g + i, h + i);
        add_to(sums[3] + i, g[i], g[i + 1]);
      }
    }
    if (columns) {
      f.param(GATE, smem, w);
#pragma unroll
      for (int i = 0; i < E; i += 2) mul_to(g + i, w[i], w[i + 1]);
    }
    if (post) {
      if (a.param[POST_WEIGHT] != nullptr) {
        f.param(POST_WEIGHT, smem, w);
#pragma unroll
        for (int i = 0; i < E; i += 2) mul_to(g + i, w[i], w[i + 1]);
      }
      norm_back<TPR, E>(f, post_layer, a.D, post_r, h, g, &of_row, red[1]);
    } else if (a.row_gate != nullptr) {
      float s[1] = {of_row};
      row_sums<TPR, 1>(s, red[1]);
      of_row = s[0];
    }
    if (a.dy != nullptr) f.put(a.dy, row, there, g);
    if (a.row_gate != nullptr && a.dgate != nullptr && there && f.t == 0) static_cast<T*>(a.dgate)[row] = from_float<T>(of_row);
    if constexpr (TPR > 32) {
      // (a row with one sum alone: `red` must not be written before all have read it)
      if (!pre || (!post && a.row_gate == nullptr)) row_barrier<TPR>();
    }
  }
  if (a.partial == nullptr) return;
  float* to = a.partial + static_cast<int64_t>(blockIdx.x) * RN_SUMS * a.D;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int q = 0; q < RN_SUMS; ++q)
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (f.in(i / VEC)) to[q * a.D + f.column(i / VEC) + i % VEC] = sums[q][i];
  } else {
    // the CTA's groups, in their order
    constexpr int WIDTH = TPR * E;
    float* all = reinterpret_cast<float*>(smem);  // [ROWS][WIDTH]
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int q = 0; q < RN_SUMS; ++q) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i) all[(threadIdx.x / TPR) * WIDTH + f.column(i / VEC) + i % VEC] = sums[q][i];
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
  const void *post_weight, *post_bias, *gate;
  void* to[RN_GRADS];
};
// partial rows added in their order: 32 columns a CTA, a warp for every 32nd row
__global__ __launch_bounds__(RN_JOIN_THREADS) void residual_norm_join_kernel(const __grid_constant__ JoinArgs a) {
  __shared__ float part[RN_SUMS][32][33];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s[RN_SUMS] = {};
  if (c < a.D) {
#pragma unroll 4
    for (int r = warp; r < a.partials; r += 32)
#pragma unroll
      for (int q = 0; q < RN_SUMS; ++q) s[q] += a.partial[(static_cast<int64_t>(r) * RN_SUMS + q) * a.D + c];
  }
#pragma unroll
  for (int q = 0; q < RN_SUMS; ++q) part[q][warp][lane] = s[q];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < RN_SUMS; ++q) {
    s[q] = part[q][lane][warp];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[q] += __shfl_xor_sync(FULL_MASK, s[q], o);
  }
  const int column = blockIdx.x * 32 + warp;
  if (lane != 0 || column >= a.D) return;
  const float gate = a.gate != nullptr ? load_as_float(a.gate, a.param_dtype, column) : 1.0f;
  const float w = a.post_weight != nullptr ? load_as_float(a.post_weight, a.param_dtype, column) : 1.0f;
  const float b = a.post_bias != nullptr ? load_as_float(a.post_bias, a.param_dtype, column) : 0.0f;
  const float grads[RN_GRADS] = {s[0], s[1], gate * s[2], gate * s[3], fmaf(w, s[2], b * s[3])};
#pragma unroll
  for (int q = 0; q < RN_GRADS; ++q)
    if (a.to[q] != nullptr) store_from_float(a.to[q], a.param_dtype, column, grads[q]);
}

// ---- host ------------------------------------------------------------------------------------------------------------
int64_t partial_rows(int64_t n) {
  const int64_t most = static_cast<int64_t>(sm_count()) * RN_MAX_CTAS_PER_SM;
  return n < most ? n : most;
}

template <typename T, int VEC, int TPR, int E, bool BACK>
int launch_rows(NormArgs a, int arrays, int* ctas, cudaStream_t s) {
  constexpr int THREADS = threads_of<TPR, BACK>(), ROWS = THREADS / TPR, NV = E / VEC, BYTES = VEC * static_cast<int>(sizeof(T));
  void (*kernel)(NormArgs);
  if constexpr (BACK) kernel = residual_norm_backward_kernel<T, VEC, TPR, E>;
  else kernel = residual_norm_kernel<T, VEC, TPR, E>;
  a.ring_at = 0;
  for (int q = 0; q < RN_PARAMS; ++q) {
    a.param_at[q] = a.ring_at;
    if (a.param[q] != nullptr) a.ring_at += TPR * E * static_cast<int>(sizeof(float));
  }
  a.stage_bytes = BYTES >= 4 ? arrays * NV * THREADS * BYTES : 0;
  if (a.ring_at + a.stage_bytes > RN_MAX_SMEM) {  // (the widest rows of 32 bits: weights out of global memory)
    a.ring_at = 0;
    for (int& at : a.param_at) at = -1;
  }
  // what a CTA has under way: a quarter of an SM's shared memory where an SM holds four, else all
  const int room = (THREADS <= 256 ? RN_MAX_SMEM / 4 : RN_MAX_SMEM) - a.ring_at;
  a.stages = a.stage_bytes == 0 ? 1 : a.stage_bytes * RN_MAX_STAGES <= room ? RN_MAX_STAGES : room / a.stage_bytes;
  if (a.stages < 2 && a.stage_bytes > 0) a.stages = (RN_MAX_SMEM - a.ring_at) / a.stage_bytes;  // (one CTA an SM, then)
  if (a.stages > RN_MAX_STAGES) a.stages = RN_MAX_STAGES;
  DGS_REQUIRE(a.stages >= 1, DGS_ERR_UNSUPPORTED, "residual_norm: rows of %d elements", a.D);
  size_t smem = static_cast<size_t>(a.ring_at) + static_cast<size_t>(a.stages) * a.stage_bytes;
  const size_t joined = BACK && ROWS > 1 ? static_cast<size_t>(THREADS) * E * sizeof(float) : 0;
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
  if constexpr (VEC == 1) {  // single elements: a warp a row as soon as it can, so that a load takes them side by side
    if (a.D <= 32) return launch_rows<T, 1, 8, 4, BACK>(a, arrays, ctas, s);
    if (a.D <= 128) return launch_rows<T, 1, 32, 4, BACK>(a, arrays, ctas, s);
  } else {
    if (a.D <= 64) return launch_rows<T, VEC, 4, 16, BACK>(a, arrays, ctas, s);
    if (a.D <= 128) return launch_rows<T, VEC, 8, 16, BACK>(a, arrays, ctas, s);
    if (a.D <= 256) return launch_rows<T, VEC, 16, 16, BACK>(a, arrays, ctas, s);
  }
  if (a.D <= 512) return launch_rows<T, VEC, 32, 16, BACK>(a, arrays, ctas, s);
  if (a.D <= 2048) return launch_rows<T, VEC, 128, 16, BACK>(a, arrays, ctas, s);
  if (a.D <= 4096) return launch_rows<T, VEC, 256, 16, BACK>(a, arrays, ctas, s);
  return launch_rows<T, VEC, 512, 16, BACK>(a, arrays, ctas, s);
}

template <typename T, bool BACK>
int with_type(const NormArgs& a, int vec, int arrays, int* ctas, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return with_row<T, 8, BACK>(a, arrays, ctas, s);
  return vec >= 4 ? with_row<T, 4, BACK>(a, arrays, ctas, s) : with_row<T, 1, BACK>(a, arrays, ctas, s);
}
template <bool BACK>
int run_rows(const NormArgs& a, int32_t dtype, int vec, int arrays, int* ctas, cudaStream_t s) {
  if (dtype == DGS_F32) return with_type<float, BACK>(a, vec, arrays, ctas, s);
  return dtype == DGS_BF16 ? with_type<__nv_bfloat16, BACK>(a, vec, arrays, ctas, s) : with_type<__half, BACK>(a, vec, arrays, ctas, s);
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
  a.param[POST_WEIGHT] = p.post_weight;
  a.param[POST_BIAS] = p.post_bias;
  a.param[GATE] = p.gate_kind == DGS_GATE_COLUMN ? p.gate : nullptr;
  a.param[WEIGHT] = p.weight;
  a.param[BIAS] = p.bias;
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

// the widest vectors in which every row of every array can be moved: 16 bytes, four elements, or one element
int vectors(const dgs_residual_norm& p, const NormArgs& a, int count, std::initializer_list<const void*> results) {
  const int esz = dtype_bytes(p.dtype);
  for (int vec = 16 / esz; vec >= 4; vec /= 2) {
    const size_t bytes = static_cast<size_t>(vec) * esz;
    bool fits = p.D % vec == 0;
    for (int q = 0; q < count; ++q)
      fits &= a.in[q].p == nullptr || (aligned_to(a.in[q].p, bytes) && (a.in[q].stride % vec == 0 || p.n <= 1));
    for (const void* r : results) fits &= aligned_to(r, bytes);
    if (fits) return vec;
  }
  return 1;
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
  return run_rows<false>(a, p->dtype, vectors(*p, a, 3, {sum, out}), a.in[2].p != nullptr ? 3 : 2, &ctas, static_cast<cudaStream_t>(stream));
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
  void* to[RN_GRADS] = {dweight, dbias, dpost_weight, dpost_bias, column ? dgate : nullptr};
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
  if (a.dgate == nullptr) a.param[POST_BIAS] = nullptr;  // (rows need it for their gate's gradient alone)
  a.param[BIAS] = nullptr;
  a.partial = any ? static_cast<float*>(workspace) : nullptr;
  int arrays = 0, ctas = 0;
  for (const Source& in : a.in) arrays += in.p != nullptr;
  if (int rc = run_rows<true>(a, p->dtype, vectors(*p, a, 5, {dx, dy, a.dgate}), arrays, &ctas, s)) return rc;
  if (!any) return DGS_OK;
  JoinArgs j{a.partial, ctas, a.D, p->param_dtype, p->post_weight, p->post_bias, a.param[GATE], {}};
  for (int q = 0; q < RN_GRADS; ++q) j.to[q] = to[q];
  DGS_CUDA_TRY(launch_training(residual_norm_join_kernel, dim3(static_cast<unsigned>((p->D + 31) / 32)), RN_JOIN_THREADS, 0, s, j));
  return DGS_OK;
}
