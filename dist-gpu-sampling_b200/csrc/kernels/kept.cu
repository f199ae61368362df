// Rows kept for the backward pass in 8 bits, and the gradient of a linear layer's weight from them.
//
//   a = max |x| over 128 columns of a row,  c = rint(x (127 / a)),  x ~ c (a / 127)
//   dW[o, d] = sum_n g[n, o] v[n, d],  db[o] = sum_n g[n, o]
//
// Codes: one byte is written for every element read; bound by the issue slots.  Measured, 430 000 x 100 bfloat16: codes 70 us (1.8 TB/s), values
// 40 us (3.2 TB/s).
#include "kept.h"

namespace dgs {
namespace {

constexpr int KEEP_THREADS = 256;
constexpr int KEEP_UNROLL = 4;

// ---- codes and values -------------------------------------------------------------------------------------------------
struct KeepArgs {
  const void* x;
  int64_t x_stride;
  int8_t* codes;
  const int8_t* codes_in;
  int64_t codes_stride;
  float* scales;
  const float* scales_in;
  void* out;
  int64_t n, tasks;  // tasks: groups of all rows
  int32_t D, groups;
};

__device__ __forceinline__ void row_and_group(const KeepArgs& a, int64_t task, int64_t* row, int* group) {
  if (a.groups == 1) {
    *row = task;
    *group = 0;
  } else if (a.tasks <= 0xffffffffll) {
    *row = static_cast<uint32_t>(task) / static_cast<uint32_t>(a.groups);
    *group = static_cast<int>(static_cast<uint32_t>(task) - static_cast<uint32_t>(*row) * a.groups);
  } else {
    *row = task / a.groups;
    *group = static_cast<int>(task - *row * a.groups);
  }
}

// Magnitudes are compared as words, where nan is above infinity: a value that is not finite makes the scale one that is not.
template <typename T>
__device__ __forceinline__ uint32_t largest_word(uint32_t top, uint32_t w);  // w: one value of 32 bits or two of 16
template <>
__device__ __forceinline__ uint32_t largest_word<float>(uint32_t top, uint32_t w) {
  return max(top, w & 0x7fffffffu);
}
template <>
__device__ __forceinline__ uint32_t largest_word<__nv_bfloat16>(uint32_t top, uint32_t w) {
  return __vmaxu2(top, w & 0x7fff7fffu);
}
template <>
__device__ __forceinline__ uint32_t largest_word<__half>(uint32_t top, uint32_t w) {
  return __vmaxu2(top, w & 0x7fff7fffu);
}
template <typename T>
__device__ __forceinline__ float largest_value(uint32_t top) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(top);
  const uint16_t one = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
  return to_float<T>(*reinterpret_cast<const T*>(&one));
}

constexpr float ROUND = 12582912.0f;  // 1.5 * 2^23: a number of up to 2^22 added to it is rounded to a whole one, in the last bits of the sum
// the code of x: the product rounded to 32 bits, then to the nearest whole number (ties to the even one)
__device__ __forceinline__ uint32_t code_of(float x, float by) { return __float_as_uint(__fadd_rn(__fmul_rn(x, by), ROUND)); }

// Codes of VEC adjacent values a lane (VEC == 1: four that are 32 apart), a group of 128 in LANES lanes.
template <typename T, int VEC>
__global__ __launch_bounds__(KEEP_THREADS) void keep_kernel(const __grid_constant__ KeepArgs a) {
  constexpr int LANES = VEC == 1 ? 32 : KEPT_GROUP / VEC, E = VEC == 1 ? KEPT_GROUP / 32 : VEC, APART = VEC == 1 ? 32 : 1;
  constexpr int PER_CTA = KEEP_THREADS / LANES, WORDS = E * static_cast<int>(sizeof(T)) / 4;
  pdl_enter();
  const int lane = threadIdx.x % LANES, first = VEC == 1 ? lane : lane * VEC;
  const int64_t step = static_cast<int64_t>(gridDim.x) * PER_CTA;
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * PER_CTA + threadIdx.x / LANES; t0 - threadIdx.x / LANES < a.tasks; t0 += step * KEEP_UNROLL) {
    union Held {
      T v[E];
      uint32_t w[WORDS];
      __device__ Held() {}
    } x[KEEP_UNROLL];
    int64_t row[KEEP_UNROLL];
    int at[KEEP_UNROLL], group[KEEP_UNROLL];
#pragma unroll
    for (int u = 0; u < KEEP_UNROLL; ++u) {
      const int64_t t = t0 + u * step;
      row_and_group(a, t < a.tasks ? t : 0, &row[u], &group[u]);
      at[u] = t < a.tasks ? group[u] * KEPT_GROUP + first : a.D;
      const T* p = static_cast<const T*>(a.x) + row[u] * a.x_stride + at[u];
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[u].v[e] = at[u] + e * APART < a.D ? p[e * APART] : from_float<T>(0.0f);
      } else {
        const Vec<T, VEC> none{};
        *reinterpret_cast<Vec<T, VEC>*>(x[u].v) = at[u] < a.D ? *reinterpret_cast<const Vec<T, VEC>*>(p) : none;
      }
    }
#pragma unroll
    for (int u = 0; u < KEEP_UNROLL; ++u) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) top = largest_word<T>(top, x[u].w[i]);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = largest_word<T>(top, __shfl_xor_sync(FULL_MASK, top, o));
      const float big = largest_value<T>(top);
      float by = big > 0.0f ? 127.0f / big : 0.0f;
      if (!(big - big == 0.0f)) by = 0.0f;  // (nothing of such a group is kept)
      uint32_t c[E];
      if (by - by == 0.0f) {
#pragma unroll
        for (int e = 0; e < E; ++e) c[e] = code_of(to_float<T>(x[u].v[e]), by);
        if (!(big - big == 0.0f)) {
#pragma unroll
          for (int e = 0; e < E; ++e) c[e] = 0;
        }
      } else {  // 127 / a is no finite number
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float v = to_float<T>(x[u].v[e]);
          c[e] = v > 0.0f ? 127u : v < 0.0f ? static_cast<uint32_t>(-127) : 0u;
        }
      }
      int8_t* to = a.codes + row[u] * a.D + at[u];
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at[u] + e * APART < a.D) to[e * APART] = static_cast<int8_t>(c[e]);
      } else if (at[u] < a.D) {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
          w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
        *reinterpret_cast<Vec<uint32_t, VEC / 4>*>(to) = *reinterpret_cast<Vec<uint32_t, VEC / 4>*>(w);
      }
      if (lane == 0 && at[u] < a.D) a.scales[row[u] * a.groups + group[u]] = big / 127.0f;
    }
  }
}

// E codes a lane, adjacent (VEC > 1) or 32 apart
template <typename T, int VEC>
__global__ __launch_bounds__(KEEP_THREADS) void kept_values_kernel(const __grid_constant__ KeepArgs a) {
  constexpr int LANES = VEC == 1 ? 32 : KEPT_GROUP / VEC, E = VEC == 1 ? KEPT_GROUP / 32 : VEC, APART = VEC == 1 ? 32 : 1;
  constexpr int PER_CTA = KEEP_THREADS / LANES;
  pdl_enter();
  const int lane = threadIdx.x % LANES, first = VEC == 1 ? lane : lane * VEC;
  const int64_t step = static_cast<int64_t>(gridDim.x) * PER_CTA;
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * PER_CTA + threadIdx.x / LANES; t0 < a.tasks; t0 += step * KEEP_UNROLL) {
    union Held {
      int8_t v[E];
      uint32_t w[E / 4];
      __device__ Held() {}
    } c[KEEP_UNROLL];
    float scale[KEEP_UNROLL];
    int64_t row[KEEP_UNROLL];
    int at[KEEP_UNROLL];
#pragma unroll
    for (int u = 0; u < KEEP_UNROLL; ++u) {
      const int64_t t = t0 + u * step;
      int group;
      row_and_group(a, t < a.tasks ? t : 0, &row[u], &group);
      at[u] = t < a.tasks ? group * KEPT_GROUP + first : a.D;
      const int8_t* p = a.codes_in + row[u] * a.codes_stride + at[u];
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) c[u].v[e] = at[u] + e * APART < a.D ? p[e * APART] : 0;
      } else if (at[u] < a.D) {
        *reinterpret_cast<Vec<uint32_t, E / 4>*>(c[u].w) = *reinterpret_cast<const Vec<uint32_t, E / 4>*>(p);
      }
      scale[u] = at[u] < a.D ? __ldg(a.scales_in + row[u] * a.groups + group) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < KEEP_UNROLL; ++u) {
      if (at[u] >= a.D) continue;
      T* to = static_cast<T*>(a.out) + row[u] * a.D + at[u];
      float v[E];
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        // a byte with its sign turned in the last place of 2^23
        const uint32_t w = c[u].w[i] ^ 0x80808080u;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | e)) - 8388736.0f) * scale[u];
      }
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at[u] + e * APART < a.D) to[e * APART] = from_float<T>(v[e]);
      } else {
        constexpr int PIECE = VEC * sizeof(T) > 16 ? 16 / static_cast<int>(sizeof(T)) : VEC;
#pragma unroll
        for (int i = 0; i < VEC / PIECE; ++i) {
          float part[PIECE];
#pragma unroll
          for (int e = 0; e < PIECE; ++e) part[e] = v[i * PIECE + e];
          store_vec<T, PIECE>(to + i * PIECE, part);
        }
      }
    }
  }
}

unsigned keep_ctas(int64_t tasks, int lanes) {
  const int64_t per = static_cast<int64_t>(KEEP_THREADS / lanes) * KEEP_UNROLL, need = (tasks + per - 1) / per;
  const int64_t most = static_cast<int64_t>(sm_count()) * 8;
  return static_cast<unsigned>(need < most ? need : most);
}

// whether rows of both sides can be moved VEC elements at a time
template <typename T, int VEC>
bool by_vectors(const KeepArgs& a, const void* x, int64_t x_stride, const void* codes, int64_t codes_stride) {
  constexpr size_t bytes = VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16;
  return a.D % VEC == 0 && (x_stride % VEC == 0 || a.n <= 1) && (codes_stride % VEC == 0 || a.n <= 1) && aligned_to(x, bytes) && aligned_to(codes, VEC);
}
template <typename T, int VEC>
int keep_by(const KeepArgs& a, cudaStream_t s) {
  DGS_CUDA_TRY(launch_training(keep_kernel<T, VEC>, dim3(keep_ctas(a.tasks, VEC == 1 ? 32 : KEPT_GROUP / VEC)), KEEP_THREADS, 0, s, a));
  return DGS_OK;
}
template <typename T>
int keep(const KeepArgs& a, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  if (by_vectors<T, VEC>(a, a.x, a.x_stride, a.codes, a.D)) return keep_by<T, VEC>(a, s);
  if (VEC > 4 && by_vectors<T, 4>(a, a.x, a.x_stride, a.codes, a.D)) return keep_by<T, 4>(a, s);
  return keep_by<T, 1>(a, s);
}
template <typename T, int VEC>
int values_by(const KeepArgs& a, cudaStream_t s) {
  DGS_CUDA_TRY(launch_training(kept_values_kernel<T, VEC>, dim3(keep_ctas(a.tasks, VEC == 1 ? 32 : KEPT_GROUP / VEC)), KEEP_THREADS, 0, s, a));
  return DGS_OK;
}
template <typename T>
int values(const KeepArgs& a, cudaStream_t s) {
  if (by_vectors<T, 16>(a, a.out, a.D, a.codes_in, a.codes_stride)) return values_by<T, 16>(a, s);
  if (by_vectors<T, 4>(a, a.out, a.D, a.codes_in, a.codes_stride)) return values_by<T, 4>(a, s);
  return values_by<T, 1>(a, s);
}

// ---- the weight's gradient of 32-bit operands, on the CUDA cores ------------------------------------------------------------------------------
// A tile of 64 x 64 results a CTA over a share of the rows, 4 x 4 a thread; the shares are added in their order afterwards.
constexpr int WG_TILE = 64, WG_ROWS = 16, WG_THREADS = 256;

__global__ __launch_bounds__(WG_THREADS) void kept_grad_kernel(const __grid_constant__ KeptGradArgs a) {
  __shared__ __align__(16) float g[WG_ROWS][WG_TILE + 4], v[WG_ROWS][WG_TILE + 4];
  pdl_enter();
  const int o0 = blockIdx.y * WG_TILE, d0 = blockIdx.x * WG_TILE, split = blockIdx.z;
  const int64_t r0 = a.n * split / a.splits, r1 = a.n * (split + 1) / a.splits;
  const int to = threadIdx.x / 16 * 4, td = threadIdx.x % 16 * 4;
  float acc[4][4] = {}, db = 0.0f;
  for (int64_t r = r0; r < r1; r += WG_ROWS) {
    for (int i = threadIdx.x; i < WG_ROWS * WG_TILE; i += WG_THREADS) {
      const int row = i / WG_TILE, c = i % WG_TILE;
      const bool in = r + row < r1;
      g[row][c] = in && o0 + c < a.O ? static_cast<const float*>(a.grad)[(r + row) * a.grad_stride + o0 + c] : 0.0f;
      v[row][c] = in && d0 + c < a.D ? static_cast<float>(a.codes[(r + row) * a.codes_stride + d0 + c]) * a.scales[(r + row) * a.groups + (d0 + c) / KEPT_GROUP]
                                     : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < WG_ROWS; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(&g[k][to]), y = *reinterpret_cast<const float4*>(&v[k][td]);
      const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[i], ys[j], acc[i][j]);
    }
    if (threadIdx.x < WG_TILE)
#pragma unroll
      for (int k = 0; k < WG_ROWS; ++k) db += g[k][threadIdx.x];
    __syncthreads();
  }
  float* part = a.parts + static_cast<int64_t>(split) * a.O * a.D;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (o0 + to + i < a.O && d0 + td + j < a.D) part[static_cast<int64_t>(o0 + to + i) * a.D + d0 + td + j] = acc[i][j];
  if (d0 == 0 && threadIdx.x < WG_TILE && o0 + threadIdx.x < a.O) a.bias_parts[static_cast<int64_t>(split) * a.O + o0 + threadIdx.x] = db;
}

// Shares added in a fixed order: WAYS warps take every WAYS-th share of the same 32 results (or 128: VEC of them a lane), then one adds theirs
template <typename T, int WAYS, int VEC>
__global__ __launch_bounds__(KEEP_THREADS) void kept_join_kernel(const __grid_constant__ KeptGradArgs a) {
  __shared__ float part[KEEP_THREADS / 32][32][VEC];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, way = warp % WAYS;
  constexpr int ALONG = KEEP_THREADS / 32 / WAYS;  // sets of results a CTA
  const int64_t all = static_cast<int64_t>(a.O) * a.D, both = all + (a.dbias != nullptr ? a.O : 0);
  const int64_t i = ((static_cast<int64_t>(blockIdx.x) * ALONG + warp / WAYS) * 32 + lane) * VEC;
  float s[VEC] = {};
  // (with VEC > 1 all and O are multiples of it)
  const float* from = i < all ? a.parts + i : a.bias_parts + (i - all);
  const int64_t apart = i < all ? all : a.O;
  if (i < both) {
#pragma unroll 4
    for (int p = way; p < a.splits; p += WAYS) {
      float x[VEC];
      load_vec<float, VEC>(from + p * apart, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] += x[e];
    }
  }
  if constexpr (WAYS > 1) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[warp][lane][e] = s[e];
    __syncthreads();
    if (way != 0) return;
#pragma unroll
    for (int w = 1; w < WAYS; ++w)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] += part[warp + w][lane][e];
  }
  if (i < all) store_vec<T, VEC>(static_cast<T*>(a.dweight) + i, s);
  else if (i < both) store_vec<T, VEC>(static_cast<T*>(a.dbias) + (i - all), s);
}

// Shares of the rows: enough CTAs for four on each SM, shares of 256 rows at least
int64_t shares(int64_t n, int64_t O, int64_t D, int32_t dtype) {
  if (dtype != DGS_F32) return kept_mma_shares(n, O, D);
  const int64_t tiles = ((O + WG_TILE - 1) / WG_TILE) * ((D + WG_TILE - 1) / WG_TILE);
  int64_t want = (static_cast<int64_t>(sm_count()) * 4 + tiles - 1) / tiles;
  const int64_t most = (n + 255) / 256;
  if (want > most) want = most;
  return want < 1 ? 1 : want;
}

template <typename T, int WAYS, int VEC>
int join_by(const KeptGradArgs& a, cudaStream_t s) {
  const int64_t both = static_cast<int64_t>(a.O) * a.D + (a.dbias != nullptr ? a.O : 0), per = KEEP_THREADS / WAYS * VEC;
  DGS_CUDA_TRY(launch_training(kept_join_kernel<T, WAYS, VEC>, dim3(static_cast<unsigned>((both + per - 1) / per)), KEEP_THREADS, 0, s, a));
  return DGS_OK;
}
template <typename T>
int join(const KeptGradArgs& a, cudaStream_t s) {
  const bool wide = (static_cast<int64_t>(a.O) * a.D) % 4 == 0 && (a.dbias == nullptr || a.O % 4 == 0) && aligned_to(a.dweight, 16) && aligned_to(a.dbias, 16);
  if (a.splits > 8) return wide ? join_by<T, 8, 4>(a, s) : join_by<T, 8, 1>(a, s);
  return wide ? join_by<T, 1, 4>(a, s) : join_by<T, 1, 1>(a, s);
}

int weight_grad(const KeptGradArgs& a, int32_t dtype, cudaStream_t s) {
  if (dtype != DGS_F32) {
    if (int rc = kept_mma_weight_grad(a, dtype, s)) return rc;
    return a.splits == 1 ? DGS_OK : dtype == DGS_BF16 ? join<__nv_bfloat16>(a, s) : join<__half>(a, s);
  }
  const dim3 grid(static_cast<unsigned>((a.D + WG_TILE - 1) / WG_TILE), static_cast<unsigned>((a.O + WG_TILE - 1) / WG_TILE),
                  static_cast<unsigned>(a.splits));
  DGS_CUDA_TRY(launch_training(kept_grad_kernel, grid, WG_THREADS, 0, s, a));
  return join<float>(a, s);
}

constexpr int64_t KEPT_MAX_SIDE = int64_t(1) << 22;  // elements of a row

int check(const char* who, int64_t n, int64_t D, int32_t dtype) {
  DGS_REQUIRE(dtype_bytes(dtype) != 0, DGS_ERR_UNSUPPORTED, "%s: element type %d", who, dtype);
  DGS_REQUIRE(n >= 0 && D >= 1 && D <= KEPT_MAX_SIDE && n < (int64_t(1) << 31), DGS_ERR_INVALID, "%s: %lld rows of %lld elements", who,
              static_cast<long long>(n), static_cast<long long>(D));
  return DGS_OK;
}

}  // namespace
}  // namespace dgs

using namespace dgs;

extern "C" int dgs_keep_8bit(const void* x, int64_t x_stride, int32_t dtype, int64_t n, int64_t D, int8_t* codes, float* scales,
                             dgs_stream_t stream) {
  if (int rc = check("keep_8bit", n, D, dtype)) return rc;
  DGS_REQUIRE(x_stride >= D || n <= 1, DGS_ERR_INVALID, "keep_8bit: rows that overlap");
  if (n == 0) return DGS_OK;
  DGS_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, DGS_ERR_INVALID, "keep_8bit: null argument");
  KeepArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.codes = codes;
  a.scales = scales;
  a.n = n;
  a.D = static_cast<int32_t>(D);
  a.groups = static_cast<int32_t>((D + KEPT_GROUP - 1) / KEPT_GROUP);
  a.tasks = n * a.groups;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == DGS_F32 ? keep<float>(a, s) : dtype == DGS_BF16 ? keep<__nv_bfloat16>(a, s) : keep<__half>(a, s);
}

extern "C" int dgs_kept_8bit_values(const int8_t* codes, int64_t codes_stride, const float* scales, int64_t n, int64_t D, int32_t dtype,
                                    void* out, dgs_stream_t stream) {
  if (int rc = check("kept_8bit_values", n, D, dtype)) return rc;
  DGS_REQUIRE(codes_stride >= D || n <= 1, DGS_ERR_INVALID, "kept_8bit_values: rows that overlap");
  if (n == 0) return DGS_OK;
  DGS_REQUIRE(codes != nullptr && scales != nullptr && out != nullptr, DGS_ERR_INVALID, "kept_8bit_values: null argument");
  KeepArgs a{};
  a.codes_in = codes;
  a.codes_stride = codes_stride;
  a.scales_in = scales;
  a.out = out;
  a.n = n;
  a.D = static_cast<int32_t>(D);
  a.groups = static_cast<int32_t>((D + KEPT_GROUP - 1) / KEPT_GROUP);
  a.tasks = n * a.groups;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == DGS_F32 ? values<float>(a, s) : dtype == DGS_BF16 ? values<__nv_bfloat16>(a, s) : values<__half>(a, s);
}

extern "C" size_t dgs_kept_8bit_weight_grad_workspace_bytes(int64_t n, int64_t O, int64_t D, int32_t dtype) {
  if (n <= 0 || O <= 0 || D <= 0 || dtype_bytes(dtype) == 0) return 0;
  const size_t splits = static_cast<size_t>(shares(n, O, D, dtype));
  return splits * (static_cast<size_t>(O) * D + O) * sizeof(float);
}

extern "C" int dgs_kept_8bit_weight_grad(const void* grad, int64_t grad_stride, int32_t dtype, const int8_t* codes, int64_t codes_stride,
                                         const float* scales, int64_t n, int64_t O, int64_t D, void* dweight, void* dbias,
                                         void* workspace, size_t workspace_bytes, dgs_stream_t stream) {
  return dgs_kept_8bit_weight_grad_reported(grad, grad_stride, dtype, codes, codes_stride, scales, n, O, D, dweight, dbias, workspace,
                                            workspace_bytes, nullptr, stream);
}

extern "C" int dgs_kept_8bit_weight_grad_reported(const void* grad, int64_t grad_stride, int32_t dtype, const int8_t* codes,
                                                  int64_t codes_stride, const float* scales, int64_t n, int64_t O, int64_t D, void* dweight,
                                                  void* dbias, void* workspace, size_t workspace_bytes, int32_t* status,
                                                  dgs_stream_t stream) {
  if (int rc = check("kept_8bit_weight_grad", n, D, dtype)) return rc;
  // (tiles of the weight's rows are the grid's second extent, below 2^16; the join's CTAs its first, below 2^31)
  DGS_REQUIRE(O >= 1 && O < KEPT_MAX_SIDE / 2 && O * D < (int64_t(1) << 35), DGS_ERR_INVALID, "kept_8bit_weight_grad: a weight of %lld rows of %lld",
              static_cast<long long>(O), static_cast<long long>(D));
  DGS_REQUIRE((grad_stride >= O && codes_stride >= D) || n <= 1, DGS_ERR_INVALID, "kept_8bit_weight_grad: rows that overlap");
  DGS_REQUIRE(dweight != nullptr, DGS_ERR_INVALID, "kept_8bit_weight_grad: null argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n == 0) {
    DGS_CUDA_TRY(cudaMemsetAsync(dweight, 0, static_cast<size_t>(O) * D * dtype_bytes(dtype), s));
    if (dbias != nullptr) DGS_CUDA_TRY(cudaMemsetAsync(dbias, 0, static_cast<size_t>(O) * dtype_bytes(dtype), s));
    return DGS_OK;
  }
  const size_t need = dgs_kept_8bit_weight_grad_workspace_bytes(n, O, D, dtype);
  DGS_REQUIRE(grad != nullptr && codes != nullptr && scales != nullptr, DGS_ERR_INVALID, "kept_8bit_weight_grad: null argument");
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "kept_8bit_weight_grad: workspace of %zu bytes, 256-byte aligned, is needed", need);
  KeptGradArgs a{};
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.codes = codes;
  a.codes_stride = codes_stride;
  a.scales = scales;
  a.n = n;
  a.O = static_cast<int32_t>(O);
  a.D = static_cast<int32_t>(D);
  a.groups = static_cast<int32_t>((D + KEPT_GROUP - 1) / KEPT_GROUP);
  a.splits = static_cast<int32_t>(shares(n, O, D, dtype));
  a.parts = static_cast<float*>(workspace);
  a.bias_parts = a.parts + static_cast<int64_t>(a.splits) * O * D;
  a.dweight = dweight;
  a.dbias = dbias;
  a.status = status;
  a.wait_limit = wait_limit();
  return weight_grad(a, dtype, s);
}
