// The gradient of a linear layer's weight from rows kept in 8 bits, 16-bit gradients, on the tensor cores:
//   dW[o, d] = sum_n g[n, o] v[n, d],  v = code * scale rounded to g's type (so that products are exact; sums are in 32 bits)
//
// A CTA takes 256 x 256 results over a share of the rows, 64 at a time: sixteen warps fetch rows of g and codes, turn the codes into
// values and leave both in shared memory as they lie (the sum's index outermost: MN-major tiles), a thread of a seventeenth issues the
// products (cta_group::1, two accumulators of 128 x 256 in TMEM).  The next blocks are on their way in registers.
// With few results the rows are cut into shares that fill the SMs; shares are added in their order by a second launch.
// Every wait is bounded; one that runs out raises DGS_ERR_CUDA in the status word, leaves no number among the CTA's results, and all roles leave.
// Bound by turning codes into operands: 430 000 rows of 256 against 47 (358 bytes a row) 55 us = 2.8 TB/s, 16 384 x 4 096 against 1 024 165 us =
// 833 TFLOP/s with the tensor pipe 41 % active, each with 9 to 10 us of joins behind it.
#include "kept.h"
#include "tensor_core.cuh"

namespace dgs {
namespace {
using namespace tc;

constexpr int TILE = 256, ROWS = 64, FETCH_WARPS = 16, FETCHERS = FETCH_WARPS * 32, THREADS = FETCHERS + 128, STAGES = 3;
// Registers: 5 x 128 x 96 at the launch; the four warpgroups that fetch take what the products' one leaves
constexpr int MANY_REGISTERS = 104, FEW_REGISTERS = 64;
constexpr uint32_t PANEL = ROWS * 128;                 // 64 columns of 64 rows
constexpr uint32_t OPERAND = TILE / 64 * PANEL, STAGE = 2 * OPERAND;
constexpr uint32_t BARS = STAGES * STAGE, SMEM = BARS + 128;
constexpr int NARROW = 64;  // results a row of the weight: up to here one piece of a row a thread instead of four, and more blocks on their way
constexpr int C_CHUNKS = TILE / 16, C_TASKS = ROWS * C_CHUNKS / FETCHERS;  // 16 codes
constexpr int MAX_DEVICES = 64;

// 16 bytes from `p` on, of which `left` belong to the row (none: zeros).  ALIGNED: at 16-byte boundaries, whole; else put together out of
// the aligned words that hold them (what lies behind the row comes as anything, a word that holds none of it is not read).
template <bool ALIGNED>
struct Piece {
  uint32_t w[ALIGNED ? 4 : 5];
  __device__ __forceinline__ void fetch(const char* p, int left) {
    if constexpr (ALIGNED) {
      const uint4 v = left > 0 ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
      const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p - off);
      const int stop = left > 0 ? left + off : 0;
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = 4 * i < stop ? __ldg(q + i) : 0u;
    }
  }
  __device__ __forceinline__ void line_up(const char* p) {
    if constexpr (!ALIGNED) {
      const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], shift);
    }
  }
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// four codes to four values, 16 bits each: a byte with its sign turned, in the last place of 2^23, is a number that 2^23 + 128 takes to the code
template <bool BF16>
__device__ __forceinline__ void values_of(uint32_t codes, float scale, uint32_t* lo, uint32_t* hi) {
  const uint32_t u = codes ^ 0x80808080u;
  const uint64_t less = two(-8388736.0f, -8388736.0f), by = two(scale, scale);
  const auto number = [&](int i) { return __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | i)); };
  float v[4];
  split2(mul2(add2(two(number(0), number(1)), less), by), &v[0], &v[1]);
  split2(mul2(add2(two(number(2), number(3)), less), by), &v[2], &v[3]);
  *lo = pack2<BF16>(v[0], v[1]);
  *hi = pack2<BF16>(v[2], v[3]);
}

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t w, float* lo, float* hi) {
  if constexpr (BF16) {
    *lo = __uint_as_float(w << 16);
    *hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    *lo = f.x;
    *hi = f.y;
  }
}

// A thread's share of 64 rows on their way: the same pieces of some rows of g, 16 codes and their scale of others
template <bool G_ALIGNED, bool C_ALIGNED, int G_TASKS>
struct Block {
  Piece<G_ALIGNED> g[G_TASKS];
  Piece<C_ALIGNED> c[C_TASKS];
  float scale[C_TASKS];
};

template <bool BF16, bool G_ALIGNED, bool C_ALIGNED, bool FEW>
__global__ __launch_bounds__(THREADS, 1) void kept_mma_kernel(const __grid_constant__ KeptGradArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int G_CHUNKS = (FEW ? NARROW : TILE) / 8, G_TASKS = ROWS * G_CHUNKS / FETCHERS;  // 16-byte pieces of g's rows
  constexpr int DEPTH = FEW ? 4 : 2;                                                        // blocks of rows on their way
  const uint32_t smem = smem_addr(smem_raw), full = smem + BARS, empty = full + 8 * STAGES, done = empty + 8 * STAGES, summed = done + 8,
                 tmem_word = summed + 8;
  volatile int* dead = reinterpret_cast<volatile int*>(smem_raw + (tmem_word + 4 - smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      bar_init(full + 8 * i, FETCHERS);
      bar_init(empty + 8 * i, 1);
    }
    bar_init(done, 1);
    bar_init(summed, FETCHERS);
    *dead = 0;
    bar_init_fence();
  }
  if (warp == 0) tmem_alloc_one(tmem_word, 512);
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_word) : "memory");
  pdl_enter();
  const int d0 = blockIdx.x * TILE, o0 = blockIdx.y * TILE, split = blockIdx.z;
  const int64_t r0 = a.n * split / a.splits, r1 = a.n * (split + 1) / a.splits;
  const int blocks = static_cast<int>((r1 - r0 + ROWS - 1) / ROWS);
  const int cols = min(TILE, a.D - d0), outs = min(TILE, a.O - o0);
  const Waits wait{dead, a.wait_limit};
  bool ok = true;

  if (warp < FETCH_WARPS) {
    more_registers<MANY_REGISTERS>();
    const int g_chunk = threadIdx.x % G_CHUNKS, g_row = threadIdx.x / G_CHUNKS;  // (the same piece of every row of this thread)
    // eight neighbouring lanes: four pieces of one panel's rows, in two rows, so that their 16 bytes lie in different banks
    const int c_chunk = (lane & 3) | (lane >> 3 << 2), c_row = warp * 2 + (lane >> 2 & 1);
    constexpr int G_STEP = FETCHERS / G_CHUNKS, C_STEP = FETCHERS / C_CHUNKS;  // (both multiples of 8: the swizzle is a thread's own)
    const int64_t g_pitch = a.grad_stride * 2, c_pitch = a.codes_stride;
    const int g_left = outs * 2 - g_chunk * 16, c_left = cols - c_chunk * 16;
    const bool g_in = g_left > 0, c_in = c_left > 0;
    const bool sums = a.dbias != nullptr && blockIdx.x == 0;
    // where this thread's first row of the next block to be fetched is; rows of the share from there on
    const char* g = static_cast<const char*>(a.grad) + static_cast<int64_t>(o0) * 2 + (r0 + g_row) * g_pitch + g_chunk * 16;
    const char* c = reinterpret_cast<const char*>(a.codes) + d0 + (r0 + c_row) * c_pitch + c_chunk * 16;
    const float* scales = a.scales + (r0 + c_row) * a.groups + (d0 + c_chunk * 16) / KEPT_GROUP;
    int rows = static_cast<int>(r1 - r0);
    float db[8] = {};
    Block<G_ALIGNED, C_ALIGNED, G_TASKS> on_way[DEPTH];
    const auto fetch = [&](Block<G_ALIGNED, C_ALIGNED, G_TASKS>& x) {
#pragma unroll
      for (int i = 0; i < G_TASKS; ++i) x.g[i].fetch(g + i * (G_STEP * g_pitch), g_row + i * G_STEP < rows ? g_left : 0);
#pragma unroll
      for (int i = 0; i < C_TASKS; ++i) {
        const bool in = c_row + i * C_STEP < rows;
        x.c[i].fetch(c + i * (C_STEP * c_pitch), in ? c_left : 0);
        x.scale[i] = in && c_in ? __ldg(scales + i * (C_STEP * a.groups)) : 0.0f;
      }
      g += ROWS * g_pitch;
      c += ROWS * c_pitch;
      scales += static_cast<int64_t>(ROWS) * a.groups;
      rows -= ROWS;
    };
    int slot = 0;
    uint32_t phase = 0;
    const uint32_t g_to = smem + (g_chunk / 8) * PANEL + g_row * 128 + (((g_chunk & 7) ^ (g_row & 7)) << 4);
    const uint32_t c_to = smem + OPERAND + (c_chunk / 4) * PANEL + c_row * 128, c_low = ((c_chunk & 3) * 2 ^ (c_row & 7)) << 4;
    const auto store = [&](Block<G_ALIGNED, C_ALIGNED, G_TASKS>& x) {
      const uint32_t at = slot * STAGE;
      if (g_in) {
#pragma unroll
        for (int i = 0; i < G_TASKS; ++i) {
          // (DEPTH blocks of 64 rows on: the same place within a word as then)
          x.g[i].line_up(g + i * (G_STEP * g_pitch));
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(g_to + at + i * (G_STEP * 128)), "r"(x.g[i].w[0]), "r"(x.g[i].w[1]),
                       "r"(x.g[i].w[2]), "r"(x.g[i].w[3])
                       : "memory");
          if (sums) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo, hi;
              unpack2<BF16>(x.g[i].w[e], &lo, &hi);
              db[2 * e] += lo;
              db[2 * e + 1] += hi;
            }
          }
        }
      }
      if (c_in) {
#pragma unroll
        for (int i = 0; i < C_TASKS; ++i) {
          x.c[i].line_up(c + i * (C_STEP * c_pitch));
          uint32_t v[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) values_of<BF16>(x.c[i].w[e], x.scale[i], &v[2 * e], &v[2 * e + 1]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(c_to + at + i * (C_STEP * 128) + (c_low ^ (h << 4))), "r"(v[4 * h]),
                         "r"(v[4 * h + 1]), "r"(v[4 * h + 2]), "r"(v[4 * h + 3])
                         : "memory");
        }
      }
    };
#pragma unroll
    for (int w = 0; w < DEPTH; ++w) fetch(on_way[w]);  // (rows behind the share are not read)
    for (int b0 = 0; ok && b0 < blocks; b0 += DEPTH) {
#pragma unroll
      for (int w = 0; w < DEPTH; ++w) {
        if (!ok || b0 + w >= blocks) continue;
        if (!(ok = wait(empty + 8 * slot, phase ^ 1))) continue;
        store(on_way[w]);
        fence_async_smem();
        bar_arrive(full + 8 * slot);
        fetch(on_way[w]);
        if (++slot == STAGES) slot = 0, phase ^= 1;
      }
    }
    ok = __all_sync(FULL_MASK, ok && (blocks == 0 || wait(done, 0)));  // (the loads below are the whole warp's)
    if (ok) {
      // ---- results: a row of the weight a thread
      fence_after();
      const int which = warp / 8, o = which * 128 + warp % 4 * 32 + lane;  // an accumulator, every second 32 of its columns
      const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
      if (which * 128 < outs) {
#pragma unroll 1
        for (int q = warp / 4 % 2; q * 32 < cols; q += 2) {
          uint32_t v[32];
          if (blocks > 0) {
            tmem_load32(tmem + which * 256 + q * 32 + lanes, v);
            tmem_wait(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0;
          }
          if (o < outs) {
            const int64_t at = static_cast<int64_t>(o0 + o) * a.D + d0 + q * 32;
            const int left = cols - q * 32;
            if (a.splits == 1) {
              uint16_t* to = static_cast<uint16_t*>(a.dweight) + at;
              if (left >= 32 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  uint32_t y[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) y[e] = pack2<BF16>(__uint_as_float(v[i * 8 + e * 2]), __uint_as_float(v[i * 8 + e * 2 + 1]));
                  reinterpret_cast<uint4*>(to)[i] = make_uint4(y[0], y[1], y[2], y[3]);
                }
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (i < left) to[i] = static_cast<uint16_t>(pack2<BF16>(__uint_as_float(v[i]), 0.0f));
              }
            } else {
              float* to = a.parts + static_cast<int64_t>(split) * a.O * a.D + at;
              if (left >= 32 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (i < left) to[i] = __uint_as_float(v[i]);
              }
            }
          }
          __syncwarp();
        }
      }
      if (sums) {
        // the threads that took the same columns, in their order (the tiles' memory is free)
        float* part = reinterpret_cast<float*>(smem_raw);
#pragma unroll
        for (int e = 0; e < 8; ++e) part[g_row * G_CHUNKS * 8 + g_chunk * 8 + e] = db[e];
        bar_arrive(summed);
        ok = wait(summed, 0);
        if (ok && static_cast<int>(threadIdx.x) < outs) {
          float s = 0.0f;
#pragma unroll 8
          for (int q = 0; q < G_STEP; ++q) s += part[q * G_CHUNKS * 8 + threadIdx.x];
          if (a.splits > 1) a.bias_parts[static_cast<int64_t>(split) * a.O + o0 + threadIdx.x] = s;
          else static_cast<uint16_t*>(a.dbias)[o0 + threadIdx.x] = static_cast<uint16_t>(pack2<BF16>(s, 0.0f));
        }
      }
      fence_before();
    }
  } else {
    fewer_registers<FEW_REGISTERS>();
    if (warp == FETCH_WARPS && lane == 0) {
      // ---- products
      const uint32_t n = static_cast<uint32_t>((cols + 15) / 16 * 16), idesc = mma_desc(BF16, true, true, 128, n);
      int slot = 0;
      uint32_t phase = 0;
      for (int b = 0; b < blocks; ++b) {
        if (!(ok = wait(full + 8 * slot, phase))) break;
        fence_after();
        const uint64_t da = smem_desc(smem + slot * STAGE, PANEL, 1024), dv = smem_desc(smem + slot * STAGE + OPERAND, PANEL, 1024);
#pragma unroll
        for (int k = 0; k < ROWS / 16; ++k) {
          mma_one(tmem, da + k * (2048 >> 4), dv + k * (2048 >> 4), idesc, b > 0 || k > 0);
          if (outs > 128) mma_one(tmem + 256, da + (2 * PANEL >> 4) + k * (2048 >> 4), dv + k * (2048 >> 4), idesc, b > 0 || k > 0);
        }
        mma_commit_one(empty + 8 * slot);
        if (++slot == STAGES) slot = 0, phase ^= 1;
      }
      if (ok) mma_commit_one(done);
    }
  }
  __syncwarp();
  if (!ok) {
    *dead = 1;
    raise_status(a.status, DGS_ERR_CUDA);
  }
  __syncthreads();
  if (*dead) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    // (found anew, so that nothing of it is held all the way here)
    const int d0 = blockIdx.x * TILE, o0 = blockIdx.y * TILE, split = blockIdx.z, cols = min(TILE, a.D - d0), outs = min(TILE, a.O - o0);
    // a call without a status word shows it too: none of this CTA's results is a number
    for (int i = threadIdx.x; i < outs * cols; i += THREADS) {
      const int64_t at = static_cast<int64_t>(o0 + i / cols) * a.D + d0 + i % cols;
      if (a.splits > 1) a.parts[static_cast<int64_t>(split) * a.O * a.D + at] = __uint_as_float(0x7fffffffu);
      else static_cast<uint16_t*>(a.dweight)[at] = 0x7fffu;
    }
    if (a.dbias != nullptr && blockIdx.x == 0) {
      for (int i = threadIdx.x; i < outs; i += THREADS) {
        if (a.splits > 1) a.bias_parts[static_cast<int64_t>(split) * a.O + o0 + i] = __uint_as_float(0x7fffffffu);
        else static_cast<uint16_t*>(a.dbias)[o0 + i] = 0x7fffu;
      }
    }
  }
  if (warp == 0) {
    fence_after();
    tmem_free_one(tmem, 512);
  }
}

template <bool BF16, bool G_ALIGNED, bool C_ALIGNED, bool FEW>
int launch(const KeptGradArgs& a, cudaStream_t s) {
  static_assert(SMEM <= 232448, "shared memory");
  static std::atomic<bool> known[MAX_DEVICES] = {};
  auto kernel = kept_mma_kernel<BF16, G_ALIGNED, C_ALIGNED, FEW>;
  int dev = 0;
  DGS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= MAX_DEVICES || !known[dev].load(std::memory_order_relaxed)) {
    DGS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SMEM)));
    if (dev < MAX_DEVICES) known[dev].store(true, std::memory_order_relaxed);
  }
  const dim3 grid(static_cast<unsigned>((a.D + TILE - 1) / TILE), static_cast<unsigned>((a.O + TILE - 1) / TILE), static_cast<unsigned>(a.splits));
  DGS_CUDA_TRY(launch_training(kernel, grid, THREADS, SMEM, s, a));
  return DGS_OK;
}
template <bool BF16>
int launch_aligned(const KeptGradArgs& a, cudaStream_t s) {
  const bool g = a.grad_stride % 8 == 0 && a.O % 8 == 0 && aligned_to(a.grad, 16);
  const bool c = a.codes_stride % 16 == 0 && a.D % 16 == 0 && aligned_to(a.codes, 16);
  if (a.O <= NARROW)
    return g ? (c ? launch<BF16, true, true, true>(a, s) : launch<BF16, true, false, true>(a, s))
             : (c ? launch<BF16, false, true, true>(a, s) : launch<BF16, false, false, true>(a, s));
  return g ? (c ? launch<BF16, true, true, false>(a, s) : launch<BF16, true, false, false>(a, s))
           : (c ? launch<BF16, false, true, false>(a, s) : launch<BF16, false, false, false>(a, s));
}

}  // namespace

// Shares of the rows: what a share takes (rows at a tile's 16 cycles each, in as many rounds of CTAs as there are) against writing and
// adding one more (8 bytes a result): both in units of a row of a tile, some 9.4 ns; 4 TB/s.
int64_t kept_mma_shares(int64_t n, int64_t O, int64_t D) {
  const int64_t tiles = ((O + TILE - 1) / TILE) * ((D + TILE - 1) / TILE), sms = sm_count();
  int64_t most = (n + 8 * ROWS - 1) / (8 * ROWS), best = 1;
  if (most > sms) most = sms;
  double least = 0.0;
  for (int64_t s = 1; s <= most; ++s) {
    const double rounds = static_cast<double>((tiles * s + sms - 1) / sms);
    const double cost = rounds * static_cast<double>(n) / static_cast<double>(s) + (s > 1 ? static_cast<double>(s) * O * D * 8.0 / 4e12 / 9.4e-9 : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

int kept_mma_weight_grad(const KeptGradArgs& a, int32_t dtype, cudaStream_t s) {
  return dtype == DGS_BF16 ? launch_aligned<true>(a, s) : launch_aligned<false>(a, s);
}

}  // namespace dgs
