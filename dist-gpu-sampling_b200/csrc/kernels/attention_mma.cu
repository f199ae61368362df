// Attention of long sequences in 16 bits on the tensor cores (formulas: attention.cu).
//
// Forward: a CTA takes 256 queries of one head as two tiles of 128 and runs over the keys 128 at a time.
//   S = Q K^T           both operands out of shared memory, 128 columns of TMEM for each query tile
//   P = exp2(S c - ref) a thread a row: TMEM -> registers -> TMEM, 16 bits, in S's place
//   O += P V            P out of TMEM, V as it lies (its rows are the sum's index), O stays in TMEM for all keys
// While one tile's exponentials run, the tensor cores work on the other's products.  `ref` follows the running maximum of a row only
// when that has grown by more than 2^8 (the sums are in 32 bits and divided in the end), so O is hardly ever rescaled.
// Rows travel by cp.async: rows behind a sequence's end, and elements behind a head's, are zeros and never those of a neighbour.
// Every wait is bounded; a wait that runs out raises DGS_ERR_CUDA in the status word and all roles leave.
#include "attention.h"
#include "tensor_core.cuh"

namespace dgs {
namespace {
using namespace tc;

constexpr int SOFTMAX_WARPS = 8, LOAD_WARPS = 2;
constexpr int LOAD_THREADS = LOAD_WARPS * 32;
constexpr int TILE_THREADS = 384;  // three warpgroups: two of a row (or half of one) a thread, one of the products' and the loading warps
// Registers: 3 x 128 x 168 at the launch; the first two take what the third leaves
constexpr int MANY_REGISTERS = 208, FEW_REGISTERS = 80;
constexpr uint32_t TMEM_COLS = 512;
constexpr int MAX_SMEM = 232448;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LAZY = 8.0f;  // powers of two by which a row's maximum may outgrow its reference
constexpr int MAX_DEVICES = 64;

template <int DP>
constexpr uint32_t tile_bytes() {
  return ATTN_TILE * DP * 2;
}
constexpr uint32_t PANEL = ATTN_TILE * 128;  // 128 rows of 64 elements

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---- rows into shared memory ------------------------------------------------------------------------------------------
// 128 rows of a head (`there` of them exist), panels of 64 elements, 128-byte swizzle, asked for with cp.async by the loading threads
template <int DP>
__device__ __forceinline__ void ask_tile(uint32_t dst, const char* p, int64_t row_bytes, int there, int d, int t) {
  constexpr int CHUNKS = DP / 8, ROWS = LOAD_THREADS / CHUNKS;  // 16-byte pieces of a row; rows a pass (a multiple of 8, or half of it)
  const int c = t % CHUNKS, r0 = t / CHUNKS;
  const bool in_d = c * 8 < d;
  const char* src = p + r0 * row_bytes + c * 16;
  const uint32_t base = dst + (c / 8) * PANEL + r0 * 128;
#pragma unroll
  for (int i = 0; i < ATTN_TILE / ROWS; ++i) {
    const int r = r0 + i * ROWS;
    const bool in = in_d && r < there;
    const uint32_t to = base + i * ROWS * 128 + (((c & 7) ^ (r & 7)) << 4);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(in ? src : p), "r"(in ? 16 : 0) : "memory");
    src += ROWS * row_bytes;
  }
}
__device__ __forceinline__ void ask_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void ask_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A ring of stages that the loading threads fill in order; a stage is handed over once the two asked for after it are under way.
template <int STAGES>
struct Ring {
  uint32_t full, empty;
  int at = 0, handed = 0;  // stages asked for, handed over
  __device__ __forceinline__ int slot() const { return at % STAGES; }
  __device__ __forceinline__ bool wait_empty(const volatile int* dead) const {
    return !*dead && bar_wait(empty + 8 * (at % STAGES), ((at / STAGES) & 1) ^ 1);
  }
  template <int LEFT>
  __device__ __forceinline__ void hand_over() {  // all but the newest LEFT
    ask_wait<LEFT>();
    fence_async_smem();
    for (; handed < at - LEFT; ++handed) bar_arrive(full + 8 * (handed % STAGES));
  }
  __device__ __forceinline__ void asked() {
    ask_commit();
    ++at;
    hand_over<2>();
  }
};

// ---- products ---------------------------------------------------------------------------------------------------------
// D[128, 128] = A[128, DP] B[128, DP]^T, both K-major tiles in shared memory
template <int DP>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  const uint64_t da = smem_desc(a, 16, 1024), db = smem_desc(b, 16, 1024);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint64_t step = (k / 4) * (PANEL >> 4) + (k % 4) * 2;
    mma_one(d, da + step, db + step, idesc, k > 0);
  }
}
// D[128, DP] += A[128, 128] B[128, DP]: A in TMEM (the second half of its columns begins at `half`), B's rows are the sum's index
template <int DP>
__device__ __forceinline__ void product_columns(uint32_t d, uint32_t a, uint32_t half, uint32_t b, uint32_t idesc, bool accumulate) {
  const uint64_t db = smem_desc(b, PANEL, 1024);
#pragma unroll
  for (int k = 0; k < ATTN_TILE / 16; ++k)
    mma_one_tmem(d, a + (k / 4) * half + (k % 4) * 8, db + k * (2048 >> 4), idesc, accumulate || k > 0);
}

__device__ __forceinline__ void take(int4* to, const AttnTile* p) {
  to[0] = reinterpret_cast<const int4*>(p)[0];
  to[1] = reinterpret_cast<const int4*>(p)[1];
}
__device__ __forceinline__ AttnTile tile_at(const AttnTile* p) {
  AttnTile t;
  take(reinterpret_cast<int4*>(&t), p);
  return t;
}

// ---- forward ----------------------------------------------------------------------------------------------------------
template <int DP>
struct ForwardShape {
  static constexpr int STAGES = DP == 128 ? 5 : 8;
  static constexpr uint32_t RING = 2 * tile_bytes<DP>(), BARS = RING + STAGES * tile_bytes<DP>(), SMEM = BARS + 256;
};

// 128 scores of a row in powers of two: the largest, with those that the row does not see at minus infinity
template <bool MASK>
__device__ __forceinline__ float scores(uint32_t tmem, int seen, uint32_t (&v)[4][32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_load32(tmem + c * 32, v[c]);
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_wait(v[c]);
  float top = -INFINITY;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (MASK && c * 32 + i >= seen) v[c][i] = __float_as_uint(-INFINITY);
      top = fmaxf(top, __uint_as_float(v[c][i]));
    }
  return top;
}

template <int DP, bool BF16>
__global__ __launch_bounds__(TILE_THREADS, 1) void attn_forward_kernel(const __grid_constant__ AttnArgs a) {
  using Shape = ForwardShape<DP>;
  constexpr int STAGES = Shape::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t smem = smem_addr(smem_raw), bars = smem + Shape::BARS;
  const uint32_t q_full = bars, q_empty = bars + 8, s_full = bars + 16, p_full = bars + 32, o_full = bars + 48, full = bars + 64,
                 empty = full + 8 * STAGES, tmem_word = empty + 8 * STAGES;
  volatile int* dead = reinterpret_cast<volatile int*>(smem_raw + (tmem_word + 4 - smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    bar_init(q_full, LOAD_THREADS);
    bar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(s_full + 8 * i, 1);
      bar_init(p_full + 8 * i, 128);
      bar_init(o_full + 8 * i, 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      bar_init(full + 8 * i, LOAD_THREADS);
      bar_init(empty + 8 * i, 1);
    }
    *dead = 0;
    bar_init_fence();
  }
  if (warp == 0) tmem_alloc_one(tmem_word, TMEM_COLS);
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_word) : "memory");
  pdl_enter();
  const int n_items = min(a.counts[ATTN_N_Q_TILES], a.q_tile_bound);
  const int64_t items = static_cast<int64_t>(n_items) * a.heads;
  const int group = a.heads / a.kv_heads;
  bool ok = true;

  if (warp > SOFTMAX_WARPS) {
    // ---- rows
    fewer_registers<FEW_REGISTERS>();
    if (warp <= SOFTMAX_WARPS + LOAD_WARPS) {  // (the last warp fills the warpgroup)
    const int t = threadIdx.x - (SOFTMAX_WARPS + 1) * 32;
    Ring<STAGES> ring{full, empty};
    int n = 0;  // items with keys so far
    for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int index = static_cast<int>(item / a.heads), head = static_cast<int>(item - static_cast<int64_t>(index) * a.heads);
      const AttnTile x = tile_at(a.q_tiles + index);
      if (x.steps == 0) continue;
      const char* q = static_cast<const char*>(a.q.p) + (x.row * a.q.row + head * a.q.head) * 2;
      const char* k = static_cast<const char*>(a.k.p) + (x.other * a.k.row + (head / group) * a.k.head) * 2;
      const char* v = static_cast<const char*>(a.v.p) + (x.other * a.v.row + (head / group) * a.v.head) * 2;
      if (!(ok = !*dead && bar_wait(q_empty, (n & 1) ^ 1))) break;
      ask_tile<DP>(smem, q, a.q.row * 2, x.rows, a.d, t);
      if (x.rows > ATTN_TILE) ask_tile<DP>(smem + tile_bytes<DP>(), q + ATTN_TILE * a.q.row * 2, a.q.row * 2, x.rows - ATTN_TILE, a.d, t);
      ask_commit();
      // K0, V0, K1, V1, ..
      for (int j = 0; ok && j < 2 * x.steps; ++j) {
        if (!(ok = ring.wait_empty(dead))) break;
        const int at = (j >> 1) * ATTN_TILE;
        const bool key = (j & 1) == 0;
        const AttnView& view = key ? a.k : a.v;
        ask_tile<DP>(smem + Shape::RING + ring.slot() * tile_bytes<DP>(), (key ? k : v) + at * view.row * 2, view.row * 2, x.others - at, a.d, t);
        if (j == 0) {
          ask_commit();
          ++ring.at;
          ask_wait<1>();
          fence_async_smem();
          bar_arrive(q_full);
        } else {
          ring.asked();
        }
      }
      ring.template hand_over<0>();
      ++n;
    }
    ask_wait<0>();
    }
  } else if (warp == SOFTMAX_WARPS) {
    // ---- products
    fewer_registers<FEW_REGISTERS>();
    if (lane == 0) {
      const uint32_t by_rows = mma_desc(BF16, false, false, ATTN_TILE, ATTN_TILE), by_columns = mma_desc(BF16, false, true, ATTN_TILE, DP);
      const uint32_t s[2] = {tmem, tmem + 128}, o[2] = {tmem + 256, tmem + 256 + DP};
      int st = 0, p_at[2] = {0, 0}, n = 0;
      const auto stage = [&](int i) { return smem + Shape::RING + (i % STAGES) * tile_bytes<DP>(); };
      const auto ready = [&](int i) { return !*dead && bar_wait(full + 8 * (i % STAGES), (i / STAGES) & 1); };
      for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const AttnTile x = tile_at(a.q_tiles + item / a.heads);
        if (x.steps == 0) continue;
        const int two = x.rows > ATTN_TILE ? 2 : 1;
        if (!(ok = !*dead && bar_wait(q_full, n & 1) && ready(st))) break;
        fence_after();
        for (int w = 0; w < two; ++w) {
          product_rows<DP>(s[w], smem + w * tile_bytes<DP>(), stage(st), by_rows);
          mma_commit_one(s_full + 8 * w);
        }
        mma_commit_one(empty + 8 * (st % STAGES));
        for (int j = 0; ok && j < x.steps; ++j) {
          const bool more = j + 1 < x.steps;
          if (!(ok = ready(st + 1) && (!more || ready(st + 2)))) break;
          for (int w = 0; w < two; ++w) {
            if (!(ok = !*dead && bar_wait(p_full + 8 * w, p_at[w]++ & 1))) break;
            fence_after();
            product_columns<DP>(o[w], s[w], 32, stage(st + 1), by_columns, j > 0);
            if (more) {
              product_rows<DP>(s[w], smem + w * tile_bytes<DP>(), stage(st + 2), by_rows);
              mma_commit_one(s_full + 8 * w);
            } else {
              mma_commit_one(o_full + 8 * w);
            }
          }
          if (!ok) break;
          mma_commit_one(empty + 8 * ((st + 1) % STAGES));
          if (more) mma_commit_one(empty + 8 * ((st + 2) % STAGES));
          st += 2;
        }
        if (!ok) break;
        mma_commit_one(q_empty);
        ++n;
      }
    }
    __syncwarp();
  } else {
    // ---- exponentials: a row a thread
    more_registers<MANY_REGISTERS>();
    const int w = warp / 4;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t s = tmem + w * 128 + lanes, o = tmem + 256 + w * DP + lanes;
    const int mine = w * ATTN_TILE + warp % 4 * 32 + lane;
    const float c = a.scale * LOG2E;
    // 2^4: weights of 16 bits that are far below a row's largest keep more of their digits
    constexpr float LIFT = BF16 ? 0.0f : 4.0f;
    int at = 0, o_at = 0;
    for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int index = static_cast<int>(item / a.heads), head = static_cast<int>(item - static_cast<int64_t>(index) * a.heads);
      const AttnTile x = tile_at(a.q_tiles + index);
      const bool there = mine < x.rows;
      float l = 0.0f, ref = -INFINITY;
      if (x.steps > 0 && w * ATTN_TILE < x.rows) {
        const int first = a.causal ? x.seen + w * ATTN_TILE : x.others;  // keys that the first row of this tile sees
        const int seen = a.causal ? min(x.others, x.seen + mine) : x.others;
        for (int j = 0; j < x.steps; ++j) {
          if (!(ok = !*dead && bar_wait(s_full + 8 * w, at++ & 1))) break;
          fence_after();
          uint32_t v[4][32];
          const int left = seen - j * ATTN_TILE;
          float top;
          if (first >= (j + 1) * ATTN_TILE && x.others >= (j + 1) * ATTN_TILE) {
            top = scores<false>(s, ATTN_TILE, v);
          } else {
            top = scores<true>(s, left, v);
          }
          top *= c;
          if (__any_sync(FULL_MASK, top > ref + LAZY)) {
            const float next = fmaxf(top, ref), by = next == -INFINITY ? 1.0f : ex2(ref - next);
            ref = next;
            l *= by;
            if (j > 0) {
#pragma unroll
              for (int q = 0; q < DP / 32; ++q) {
                uint32_t r[32];
                tmem_load32(o + q * 32, r);
                tmem_wait(r);
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * by);
                tmem_store32(o + q * 32, r);
              }
            }
          }
          const float base = ref == -INFINITY ? 0.0f : ref - LIFT;
          const uint64_t c2 = two(c, c), base2 = two(-base, -base);
          uint64_t sum = two(0.0f, 0.0f), sum_b = sum;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int q = h * 2 + i / 16, at2 = (i % 16) * 2;
              float lo, hi;
              split2(fma2(two(__uint_as_float(v[q][at2]), __uint_as_float(v[q][at2 + 1])), c2, base2), &lo, &hi);
              lo = ex2(lo);
              hi = ex2(hi);
              if (i & 1) sum_b = add2(sum_b, two(lo, hi));
              else sum = add2(sum, two(lo, hi));
              p[i] = pack2<BF16>(lo, hi);
            }
            tmem_store32(s + h * 32, p);
          }
          float lo, hi;
          split2(add2(sum, sum_b), &lo, &hi);
          l += lo + hi;
          tmem_store_wait();
          fence_before();
          bar_arrive(p_full + 8 * w);
        }
        if (!ok) break;
        if (!(ok = !*dead && bar_wait(o_full + 8 * w, o_at++ & 1))) break;
        fence_after();
      }
      if (w * ATTN_TILE >= x.rows) continue;
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // (nan stays nan)
      char* to = static_cast<char*>(a.out) + ((static_cast<int64_t>(x.row + mine) * a.heads + head) * a.d) * 2;
#pragma unroll
      for (int q = 0; q < DP / 32; ++q) {
        uint32_t r[32];
        if (x.steps > 0) {
          tmem_load32(o + q * 32, r);
          tmem_wait(r);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float lo = __uint_as_float(r[i * 8 + e * 2]) * inv, hi = __uint_as_float(r[i * 8 + e * 2 + 1]) * inv;
            y[e] = l == 0.0f ? 0u : pack2<BF16>(lo, hi);
          }
          if (there && q * 32 + i * 8 < a.d) *reinterpret_cast<uint4*>(to + (q * 32 + i * 8) * 2) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      fence_before();
      if (there) a.lse[static_cast<int64_t>(head) * a.n_q + x.row + mine] = l == 0.0f ? -INFINITY : (ref - LIFT + log2f(l)) * LN2;
    }
  }
  if (!ok) {
    *dead = 1;
    raise_status(a.status, DGS_ERR_CUDA);
  }
  __syncthreads();
  if (*dead) {
    // products still under way land within microseconds; nobody reads them, but they must not outlive the tile memory
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (warp == 0) {
    fence_after();
    tmem_free_one(tmem, TMEM_COLS);
  }
}

template <typename Kernel>
int launch_tiles(Kernel kernel, const AttnArgs& a, int64_t items, uint32_t smem, std::atomic<bool>* known, cudaStream_t s) {
  int dev = 0;
  DGS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= MAX_DEVICES || !known[dev].load(std::memory_order_relaxed)) {
    DGS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    if (dev < MAX_DEVICES) known[dev].store(true, std::memory_order_relaxed);
  }
  const int64_t most = sm_count();
  DGS_CUDA_TRY(launch_training(kernel, dim3(static_cast<unsigned>(items < most ? items : most)), TILE_THREADS, smem, s, a));
  return DGS_OK;
}

template <int DP, bool BF16>
int forward(const AttnArgs& a, cudaStream_t s) {
  static_assert(ForwardShape<DP>::SMEM <= MAX_SMEM, "shared memory");
  static std::atomic<bool> known[MAX_DEVICES] = {};
  return launch_tiles(attn_forward_kernel<DP, BF16>, a, static_cast<int64_t>(a.q_tile_bound) * a.heads, ForwardShape<DP>::SMEM, known, s);
}

}  // namespace

int attn_tiles_forward(const AttnArgs& a, int32_t dtype, cudaStream_t s) {
  if (a.d <= 64) return dtype == DGS_BF16 ? forward<64, true>(a, s) : forward<64, false>(a, s);
  return dtype == DGS_BF16 ? forward<128, true>(a, s) : forward<128, false>(a, s);
}

int attn_tiles_backward(const AttnArgs&, int32_t, cudaStream_t) { return DGS_OK; }

}  // namespace dgs
