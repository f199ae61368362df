// Attention of long sequences in 16 bits on the tensor cores (formulas: attention.cu).
//
// Forward: a CTA takes two tiles of 128 queries (the same rows of two heads that share their keys, or neighbouring rows of one head) and runs
// over the keys 128 at a time.
//   S = Q K^T           both operands out of shared memory, 128 columns of TMEM for each query tile
//   P = exp2(S c - ref) a thread a row: TMEM -> registers -> TMEM, 16 bits, in S's place
//   O += P V            P out of TMEM, V as it lies (its rows are the sum's index), O stays in TMEM for all keys
// While one tile's exponentials run, the tensor cores work on the other's products.  `ref` follows the running maximum of a row only
// when that has grown by more than 2^8 (the sums are in 32 bits and divided in the end), so O is hardly ever rescaled.
// Backward: the gradients of keys and values by tiles of 128 keys, those of the queries by tiles of 128 queries, so every sum is
// made by one CTA in a fixed order, for the price of the scores and of dO V^T computed twice (7 products a pair of tiles, not 5).
//   keys     S^T = K Q^T, P^T = exp2(S^T c - lse), dV += P^T dO;  E^T = V dO^T, dS^T = P^T (E^T - delta), dK += dS^T Q
//   queries  S = Q K^T, E = dO V^T, dQ += dS K
// with P^T, dS^T and dS out of TMEM; S^T's products run while dS^T is made and the other way round.
// Whole tiles travel by TMA.  Where a product's sum runs over a tile's rows, rows behind a sequence's end have to be zeros, not the next
// sequence's: such last tiles come row by row through cp.async.
// Every wait is bounded; a wait that runs out raises DGS_ERR_CUDA in the status word and all roles leave.
// Measured, bfloat16: 4 causal sequences of 8 192 tokens, 16 heads of 128 on 4, forward 1 053 us = 1 044 TFLOP/s, backward 4 310 us = 638 of
// the 5 products that are needed; bound by the exponentials and slopes beside the products.  320 of 100 tokens, 8 heads of 64 on 2: 86 and
// 185 us, bound by launches and half-filled tiles (tensor pipe 17 to 23 % active on ragged lengths).
#include <type_traits>

#include "attention.h"
#include "tensor_core.cuh"

namespace dgs {
namespace {
using namespace tc;

constexpr int SOFTMAX_WARPS = 8, LOAD_WARPS = 2;
constexpr int LOAD_THREADS = LOAD_WARPS * 32;
constexpr int TILE_THREADS = 384;  // three warpgroups: two of a row (or half of one) a thread, one of the products' and the loading warps
// Registers: 3 x 128 x 168 at the launch; the first two take what the third leaves
constexpr int MANY_REGISTERS = 200, FEW_REGISTERS = 104;
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

struct TileArgs {
  AttnArgs a;
  CUtensorMap q, k, v, dout;
};

// ---- rows into shared memory ------------------------------------------------------------------------------------------
// 128 rows of a head (`there` of them exist, the others become zeros), panels of 64 elements, 128-byte swizzle, by the loading threads
template <int DP>
__device__ __forceinline__ void ask_tile(uint32_t dst, const char* p, int64_t row_bytes, int there, int d, int t) {
  constexpr int CHUNKS = DP / 8, ROWS = LOAD_THREADS / CHUNKS;  // 16-byte pieces of a row; rows a pass
  const int c = t % CHUNKS, r0 = t / CHUNKS;
  const bool in_d = c * 8 < d;
  const char* src = p + r0 * row_bytes + c * 16;
  const uint32_t base = dst + (c / 8) * PANEL + r0 * 128;
#pragma unroll 4
  for (int i = 0; i < ATTN_TILE / ROWS; ++i) {
    const int r = r0 + i * ROWS;
    const bool in = in_d && r < there;
    const uint32_t to = base + i * ROWS * 128 + (((c & 7) ^ (r & 7)) << 4);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(in ? src : p), "r"(in ? 16 : 0) : "memory");
    src += ROWS * row_bytes;
  }
}

// What the loading threads do, each of them: a ring of stages filled in order.
template <int DP, int STAGES>
struct Loader {
  uint32_t tiles, full, empty;  // shared memory of the stages, their barriers
  int t;
  Waits wait;
  int at = 0;        // stages filled
  int waiting = 0;   // the newest of them that came by cp.async and are not handed over

  __device__ __forceinline__ void panels(uint32_t dst, const CUtensorMap* map, int32_t head, int32_t row, uint32_t bar) const {
#pragma unroll
    for (int p = 0; p < DP / 64; ++p) load_box_one(dst + p * PANEL, map, p * 64, head, row, bar);
  }
  // a whole tile by TMA; `bar` counts every loading thread
  __device__ __forceinline__ void box(uint32_t dst, const CUtensorMap* map, int32_t head, int32_t row, uint32_t bar) const {
    if (t == 0) {
      bar_expect(bar, tile_bytes<DP>());
      panels(dst, map, head, row, bar);
    } else {
      bar_arrive(bar);
    }
  }
  // two tiles side by side behind one barrier (or the first alone)
  __device__ __forceinline__ void boxes(uint32_t dst, const CUtensorMap* map, int32_t head, int32_t row, const CUtensorMap* map2, int32_t head2,
                                        int32_t row2, bool both, uint32_t bar) const {
    if (t == 0) {
      bar_expect(bar, (both ? 2 : 1) * tile_bytes<DP>());
      panels(dst, map, head, row, bar);
      if (both) panels(dst + tile_bytes<DP>(), map2, head2, row2, bar);
    } else {
      bar_arrive(bar);
    }
  }
  __device__ __forceinline__ bool free_stage() const { return wait(empty + 8 * (at % STAGES), ((at / STAGES) & 1) ^ 1); }
  // the next stage: rows row.. of a head, `there` of them; zeros: whether those behind them must be zeros
  __device__ __forceinline__ void fill(const CUtensorMap* map, const AttnView& view, int32_t head, int32_t row, int there, bool zeros, int d) {
    const uint32_t dst = tiles + (at % STAGES) * tile_bytes<DP>();
    if (there >= ATTN_TILE || !zeros) {
      box(dst, map, head, row, full + 8 * (at % STAGES));
    } else {
      ask_tile<DP>(dst, static_cast<const char*>(view.p) + (row * view.row + head * view.head) * 2, view.row * 2, there, d, t);
      ++waiting;
    }
    ++at;
  }
  // (called with those that wait being the newest stages)
  __device__ __forceinline__ void hand_over() {
    if (waiting == 0) return;
    asm volatile("cp.async.wait_all;" ::: "memory");
    fence_async_smem();
    for (; waiting > 0; --waiting) bar_arrive(full + 8 * ((at - waiting) % STAGES));
  }
};

// ---- products ---------------------------------------------------------------------------------------------------------
// The products' thread: a stage of the ring, ahead of which it may look.
template <int DP, int STAGES>
struct Stage {
  uint32_t tiles, full, empty;
  Waits wait;
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ int slot_of(int ahead) const { return slot + ahead < STAGES ? slot + ahead : slot + ahead - STAGES; }
  __device__ __forceinline__ uint32_t tile(int ahead) const { return tiles + slot_of(ahead) * tile_bytes<DP>(); }
  __device__ __forceinline__ bool ready(int ahead) const {
    return wait(full + 8 * slot_of(ahead), slot + ahead < STAGES ? phase : phase ^ 1);
  }
  __device__ __forceinline__ void release(int ahead) const { mma_commit_one(empty + 8 * slot_of(ahead)); }
  __device__ __forceinline__ void advance(int by) {
    slot += by;
    if (slot >= STAGES) slot -= STAGES, phase ^= 1;
  }
};

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

__device__ __forceinline__ AttnTile tile_at(const AttnTile* p) {
  AttnTile t;
  reinterpret_cast<int4*>(&t)[0] = reinterpret_cast<const int4*>(p)[0];
  reinterpret_cast<int4*>(&t)[1] = reinterpret_cast<const int4*>(p)[1];
  return t;
}
// The items of a CTA: every gridDim.x-th (tile, head), the next tile's words on their way.
struct Items {
  const AttnTile* list;
  int tiles, heads, index, head;
  AttnTile x, next;
  __device__ __forceinline__ Items(const AttnTile* tiles_list, int n_tiles, int n_heads) : list(tiles_list), tiles(n_tiles), heads(n_heads) {
    index = blockIdx.x / heads;
    head = blockIdx.x % heads;
    if (index < tiles) x = tile_at(list + index);
    ask();
  }
  __device__ __forceinline__ bool more() const { return index < tiles; }
  __device__ __forceinline__ void step(int* to_index, int* to_head) const {
    *to_index = index + static_cast<int>(gridDim.x) / heads;
    *to_head = head + static_cast<int>(gridDim.x) % heads;
    if (*to_head >= heads) *to_head -= heads, ++*to_index;
  }
  __device__ __forceinline__ void ask() {
    int i, h;
    step(&i, &h);
    if (i < tiles) next = tile_at(list + i);
  }
  __device__ __forceinline__ void advance() {
    step(&index, &head);
    x = next;
    ask();
  }
};

// a row that the rows' kernels have to make again (ATTN_AGAIN)
__device__ __forceinline__ void leave_row(const AttnArgs& a, int32_t* map, int row) {
  atomicOr(&map[row], ATTN_AGAIN);
  atomicOr(&a.counts[ATTN_KINDS], 1 << ATTN_HAS_AGAIN);
}

// ---- forward ----------------------------------------------------------------------------------------------------------
template <int DP>
struct ForwardShape {
  static constexpr int STAGES = DP == 128 ? 5 : 8;
  static constexpr int QUERIES = DP == 128 ? 1 : 2;  // items whose queries fit: the next one's come while this one is worked on
  static constexpr uint32_t QUERY_BYTES = 2 * tile_bytes<DP>(), RING = QUERIES * QUERY_BYTES, BARS = RING + STAGES * tile_bytes<DP>(), SMEM = BARS + 256;
};

// One tile's 128 scores of a row: read for the largest, read again for the weights, 32 columns at a time with the next 32 on their way
// (held in registers between the two they spill).  `seen`: columns that the row sees (MASK: fewer than 128 may be).
template <bool MASK>
__device__ __forceinline__ float largest(uint32_t s, int seen) {
  uint32_t v[2][32];
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  tmem_load32(s, v[0]);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    tmem_wait(v[q & 1]);
    if (q < 3) tmem_load32(s + (q + 1) * 32, v[(q + 1) & 1]);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float x = __uint_as_float(v[q & 1][i]);
      if (MASK) x = q * 32 + i < seen ? x : -INFINITY;
      top[i & 3] = fmaxf(top[i & 3], x);
    }
  }
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// weights exp2(score c - base) into the scores' place, 16 bits each; returns their sum
template <bool MASK, bool BF16>
__device__ __forceinline__ float weigh(uint32_t s, int seen, float c, float base) {
  const uint64_t c2 = two(c, c), base2 = two(-base, -base);
  uint64_t sum[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
  uint32_t v[2][32];
  tmem_load32(s, v[0]);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    tmem_wait(v[q & 1]);
    if (q < 3) tmem_load32(s + (q + 1) * 32, v[(q + 1) & 1]);
    uint32_t p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float lo, hi;
      split2(fma2(two(__uint_as_float(v[q & 1][2 * i]), __uint_as_float(v[q & 1][2 * i + 1])), c2, base2), &lo, &hi);
      lo = ex2(lo);
      hi = ex2(hi);
      if (MASK) {
        lo = q * 32 + 2 * i < seen ? lo : 0.0f;
        hi = q * 32 + 2 * i + 1 < seen ? hi : 0.0f;
      }
      sum[i & 1] = add2(sum[i & 1], two(lo, hi));
      p[i] = pack2<BF16>(lo, hi);
    }
    tmem_store16(s + q * 16, p);
  }
  float lo, hi;
  split2(add2(sum[0], sum[1]), &lo, &hi);
  return lo + hi;
}

template <int DP, bool BF16>
__global__ __launch_bounds__(TILE_THREADS, 1) void attn_forward_kernel(const __grid_constant__ TileArgs args) {
  using Shape = ForwardShape<DP>;
  constexpr int STAGES = Shape::STAGES;
  const AttnArgs& a = args.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t smem = smem_addr(smem_raw), bars = smem + Shape::BARS;
  constexpr int QUERIES = Shape::QUERIES;
  const uint32_t q_full = bars, q_empty = bars + 16, s_full = bars + 32, p_full = bars + 48, o_full = bars + 64, full = bars + 80,
                 empty = full + 8 * STAGES, tmem_word = empty + 8 * STAGES;
  volatile int* dead = reinterpret_cast<volatile int*>(smem_raw + (tmem_word + 4 - smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(q_full + 8 * i, LOAD_THREADS);
      bar_init(q_empty + 8 * i, 1);
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
  const int group = a.heads / a.kv_heads, heads = a.head_pairs ? a.heads / 2 : a.heads;  // an item is a tile of queries and a head, or two of them
  const int64_t items = static_cast<int64_t>(min(a.counts[ATTN_N_Q_TILES], a.q_tile_bound)) * heads;
  const Waits wait{dead, a.wait_limit};
  bool ok = true;

  if (warp > SOFTMAX_WARPS) {
    // ---- rows
    fewer_registers<FEW_REGISTERS>();
    if (warp <= SOFTMAX_WARPS + LOAD_WARPS) {  // (the last warp fills the warpgroup)
      fence_async_global();  // rows that ordinary stores of an earlier launch wrote
      Loader<DP, STAGES> load{smem + Shape::RING, full, empty, static_cast<int>(threadIdx.x) - (SOFTMAX_WARPS + 1) * 32, wait};
      int n = 0;  // items with keys so far
      for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const int index = static_cast<int>(item / heads), head = static_cast<int>(item - static_cast<int64_t>(index) * heads) << a.head_pairs;
        const AttnTile x = tile_at(a.q_tiles + index);
        if (x.steps == 0) continue;
        const int slot = n % QUERIES;
        if (!(ok = wait(q_empty + 8 * slot, ((n / QUERIES) & 1) ^ 1))) break;
        load.boxes(smem + slot * Shape::QUERY_BYTES, &args.q, head, x.row, &args.q, head + a.head_pairs, a.head_pairs ? x.row : x.row + ATTN_TILE,
                   a.head_pairs || x.rows > ATTN_TILE, q_full + 8 * slot);
        // K0, V0, K1, V1, ..  (only V's rows are summed over)
        for (int j = 0; ok && j < x.steps; ++j) {
          const int at = j * ATTN_TILE;
          if (!(ok = load.free_stage())) break;
          load.fill(&args.k, a.k, head / group, x.other + at, x.others - at, false, a.d);
          if (!(ok = load.free_stage())) break;
          load.fill(&args.v, a.v, head / group, x.other + at, x.others - at, true, a.d);
        }
        load.hand_over();
        ++n;
      }
    }
  } else if (warp == SOFTMAX_WARPS) {
    // ---- products
    fewer_registers<FEW_REGISTERS>();
    if (lane == 0) {
      const uint32_t by_rows = mma_desc(BF16, false, false, ATTN_TILE, ATTN_TILE), by_columns = mma_desc(BF16, false, true, ATTN_TILE, DP);
      Stage<DP, STAGES> st{smem + Shape::RING, full, empty, wait};
      uint32_t p_phase[2] = {0, 0};
      int n = 0;
      // O += P V of the tile of queries w, then S of the next keys
      const auto step = [&](auto which, uint32_t q, bool first, bool more) {
        constexpr uint32_t w = decltype(which)::value;
        const uint32_t s = tmem + w * 128;
        if (!wait(p_full + 8 * w, p_phase[w])) return false;
        p_phase[w] ^= 1;
        fence_after();
        product_columns<DP>(tmem + 256 + w * DP, s, 32, st.tile(1), by_columns, !first);
        if (more) {
          product_rows<DP>(s, q + w * tile_bytes<DP>(), st.tile(2), by_rows);
          mma_commit_one(s_full + 8 * w);
        } else {
          mma_commit_one(o_full + 8 * w);
        }
        return true;
      };
      using One = std::integral_constant<uint32_t, 0>;
      using Two = std::integral_constant<uint32_t, 1>;
      for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
        const AttnTile x = tile_at(a.q_tiles + item / heads);
        if (x.steps == 0) continue;
        const bool two = a.head_pairs || x.rows > ATTN_TILE;
        const int slot = n % QUERIES;
        const uint32_t q = smem + slot * Shape::QUERY_BYTES;
        if (!(ok = wait(q_full + 8 * slot, (n / QUERIES) & 1) && st.ready(0))) break;
        fence_after();
        product_rows<DP>(tmem, q, st.tile(0), by_rows);
        mma_commit_one(s_full);
        if (two) {
          product_rows<DP>(tmem + 128, q + tile_bytes<DP>(), st.tile(0), by_rows);
          mma_commit_one(s_full + 8);
        }
        st.release(0);
        for (int j = 0; ok && j < x.steps; ++j) {
          const bool more = j + 1 < x.steps;
          if (!(ok = st.ready(1) && (!more || st.ready(2)))) break;
          if (!(ok = step(One{}, q, j == 0, more) && (!two || step(Two{}, q, j == 0, more)))) break;
          st.release(1);
          if (more) st.release(2);
          st.advance(2);
        }
        if (!ok) break;
        mma_commit_one(q_empty + 8 * slot);
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
    const int below = a.head_pairs ? 0 : w * ATTN_TILE, mine = below + warp % 4 * 32 + lane;  // rows of the item in front of this tile
    const float c = a.scale * LOG2E;
    // 2^4: weights of 16 bits that are far below a row's largest keep more of their digits
    constexpr float LIFT = BF16 ? 0.0f : 4.0f;
    int at = 0, o_at = 0;
    for (int64_t item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int index = static_cast<int>(item / heads);
      const int head = (static_cast<int>(item - static_cast<int64_t>(index) * heads) << a.head_pairs) + (a.head_pairs ? w : 0);
      const AttnTile x = tile_at(a.q_tiles + index);
      const bool there = mine < x.rows;
      float l = 0.0f, ref = -INFINITY;
      if (x.steps > 0 && below < x.rows) {
        const int first = a.causal ? x.seen + below : x.others;  // keys that the first row of this tile sees
        const int seen = a.causal ? min(x.others, x.seen + mine) : x.others;
        for (int j = 0; j < x.steps; ++j) {
          if (!(ok = wait.warp(s_full + 8 * w, at++ & 1))) break;
          fence_after();
          const int left = seen - j * ATTN_TILE;
          const bool whole = first >= (j + 1) * ATTN_TILE && x.others >= (j + 1) * ATTN_TILE;
          const float top = c * (whole ? largest<false>(s, ATTN_TILE) : largest<true>(s, left));
          // (rows behind the sequence's end, which may hold anything, have no say in how those of the sequence are rounded)
          if (__any_sync(FULL_MASK, there && top > ref + LAZY)) {
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
          l += whole ? weigh<false, BF16>(s, ATTN_TILE, c, base) : weigh<true, BF16>(s, left, c, base);
          tmem_store_wait();
          fence_before();
          bar_arrive(p_full + 8 * w);
        }
        if (!ok) break;
        if (!(ok = wait.warp(o_full + 8 * w, o_at++ & 1))) break;
        fence_after();
      }
      if (below >= x.rows) continue;
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // (nan stays nan)
      char* to = static_cast<char*>(a.out) + ((static_cast<int64_t>(x.row + mine) * a.heads + head) * a.d) * 2;
      bool nan = false;
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
            nan |= lo != lo || hi != hi;
          }
          if (there && q * 32 + i * 8 < a.d) *reinterpret_cast<uint4*>(to + (q * 32 + i * 8) * 2) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      fence_before();
      // (a sum of the weights that is not a number: neither is the row, by its own scores)
      if (a.causal && there && nan && l > 0.0f) leave_row(a, a.q_seq, x.row + mine);
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

// ---- backward -----------------------------------------------------------------------------------------------------------
// fp16 keeps few powers of two: weights are lifted by 2^12 and dS scaled so that its bound becomes 2^15 at the most.  |e| is at most B,
// the largest |do_i| times the largest |v_j|, and |p (e - delta)| = p (1 - p) |e - the others' mean| at most B / 2.
template <bool BF16>
constexpr float lift() {
  return BF16 ? 0.0f : 12.0f;
}
template <bool BF16>
__device__ __forceinline__ float slope_scale(const AttnArgs& a) {
  if constexpr (BF16) return 1.0f;
  const float b = a.norms[0] * a.norms[1];
  if (!(b > 0.0f)) return 1.0f / 4096.0f;
  int e;
  frexpf(b, &e);
  return ldexpf(1.0f, max(-100, min(100, 4 - e)));
}

constexpr int DELTA_THREADS = 256;

// the sequence of a row is one of the tiles'
__device__ __forceinline__ bool in_a_tile(const AttnArgs& a, const int32_t* map, int row, bool key) {
  const int s = map[row] & ~ATTN_AGAIN;
  if (s >= a.seqs) return false;
  const AttnSeq e = a.seq[s];
  const int at = row - (key ? e.k0 : e.q0);
  return at >= 0 && at < (key ? e.k_len : e.q_len) && attn_in_tiles(a, e);
}
// the largest of a CTA's values, into a word of which values are ordered as unsigned words
__device__ __forceinline__ void largest_of_cta(float v, float* to) {
  __shared__ unsigned top;
  if (threadIdx.x == 0) top = 0;
  __syncthreads();
  const unsigned w = __reduce_max_sync(FULL_MASK, __float_as_uint(v));
  if ((threadIdx.x & 31) == 0 && w != 0) atomicMax(&top, w);
  __syncthreads();
  if (threadIdx.x == 0 && top != 0) atomicMax(reinterpret_cast<unsigned*>(to), top);
}

// The norm of a row for the bound of the slopes.  A row that is not finite has none: its own gradients are not numbers whatever the scale, and
// the other sequences of the call keep theirs (squares of float16 numbers are far from the largest of 32 bits).
__device__ __forceinline__ float finite_norm(float square) { return square < INFINITY ? sqrtf(square) : 0.0f; }

// Rows of the tiles' sequences: delta = do.o, lse in powers of two (less the lift), the largest norm of do.  A warp looks eight rows up side by
// side and takes each of them with all its heads, LANES lanes a head.
constexpr int DELTA_ROWS = 8;
template <typename T, int LANES>
__global__ __launch_bounds__(DELTA_THREADS, 4) void attn_delta_kernel(const __grid_constant__ AttnArgs a, float down, int32_t norm) {
  pdl_enter();
  if ((a.counts[ATTN_KINDS] >> ATTN_HAS_TILES & 1) == 0) return;
  const int lane = threadIdx.x & 31, vec = lane % LANES, warps = gridDim.x * (DELTA_THREADS / 32);
  constexpr int SIDE = 32 / LANES;
  float top = 0.0f;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x * (DELTA_THREADS / 32) + threadIdx.x / 32) * DELTA_ROWS; row0 < a.n_q;
       row0 += static_cast<int64_t>(warps) * DELTA_ROWS) {
    const bool mine = lane < DELTA_ROWS && row0 + lane < a.n_q && in_a_tile(a, a.q_seq, static_cast<int>(row0) + lane, false);
    for (unsigned todo = __ballot_sync(FULL_MASK, mine); todo != 0; todo &= todo - 1) {
      const int row = static_cast<int>(row0) + __ffs(todo) - 1;
#pragma unroll 2
      for (int h0 = 0; h0 < a.heads; h0 += SIDE) {
        const int head = h0 + lane / LANES;
        const bool in = head < a.heads;
        float sum = 0.0f, square = 0.0f;
        if (in && vec * 8 < a.d) {
          float x[8], y[8];
          load_vec<T, 8>(static_cast<const T*>(a.dout.p) + row * a.dout.row + head * a.dout.head + vec * 8, x);
          load_vec<T, 8>(static_cast<const T*>(a.out) + (static_cast<int64_t>(row) * a.heads + head) * a.d + vec * 8, y);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sum = fmaf(x[i], y[i], sum);
            square = fmaf(x[i], x[i], square);
          }
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
          sum += __shfl_xor_sync(FULL_MASK, sum, o);
          square += __shfl_xor_sync(FULL_MASK, square, o);
        }
        if (in && vec == 0) {
          const int64_t at = static_cast<int64_t>(head) * a.n_q + row;
          const float lse = a.lse[at];
          a.delta[at] = sum;
          a.lse2[at] = lse == -INFINITY ? INFINITY : lse * LOG2E - down;  // (a row that sees no key has no weights)
          top = fmaxf(top, finite_norm(square));
        }
      }
    }
  }
  if (norm) largest_of_cta(top, a.norms);
}

// the largest norm of v over all rows of the tiles' sequences
template <typename T>
__global__ __launch_bounds__(DELTA_THREADS) void attn_norm_kernel(const __grid_constant__ AttnArgs a) {
  pdl_enter();
  if ((a.counts[ATTN_KINDS] >> ATTN_HAS_TILES & 1) == 0) return;
  const int lane = threadIdx.x % 16, head = blockIdx.y;
  float top = 0.0f;
  for (int row0 = blockIdx.x * (DELTA_THREADS / 16); row0 < a.n_k; row0 += gridDim.x * (DELTA_THREADS / 16)) {
    const int row = row0 + threadIdx.x / 16;
    float square = 0.0f;
    if (row < a.n_k && lane * 8 < a.d && in_a_tile(a, a.k_seq, row, true)) {
      float x[8];
      load_vec<T, 8>(static_cast<const T*>(a.v.p) + row * a.v.row + head * a.v.head + lane * 8, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) square = fmaf(x[i], x[i], square);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) square += __shfl_xor_sync(FULL_MASK, square, o);
    top = fmaxf(top, finite_norm(square));
  }
  largest_of_cta(top, a.norms + 1);
}

template <int DP>
struct BackwardShape {
  static constexpr int STAGES = DP == 128 ? 5 : 8;
  static constexpr int ITEMS = DP == 128 ? 1 : 2;  // items whose own tiles fit: the next one's come while this one is worked on
  static constexpr uint32_t OWN_BYTES = 2 * tile_bytes<DP>(), RING = ITEMS * OWN_BYTES, STATS = RING + STAGES * tile_bytes<DP>(),
                            BARS = STATS + 2 * 2 * ATTN_TILE * 4, SMEM = BARS + 256;
};

// a row of DP values out of TMEM, times `by`, into contiguous rows of d elements; whether one of them is not a number
template <int FROM, int TO, bool BF16>
__device__ __forceinline__ bool store_row(uint32_t tmem, bool there, float by, char* to, int d) {
  bool nan = false;
#pragma unroll
  for (int q = FROM / 32; q < TO / 32; ++q) {
    uint32_t r[32];
    tmem_load32(tmem + q * 32, r);
    tmem_wait(r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = __uint_as_float(r[i * 8 + e * 2]) * by, hi = __uint_as_float(r[i * 8 + e * 2 + 1]) * by;
        y[e] = pack2<BF16>(lo, hi);
        nan |= lo != lo || hi != hi;
      }
      if (there && q * 32 + i * 8 < d) *reinterpret_cast<uint4*>(to + (q * 32 + i * 8) * 2) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
  return nan;
}
template <int FROM, int TO>
__device__ __forceinline__ void store_zeros(bool there, char* to, int d) {
#pragma unroll
  for (int i = FROM / 8; i < TO / 8; ++i)
    if (there && i * 8 < d) *reinterpret_cast<uint4*>(to + i * 16) = make_uint4(0, 0, 0, 0);
}

// dK and dV of 128 keys of one key head, over the queries of all heads of its group
template <int DP, bool BF16>
__global__ __launch_bounds__(TILE_THREADS, 1) void attn_dkv_kernel(const __grid_constant__ TileArgs args) {
  using Shape = BackwardShape<DP>;
  constexpr int STAGES = Shape::STAGES;
  const AttnArgs& a = args.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t smem = smem_addr(smem_raw), bars = smem + Shape::BARS;
  constexpr int ITEMS = Shape::ITEMS;
  const uint32_t kv_full = bars, kv_empty = bars + 16, s_full = bars + 32, e_full = bars + 40, p_full = bars + 48, ds_full = bars + 56,
                 done = bars + 64, stats_full = bars + 72, stats_empty = bars + 88, full = bars + 104, empty = full + 8 * STAGES,
                 tmem_word = empty + 8 * STAGES;
  volatile int* dead = reinterpret_cast<volatile int*>(smem_raw + (tmem_word + 4 - smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    bar_init(s_full, 1);
    bar_init(e_full, 1);
    bar_init(p_full, SOFTMAX_WARPS * 32);
    bar_init(ds_full, SOFTMAX_WARPS * 32);
    bar_init(done, 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(kv_full + 8 * i, LOAD_THREADS);
      bar_init(kv_empty + 8 * i, 1);
      bar_init(stats_full + 8 * i, LOAD_THREADS);
      bar_init(stats_empty + 8 * i, SOFTMAX_WARPS * 32);
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
  Items items(a.k_tiles, min(a.counts[ATTN_N_K_TILES], a.k_tile_bound), a.kv_heads);
  const int group = a.heads / a.kv_heads;
  const Waits wait{dead, a.wait_limit};
  bool ok = true;

  if (warp > SOFTMAX_WARPS) {
    // ---- rows
    fewer_registers<FEW_REGISTERS>();
    if (warp <= SOFTMAX_WARPS + LOAD_WARPS) {
      fence_async_global();
      const int t = static_cast<int>(threadIdx.x) - (SOFTMAX_WARPS + 1) * 32;
      Loader<DP, STAGES> load{smem + Shape::RING, full, empty, t, wait};
      int n = 0, step = 0;
      for (; ok && items.more(); items.advance()) {
        const int kv = items.head;
        const AttnTile& x = items.x;
        if (x.steps == 0) continue;
        const int own = n % ITEMS;
        if (!(ok = wait(kv_empty + 8 * own, ((n / ITEMS) & 1) ^ 1))) break;
        load.boxes(smem + own * Shape::OWN_BYTES, &args.k, kv, x.row, &args.v, kv, x.row, true, kv_full + 8 * own);
        for (int u = 0; ok && u < x.steps * group; ++u, ++step) {
          const int head = kv * group + u / x.steps, at = u % x.steps * ATTN_TILE, row = x.other + at, left = x.others - at;
          if (!(ok = load.free_stage())) break;
          load.fill(&args.q, a.q, head, row, left, true, a.d);
          const int slot = step & 1;
          if (!(ok = wait(stats_empty + 8 * slot, ((step >> 1) & 1) ^ 1))) break;
          const uint32_t to = smem + Shape::STATS + slot * 2 * ATTN_TILE * 4;
          const int64_t from = static_cast<int64_t>(head) * a.n_q + row;
#pragma unroll
          for (int i = 0; i < ATTN_TILE / LOAD_THREADS; ++i) {
            const int c = t + i * LOAD_THREADS;
            const int64_t src = from + (c < left ? c : 0);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + c * 4), "l"(a.lse2 + src), "r"(c < left ? 4 : 0) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + (ATTN_TILE + c) * 4), "l"(a.delta + src),
                         "r"(c < left ? 4 : 0)
                         : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(stats_full + 8 * slot) : "memory");
          if (!(ok = load.free_stage())) break;
          load.fill(&args.dout, a.dout, head, row, left, true, a.d);
          load.hand_over();
        }
        ++n;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else if (warp == SOFTMAX_WARPS) {
    // ---- products
    fewer_registers<FEW_REGISTERS>();
    if (lane == 0) {
      const uint32_t by_rows = mma_desc(BF16, false, false, ATTN_TILE, ATTN_TILE), by_columns = mma_desc(BF16, false, true, ATTN_TILE, DP);
      const uint32_t s = tmem, e = tmem + 128, dv = tmem + 256, dk = tmem + 256 + DP;
      Stage<DP, STAGES> st{smem + Shape::RING, full, empty, wait};
      int n = 0;
      uint32_t at = 0;
      for (; ok && items.more(); items.advance()) {
        const AttnTile& x = items.x;
        if (x.steps == 0) continue;
        const int own = n % ITEMS;
        const uint32_t k = smem + own * Shape::OWN_BYTES, v = k + tile_bytes<DP>();
        if (!(ok = wait(kv_full + 8 * own, (n / ITEMS) & 1) && st.ready(0))) break;
        fence_after();
        product_rows<DP>(s, k, st.tile(0), by_rows);
        mma_commit_one(s_full);
        if (!(ok = st.ready(1))) break;
        product_rows<DP>(e, v, st.tile(1), by_rows);
        mma_commit_one(e_full);
        const int steps = x.steps * group;
        for (int u = 0; ok && u < steps; ++u, at ^= 1) {
          const bool more = u + 1 < steps;
          if (!(ok = (!more || st.ready(2)) && wait(p_full, at))) break;
          fence_after();
          product_columns<DP>(dv, s, 64, st.tile(1), by_columns, u > 0);
          if (more) {
            product_rows<DP>(s, k, st.tile(2), by_rows);
            mma_commit_one(s_full);
          }
          st.release(1);
          if (!(ok = (!more || st.ready(3)) && wait(ds_full, at))) break;
          fence_after();
          product_columns<DP>(dk, e, 64, st.tile(0), by_columns, u > 0);
          if (more) {
            product_rows<DP>(e, v, st.tile(3), by_rows);
            mma_commit_one(e_full);
          }
          st.release(0);
          st.advance(2);
        }
        if (!ok) break;
        mma_commit_one(done);
        mma_commit_one(kv_empty + 8 * own);
        ++n;
      }
    }
    __syncwarp();
  } else {
    // ---- weights and slopes: a key a thread, half of the queries a warpgroup
    more_registers<MANY_REGISTERS>();
    const int half = warp / 4, mine = warp % 4 * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t s = tmem + half * 64 + lanes, e = tmem + 128 + half * 64 + lanes;
    const float c = a.scale * LOG2E, by = slope_scale<BF16>(a);
    int at = 0, items_done = 0;
    for (; ok && items.more(); items.advance()) {
      const int kv = items.head;
      const AttnTile& x = items.x;
      const bool there = mine < x.rows;
      char* to = static_cast<char*>(half ? a.dk : a.dv) + (static_cast<int64_t>(x.row + mine) * a.kv_heads + kv) * a.d * 2;
      if (x.steps == 0) {
        store_zeros<0, DP>(there, to, a.d);
        continue;
      }
      for (int u = 0; u < x.steps * group; ++u, ++at) {
        const int slot = at & 1, q0 = u % x.steps * ATTN_TILE + half * 64;
        const float4* stats = reinterpret_cast<const float4*>(smem_raw + Shape::STATS + slot * 2 * ATTN_TILE * 4 + half * 64 * 4);
        if (!(ok = wait.warp(stats_full + 8 * slot, (at >> 1) & 1) && wait.warp(s_full, at & 1))) break;
        fence_after();
        uint32_t r[2][32];
        float p[64];
        tmem_load32(s, r[0]);
        tmem_load32(s + 32, r[1]);
        tmem_wait(r[0]);
        tmem_wait(r[1]);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          const float4 lse = stats[i / 4];
          p[i] = ex2(fmaf(__uint_as_float(r[i / 32][i % 32]), c, -lse.x));
          p[i + 1] = ex2(fmaf(__uint_as_float(r[i / 32][i % 32 + 1]), c, -lse.y));
          p[i + 2] = ex2(fmaf(__uint_as_float(r[i / 32][i % 32 + 2]), c, -lse.z));
          p[i + 3] = ex2(fmaf(__uint_as_float(r[i / 32][i % 32 + 3]), c, -lse.w));
        }
        if (x.seen + ATTN_TILE - 1 > q0) {  // (some key of the tile is behind some query)
#pragma unroll
          for (int i = 0; i < 64; ++i) p[i] = mine + x.seen <= q0 + i ? p[i] : 0.0f;
        }
        uint32_t y[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = pack2<BF16>(p[2 * i], p[2 * i + 1]);
        tmem_store32(s, y);
        tmem_store_wait();
        fence_before();
        bar_arrive(p_full);
        if (!(ok = wait.warp(e_full, at & 1))) break;
        fence_after();
        tmem_load32(e, r[0]);
        tmem_load32(e + 32, r[1]);
        tmem_wait(r[0]);
        tmem_wait(r[1]);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          const float4 delta = stats[ATTN_TILE / 4 + i / 4];
          const float d0 = p[i] * by * (__uint_as_float(r[i / 32][i % 32]) - delta.x);
          const float d1 = p[i + 1] * by * (__uint_as_float(r[i / 32][i % 32 + 1]) - delta.y);
          const float d2 = p[i + 2] * by * (__uint_as_float(r[i / 32][i % 32 + 2]) - delta.z);
          const float d3 = p[i + 3] * by * (__uint_as_float(r[i / 32][i % 32 + 3]) - delta.w);
          y[i / 2] = pack2<BF16>(d0, d1);
          y[i / 2 + 1] = pack2<BF16>(d2, d3);
        }
        tmem_store32(e, y);
        tmem_store_wait();
        fence_before();
        bar_arrive(stats_empty + 8 * slot);
        bar_arrive(ds_full);
      }
      if (!ok) break;
      if (!(ok = wait.warp(done, items_done++ & 1))) break;
      fence_after();
      const float last = half ? a.scale / (by * exp2f(lift<BF16>())) : exp2f(-lift<BF16>());
      const bool nan = store_row<0, DP, BF16>(tmem + 256 + half * DP + lanes, there, last, to, a.d);
      if (a.causal && there && nan) leave_row(a, a.k_seq, x.row + mine);
      fence_before();
    }
  }
  if (!ok) {
    *dead = 1;
    raise_status(a.status, DGS_ERR_CUDA);
  }
  __syncthreads();
  if (*dead)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  if (warp == 0) {
    fence_after();
    tmem_free_one(tmem, TMEM_COLS);
  }
}

// dQ of 128 queries of one head.  A query that sees a tile's keys at the most has delta = sum_j p_j e_j of values that its two threads hold
// anyway, in 32 bits, and leaves it for the gradients of the keys, which follow.  Errors of dq and dk, causal, against rounding the exact ones:
// 40 tokens 1.57 -> 1.41 times, 100 tokens 1.51 -> 1.41 (what is left is the rounding of dS to 16 bits, which its products ask for).  A query
// over more keys has delta = do.o from `out` as it is stored: both products and the exponentials twice would be the price of the other (7 products
// a pair of tiles -> 9).  Its rounding goes with the size of out: 1.45 times for v and do around 0, whatever the keys, but with a mean of 1 in both (of
// 3) dq is off by 2.3 (5.7) times over 200 keys, 3.2 (7.8) over 1 000, dk by 1.6 (2.9) and 1.3 (1.7).
__device__ __forceinline__ int first_seen(const AttnArgs& a, const AttnTile& x) { return a.causal ? min(x.seen, x.others) : x.others; }
// (without dq: only what the deltas need, so that the gradients of the keys are the same bits whether dq is wanted or not)
__device__ __forceinline__ int query_steps(const AttnArgs& a, const AttnTile& x) {
  return a.dq != nullptr ? x.steps : first_seen(a, x) <= ATTN_TILE ? min(x.steps, 1) : 0;
}
template <int DP, bool BF16>
__global__ __launch_bounds__(TILE_THREADS, 1) void attn_dq_kernel(const __grid_constant__ TileArgs args) {
  using Shape = BackwardShape<DP>;
  constexpr int STAGES = Shape::STAGES;
  const AttnArgs& a = args.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t smem = smem_addr(smem_raw), bars = smem + Shape::BARS;
  constexpr int ITEMS = Shape::ITEMS;
  const uint32_t q_full = bars, q_empty = bars + 16, s_full = bars + 32, e_full = bars + 48, e_read = bars + 56, ds_full = bars + 64,
                 done = bars + 80, full = bars + 88, empty = full + 8 * STAGES, tmem_word = empty + 8 * STAGES,
                 near_full = bars + 224;
  static_assert(88 + 16 * STAGES + 8 <= 224, "barriers");
  volatile int* dead = reinterpret_cast<volatile int*>(smem_raw + (tmem_word + 4 - smem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(q_full + 8 * i, LOAD_THREADS);
      bar_init(q_empty + 8 * i, 1);
      bar_init(s_full + 8 * i, 1);
    }
    bar_init(e_full, 1);
    bar_init(e_read, SOFTMAX_WARPS * 32);
    // (two: the slopes of a step may be there before the products' thread has looked for those of the step before)
    bar_init(ds_full, SOFTMAX_WARPS * 32);
    bar_init(ds_full + 8, SOFTMAX_WARPS * 32);
    bar_init(done, 1);
    bar_init(near_full, SOFTMAX_WARPS * 32);
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
  Items items(a.q_tiles, min(a.counts[ATTN_N_Q_TILES], a.q_tile_bound), a.heads);
  const int group = a.heads / a.kv_heads;
  const Waits wait{dead, a.wait_limit};
  bool ok = true;

  if (warp > SOFTMAX_WARPS) {
    // ---- rows
    fewer_registers<FEW_REGISTERS>();
    if (warp <= SOFTMAX_WARPS + LOAD_WARPS) {
      fence_async_global();
      Loader<DP, STAGES> load{smem + Shape::RING, full, empty, static_cast<int>(threadIdx.x) - (SOFTMAX_WARPS + 1) * 32, wait};
      int n = 0;
      for (; ok && items.more(); items.advance()) {
        const int head = items.head;
        const AttnTile& x = items.x;
        const int steps = query_steps(a, x);
        if (steps == 0) continue;
        const int own = n % ITEMS;
        if (!(ok = wait(q_empty + 8 * own, ((n / ITEMS) & 1) ^ 1))) break;
        load.boxes(smem + own * Shape::OWN_BYTES, &args.q, head, x.row, &args.dout, head, x.row, true, q_full + 8 * own);
        // K0, V0, K1, V1, ..  (K's rows are summed over)
        for (int j = 0; ok && j < steps; ++j) {
          const int at = j * ATTN_TILE;
          if (!(ok = load.free_stage())) break;
          load.fill(&args.k, a.k, head / group, x.other + at, x.others - at, true, a.d);
          load.hand_over();
          if (!(ok = load.free_stage())) break;
          load.fill(&args.v, a.v, head / group, x.other + at, x.others - at, false, a.d);
        }
        ++n;
      }
    }
  } else if (warp == SOFTMAX_WARPS) {
    // ---- products
    fewer_registers<FEW_REGISTERS>();
    if (lane == 0) {
      const uint32_t by_rows = mma_desc(BF16, false, false, ATTN_TILE, ATTN_TILE), by_columns = mma_desc(BF16, false, true, ATTN_TILE, DP);
      const uint32_t e = tmem + 256, dq = tmem + 384;
      Stage<DP, STAGES> st{smem + Shape::RING, full, empty, wait};
      int n = 0;
      uint32_t at = 0;
      for (; ok && items.more(); items.advance()) {
        const AttnTile& x = items.x;
        const int steps = query_steps(a, x);
        if (steps == 0) continue;
        const int own = n % ITEMS;
        const uint32_t q = smem + own * Shape::OWN_BYTES, g = q + tile_bytes<DP>();
        if (!(ok = wait(q_full + 8 * own, (n / ITEMS) & 1) && st.ready(0))) break;
        fence_after();
        product_rows<DP>(tmem + (at & 1) * 128, q, st.tile(0), by_rows);
        mma_commit_one(s_full + 8 * (at & 1));
        if (!(ok = st.ready(1))) break;
        product_rows<DP>(e, g, st.tile(1), by_rows);
        mma_commit_one(e_full);
        st.release(1);
        for (int j = 0; ok && j < steps; ++j, ++at) {
          if (j + 1 < steps) {
            if (!(ok = st.ready(2))) break;
            product_rows<DP>(tmem + ((at + 1) & 1) * 128, q, st.tile(2), by_rows);
            mma_commit_one(s_full + 8 * ((at + 1) & 1));
            if (!(ok = st.ready(3) && wait(e_read, at & 1))) break;
            fence_after();
            product_rows<DP>(e, g, st.tile(3), by_rows);
            mma_commit_one(e_full);
            st.release(3);
          }
          if (!(ok = wait(ds_full + 8 * (at & 1), (at >> 1) & 1))) break;
          fence_after();
          product_columns<DP>(dq, tmem + (at & 1) * 128, 64, st.tile(0), by_columns, j > 0);
          st.release(0);
          st.advance(2);
        }
        if (!ok) break;
        mma_commit_one(done);
        mma_commit_one(q_empty + 8 * own);
        ++n;
      }
    }
    __syncwarp();
  } else {
    // ---- slopes: a query a thread, half of the keys a warpgroup
    more_registers<MANY_REGISTERS>();
    const int half = warp / 4, mine = warp % 4 * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t e = tmem + 256 + half * 64 + lanes;
    const float c = a.scale * LOG2E, by = slope_scale<BF16>(a);
    int at = 0, items_done = 0, joined = 0;
    float* near = reinterpret_cast<float*>(smem_raw + Shape::STATS);  // [2 in turn][half][query]
    for (; ok && items.more(); items.advance()) {
      const int head = items.head;
      const AttnTile& x = items.x;
      const bool there = mine < x.rows;
      char* to = static_cast<char*>(a.dq) + (static_cast<int64_t>(x.row + mine) * a.heads + head) * a.d * 2;
      const int steps = query_steps(a, x);
      if (steps == 0) {
        if (a.dq == nullptr) continue;
        if (half) store_zeros<DP / 2, DP>(there, to, a.d);
        else store_zeros<0, DP / 2>(there, to, a.d);
        continue;
      }
      const int64_t stat = static_cast<int64_t>(head) * a.n_q + x.row + mine;
      const float lse = there ? a.lse2[stat] : INFINITY;
      float delta = there ? a.delta[stat] : 0.0f;
      const int seen = a.causal ? min(x.others, x.seen + mine) : x.others, first = first_seen(a, x);
      for (int j = 0; j < steps; ++j, ++at) {
        const uint32_t s = tmem + (at & 1) * 128 + half * 64 + lanes;
        if (!(ok = wait.warp(s_full + 8 * (at & 1), (at >> 1) & 1))) break;
        fence_after();
        uint32_t r[2][32];
        float p[64];
        tmem_load32(s, r[0]);
        tmem_load32(s + 32, r[1]);
        tmem_wait(r[0]);
        tmem_wait(r[1]);
#pragma unroll
        for (int i = 0; i < 64; ++i) p[i] = ex2(fmaf(__uint_as_float(r[i / 32][i % 32]), c, -lse));
        if (!(ok = wait.warp(e_full, at & 1))) break;
        fence_after();
        tmem_load32(e, r[0]);
        tmem_load32(e + 32, r[1]);
        tmem_wait(r[0]);
        tmem_wait(r[1]);
        fence_before();
        bar_arrive(e_read);
        const int left = seen - j * ATTN_TILE - half * 64;
        if (j == 0 && first <= ATTN_TILE) {
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 64; ++i) sum = i < left ? fmaf(p[i], __uint_as_float(r[i / 32][i % 32]), sum) : sum;
          // (a slot is written again two joins later, behind the other half's arrival of the join between, which follows its reading)
          float* slot = near + (joined & 1) * 2 * ATTN_TILE;
          slot[half * ATTN_TILE + mine] = sum;
          bar_arrive(near_full);
          if (!(ok = wait.warp(near_full, joined++ & 1))) break;
          if (seen <= ATTN_TILE) {
            delta = (slot[mine] + slot[ATTN_TILE + mine]) * exp2f(-lift<BF16>());
            if (half == 0 && there) a.delta[stat] = delta;
          }
        }
        uint32_t y[32];
#pragma unroll
        for (int i = 0; i < 64; ++i) p[i] = p[i] * by * (__uint_as_float(r[i / 32][i % 32]) - delta);
        if (first < (j + 1) * ATTN_TILE) {  // (what lies behind the keys that are seen may be anything)
#pragma unroll
          for (int i = 0; i < 64; ++i) p[i] = i < left ? p[i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = pack2<BF16>(p[2 * i], p[2 * i + 1]);
        tmem_store32(s, y);
        tmem_store_wait();
        fence_before();
        bar_arrive(ds_full + 8 * (at & 1));
      }
      if (!ok) break;
      if (!(ok = wait.warp(done, items_done++ & 1))) break;
      fence_after();
      const float last = a.scale / (by * exp2f(lift<BF16>()));
      const bool wanted = there && a.dq != nullptr;
      const bool nan = half ? store_row<DP / 2, DP, BF16>(tmem + 384 + lanes, wanted, last, to, a.d)
                            : store_row<0, DP / 2, BF16>(tmem + 384 + lanes, wanted, last, to, a.d);
      // (a delta or lse that is not a number: neither is the row, if it sees a key)
      if (a.causal && wanted && nan && !(seen > 0 && (delta != delta || lse != lse))) leave_row(a, a.q_seq, x.row + mine);
      fence_before();
    }
  }
  if (!ok) {
    *dead = 1;
    raise_status(a.status, DGS_ERR_CUDA);
  }
  __syncthreads();
  if (*dead)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  if (warp == 0) {
    fence_after();
    tmem_free_one(tmem, TMEM_COLS);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
template <typename Kernel>
int launch_tiles(Kernel kernel, const TileArgs& args, int64_t items, uint32_t smem, std::atomic<bool>* known, cudaStream_t s) {
  int dev = 0;
  DGS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= MAX_DEVICES || !known[dev].load(std::memory_order_relaxed)) {
    DGS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    if (dev < MAX_DEVICES) known[dev].store(true, std::memory_order_relaxed);
  }
  const int64_t most = sm_count();
  DGS_CUDA_TRY(launch_training(kernel, dim3(static_cast<unsigned>(items < most ? items : most)), TILE_THREADS, smem, s, args));
  return DGS_OK;
}

int heads_map(CUtensorMap* map, const AttnView& v, int32_t dtype, int d, int heads, int64_t rows) {
  return make_heads_map(map, v.p, dtype, d, heads, v.head, rows, v.row, 64, ATTN_TILE);
}

template <int DP, bool BF16>
int forward(const TileArgs& t, cudaStream_t s) {
  static_assert(ForwardShape<DP>::SMEM <= MAX_SMEM, "shared memory");
  static std::atomic<bool> known[MAX_DEVICES] = {};
  return launch_tiles(attn_forward_kernel<DP, BF16>, t, static_cast<int64_t>(t.a.q_tile_bound) * (t.a.head_pairs ? t.a.heads / 2 : t.a.heads), ForwardShape<DP>::SMEM, known, s);
}

template <int DP, bool BF16>
int backward(const TileArgs& t, cudaStream_t s) {
  static_assert(BackwardShape<DP>::SMEM <= MAX_SMEM, "shared memory");
  static std::atomic<bool> known[2][MAX_DEVICES] = {};
  const AttnArgs& a = t.a;
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  const auto ctas = [](int rows, int heads) {
    const int need = (rows + DELTA_THREADS / 16 - 1) / (DELTA_THREADS / 16), most = (sm_count() * 8 + heads - 1) / heads;
    return static_cast<unsigned>(need < most ? need : most);
  };
  DGS_CUDA_TRY(launch_training(attn_delta_kernel<T, DP / 8>, dim3(ctas((a.n_q + DELTA_ROWS - 1) / DELTA_ROWS * 2, 1)), DELTA_THREADS, 0, s, a,
                               lift<BF16>(), static_cast<int32_t>(!BF16)));
  if (!BF16) DGS_CUDA_TRY(launch_training(attn_norm_kernel<T>, dim3(ctas(a.n_k, a.kv_heads), a.kv_heads), DELTA_THREADS, 0, s, a));
  // (the queries first: they leave better deltas)
  if (int rc = launch_tiles(attn_dq_kernel<DP, BF16>, t, static_cast<int64_t>(a.q_tile_bound) * a.heads, BackwardShape<DP>::SMEM, known[1], s))
    return rc;
  if (a.dk != nullptr)
    return launch_tiles(attn_dkv_kernel<DP, BF16>, t, static_cast<int64_t>(a.k_tile_bound) * a.kv_heads, BackwardShape<DP>::SMEM, known[0], s);
  return DGS_OK;
}

}  // namespace

int attn_tiles_forward(const AttnArgs& a, int32_t dtype, cudaStream_t s) {
  TileArgs t{};
  t.a = a;
  if (int rc = heads_map(&t.q, a.q, dtype, a.d, a.heads, a.n_q)) return rc;
  if (int rc = heads_map(&t.k, a.k, dtype, a.d, a.kv_heads, a.n_k)) return rc;
  if (int rc = heads_map(&t.v, a.v, dtype, a.d, a.kv_heads, a.n_k)) return rc;
  if (a.d <= 64) return dtype == DGS_BF16 ? forward<64, true>(t, s) : forward<64, false>(t, s);
  return dtype == DGS_BF16 ? forward<128, true>(t, s) : forward<128, false>(t, s);
}

int attn_tiles_backward(const AttnArgs& a, int32_t dtype, cudaStream_t s) {
  TileArgs t{};
  t.a = a;
  if (int rc = heads_map(&t.q, a.q, dtype, a.d, a.heads, a.n_q)) return rc;
  if (int rc = heads_map(&t.k, a.k, dtype, a.d, a.kv_heads, a.n_k)) return rc;
  if (int rc = heads_map(&t.v, a.v, dtype, a.d, a.kv_heads, a.n_k)) return rc;
  if (int rc = heads_map(&t.dout, a.dout, dtype, a.d, a.heads, a.n_q)) return rc;
  if (a.d <= 64) return dtype == DGS_BF16 ? backward<64, true>(t, s) : backward<64, false>(t, s);
  return dtype == DGS_BF16 ? backward<128, true>(t, s) : backward<128, false>(t, s);
}

}  // namespace dgs
