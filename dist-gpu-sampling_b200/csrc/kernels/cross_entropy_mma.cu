// The cross entropy of 16-bit operands on the tensor cores.  The mathematics and the order of the launches are those of
// cross_entropy.cu; this file holds the products.
//
// One kernel in several forms, all of them persistent over pairs of CTAs (cta_group::2):
//   STATS    logits of a row block against a slice of the vocabulary; running maximum and sum of every row in registers
//            (NARROW, FEW_STATS: the same for few classes, few rows)
//   GRAD     logits of a piece again, left as G in 16 bits (FEW_GRAD: for few rows)
//   PRODUCT  dh += G W and dW = G^T h of a piece, the tiles of both in one launch (dW of one or two narrow rows: a kernel of its own
//            on the CUDA cores)
// A pair's tile is 256 x 256: each CTA of the pair holds 128 rows of it in its TMEM, fetches its 128 rows of A and its half
// of B, so an operand element crosses from L2 once per pair.  Roles: warp 0 fetches (TMA, five or six stages of 64 along k),
// warp 1 of the pair's first CTA issues the products, sixteen more work on finished accumulators (eight: 1.8 times as long at
// rows of 128, where they have most to do).  TMEM holds two accumulators, so the products of the next tile run beside the
// exponentials of the last one.
//
// What bounds it: at long rows the products (8 192 x 1 024 against 65 537 classes: forward 0.74 ms, 1.48 PFLOP/s; with the backward
// pass 3.6 ms, 1.22 PFLOP/s over the four products, under the power cap), whose operands come out of L2 at the 47 bytes a clock and
// SM that it gives (a fifth of the time is spent waiting for them); at rows of 128 the exponentials, 16 a clock and SM (1 024 rows
// against 2.4 M classes: 0.83 ms, the unit is busy for 79 % of it, at the 1.68 GHz that power leaves) and in the backward pass G's
// way through HBM; with few rows the reading of W (8 rows of 1 024 against 150 000 classes: 60 us, 5.1 TB/s).
// exp(s - m) = 2^((s - m) log2(e)): half a packed addition, half a packed multiplication and one ex2 an element.
//
// Every wait is bounded.  One that runs out marks the CTA's words as dead, all roles leave, the status word gets
// DGS_ERR_CUDA, and the pair frees its TMEM as usual.
#include "cross_entropy.h"
#include "tensor_core.cuh"

namespace dgs {
namespace tc {

namespace {
int encode(CUtensorMap* map, const void* base, int32_t dtype, uint32_t rank, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);
  static std::atomic<void*> known{nullptr};
  void* fn = known.load(std::memory_order_acquire);
  if (fn == nullptr) {
    cudaDriverEntryPointQueryResult found;
    DGS_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
    DGS_REQUIRE(found == cudaDriverEntryPointSuccess && fn != nullptr, DGS_ERR_CUDA, "the driver has no tensor maps");
    known.store(fn, std::memory_order_release);
  }
  const cuuint32_t step[3] = {1, 1, 1};
  const CUtensorMapDataType type = dtype == DGS_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == DGS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult rc = reinterpret_cast<Encode>(fn)(map, type, rank, const_cast<void*>(base), dims, strides, box, step,
                                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  DGS_REQUIRE(rc == CUDA_SUCCESS, DGS_ERR_CUDA, "tensor map of %lld x %lld elements, %lld bytes apart: error %d",
              static_cast<long long>(dims[1]), static_cast<long long>(dims[0]), static_cast<long long>(strides[0]), static_cast<int>(rc));
  return DGS_OK;
}
}  // namespace

int make_map(CUtensorMap* map, const void* base, int32_t dtype, int64_t cols, int64_t rows, int64_t pitch, uint32_t box_cols,
             uint32_t box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch) * dtype_bytes(dtype)};
  const cuuint32_t box[2] = {box_cols, box_rows};
  return encode(map, base, dtype, 2, dims, strides, box);
}

int make_heads_map(CUtensorMap* map, const void* base, int32_t dtype, int64_t d, int64_t heads, int64_t head_pitch, int64_t rows,
                   int64_t row_pitch, uint32_t box_cols, uint32_t box_rows) {
  // (a stride along which nothing lies is any that the encoding takes)
  if (heads <= 1 && head_pitch <= 0) head_pitch = d;
  if (rows <= 1 && row_pitch <= 0) row_pitch = d;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_pitch) * dtype_bytes(dtype),
                                 static_cast<cuuint64_t>(row_pitch) * dtype_bytes(dtype)};
  const cuuint32_t box[3] = {box_cols, 1, box_rows};
  return encode(map, base, dtype, 3, dims, strides, box);
}

}  // namespace tc

namespace {
using namespace tc;

constexpr int M_TILE = 256, N_TILE = 256, K_TILE = 64;  // of a pair
constexpr int M_CTA = M_TILE / 2;
constexpr int MMA_THREADS = 640, EPILOGUE_WARPS = 16, FIRST_EPILOGUE_WARP = 4;
constexpr int COL_GROUPS = EPILOGUE_WARPS / 4, GROUP_COLS = N_TILE / COL_GROUPS;  // the columns of a tile that a warp works on
constexpr uint32_t A_BYTES = M_CTA * K_TILE * 2, STAGE_BYTES = 2 * A_BYTES;
constexpr uint32_t BOX_BYTES = 64 * K_TILE * 2;  // 64 of m (or n) by 64 of k, MN-major
constexpr uint32_t STAGING_BYTES = 4096;         // 32 rows of 128 bytes: one store of a warp
constexpr uint32_t TMEM_COLS = 512;
constexpr float LOG2E = 1.4426950408889634f;
// Of G.  Two products read it, so it passes through HBM about three times unless L2 holds it (96 MB and less), which at D >= 200
// is hidden behind the products; larger pieces waste less on rounds that are not full (8 192 rows of 1 024, 65 537 classes:
// 48 MB 4.07 ms, 96 MB 3.64, 384 MB 3.53, 768 MB 3.57).
constexpr int64_t PIECE_BYTES = int64_t(256) << 20;

// G in 16 bits is as far from its value as results of that type are from theirs, and the errors of many rows and results average:
// gradients come out up to sqrt(2) times as far off as their own rounding.  They do not average where there are few: a row's
// results all carry the rounding of its largest entry, the target's.  There G takes two planes, its rounded value and what that
// leaves, and both products run over the two.  Forward and backward at rows of 512 and 50 000 classes: 8 rows 84 -> 98 us, 64 rows
// 86 -> 102, 256 rows 93 -> 168; so the fewer the rows, the more classes may there be.
inline bool two_planes(int64_t n, int64_t D, int64_t V) {
  return n <= 16 || (n <= 256 && n * n * V <= (int64_t(1) << 28)) || (n < V ? n : V) * D <= 1024;
}

// NARROW is STATS for no more than NARROW_COLS classes.  A tensor core cuts what it adds to an accumulator of 32 bits instead of
// rounding it, and the losses of few classes show it most.  There the products stop every NARROW_K blocks of k and the parts are added
// in registers, which hold 32 columns a lane beside the ones that arrive; the 64 of a whole tile would not fit.  So the losses of more
// classes, and of few rows, carry the cut: as a whole they are off by 4e-7 to 7e-7 of themselves at rows of 1 000, by 1.9e-6 at 4 096
// and 5e-6 at 8 192 (here 2e-7 at all of these).  Logits rounded to 16 bits would be off by 1e-3.
//
// FEW_STATS and FEW_GRAD are STATS and GRAD for no more than FEW_ROWS rows, with the operands changed over: classes are the
// accumulator's rows and the rows its 32 columns.  A lane works on its own class for eight rows; the other way round the few
// lanes that have a row would pass over all classes (8 rows of 203 against 800 000 classes, forward: 249 us, so 188).  What is left
// is the reading of W.
enum Mode { STATS, GRAD, PRODUCT, NARROW, FEW_STATS, FEW_GRAD };
constexpr int NARROW_COLS = N_TILE / 2, NARROW_K = 4;
constexpr int FEW_ROWS = 32, FEW_EACH = 8;  // rows; those that a warp works on
constexpr int FEW_PARTS = 8;                // statistics of a row and slice: four warps in each CTA of the pair
template <int MODE>
constexpr bool is_few() {
  return MODE == FEW_STATS || MODE == FEW_GRAD;
}
template <int MODE>
constexpr bool is_stats() {
  return MODE == STATS || MODE == NARROW || MODE == FEW_STATS;
}
template <int MODE>
constexpr int stages() {
  return is_stats<MODE>() ? 6 : 5;
}
// Where a row block meets all classes in one go, its CTAs join the four column groups' statistics themselves, by way of shared
// memory; JOINS of them, so that a warp that is ahead does not write over what another still reads (the accumulators let none be
// more than two tiles ahead).
constexpr int JOINS = 4;
struct JoinRows {
  float2 sum[COL_GROUPS][M_CTA];  // (maximum, sum)
  float target[M_CTA];
};
template <int MODE>
constexpr bool may_join() {
  return MODE == STATS || MODE == NARROW;
}
template <int MODE>
constexpr uint32_t smem_bytes() {  // alignment, stages, a staging buffer for each warp, barriers
  return 1024 + stages<MODE>() * STAGE_BYTES + (is_stats<MODE>() || is_few<MODE>() ? 0 : EPILOGUE_WARPS * STAGING_BYTES) + 256 +
         (may_join<MODE>() ? JOINS * static_cast<uint32_t>(sizeof(JoinRows)) : 0);
}

enum OutKind { OUT_F32_STORE, OUT_F32_ADD, OUT_TYPED, OUT_TYPED_ODD };

// One of the two products of a PRODUCT launch
struct Part {
  int32_t a_mn;     // A is held with m contiguous; its k are rows of the call (dW), else its m are (dh)
  int32_t n_tiles, n_step, splits;  // tiles of n_step columns: N_TILE, or half of it
  int32_t k_blocks;
  int32_t n_total;  // columns of the result
  int32_t m_total;
  int32_t out_kind;
  int32_t planes;      // of G: blocks of k alternate between them
  int32_t plane_rows;  // rows of G between them (a box that runs over the end of one meets rows of the other: its rows of h are
                       // zeros there, or its results are not stored)
  int64_t split_rows;  // rows between the splits' partial results
  void* odd;           // OUT_TYPED_ODD: the result itself, rows of n_total elements
};

struct alignas(64) MmaArgs {
  CUtensorMap a[2], b[2], out[2];
  Part part[2];
  int32_t items, parts;
  int32_t col_tiles, slices, k_blocks;
  int64_t n, V;  // GRAD: V is the width of the piece
  int32_t v0;    // GRAD: first class of the piece
  const int32_t* live;  // the number of packed rows, <= n; null: n
  const int32_t* word;  // of packed rows; null: the rows are those of the call, and so are the targets (STATS)
  const void* target;
  int64_t ignore_index;
  int32_t ids64;
  int32_t largest_count;
  float* target_logit;
  float* top;
  float* total;
  float *loss_out, *lse_out;  // STATS, NARROW: the rows' results, where there is one slice and rows are those of the call; else null
  const float* dloss;
  const float* lse;
  const float* hit;      // the targets' entries p - 1; null: from lse
  uint16_t* g;           // FEW_GRAD: G, rows low_pitch elements apart
  uint16_t* low;         // (FEW_)GRAD: the second plane of G, rows low_pitch elements apart; null: there is one plane
  int64_t low_pitch;
  const float* largest;  // the largest |dloss| of each CTA that packed rows
  int32_t* status;
};

struct Tile {
  int32_t m0, n0;      // of the pair
  int32_t k0, k1;      // blocks of K_TILE
  int32_t n;           // columns: N_TILE or half of it
  int32_t which;       // part
  int32_t split;
};

// What depends on the number of packed rows, which a launch learns from memory
struct Extent {
  int32_t rows, row_blocks, items, first_items;  // first_items: of part 0 (PRODUCT)
  int32_t row_k_blocks, slices;
};
template <int MODE>
__device__ __forceinline__ Extent extent_of(const MmaArgs& a) {
  Extent e;
  e.rows = a.live != nullptr ? *a.live : static_cast<int32_t>(a.n);
  e.row_blocks = e.rows > 0 ? (e.rows + M_TILE - 1) / M_TILE : 1;  // (no row at all: one block of zeros)
  e.row_k_blocks = e.rows > 0 ? (e.rows + K_TILE - 1) / K_TILE : 1;
  e.first_items = 0;
  e.slices = a.live != nullptr ? a.live[1] : a.slices;
  if constexpr (MODE == STATS) {
    e.items = e.row_blocks * e.slices;
  } else if constexpr (MODE == NARROW) {
    e.items = e.row_blocks;
  } else if constexpr (MODE == FEW_STATS) {
    e.items = a.slices;
  } else if constexpr (MODE == FEW_GRAD) {
    e.items = a.col_tiles;
  } else if constexpr (MODE == GRAD) {
    e.items = e.row_blocks * a.col_tiles;
  } else {
    e.items = 0;
    for (int i = 0; i < a.parts; ++i) {
      const int m_tiles = a.part[i].a_mn ? (a.part[i].m_total + M_TILE - 1) / M_TILE : e.row_blocks;
      const int items = m_tiles * a.part[i].n_tiles * a.part[i].splits;
      if (i == 0) e.first_items = items;
      e.items += items;
    }
  }
  return e;
}

template <int MODE>
__device__ __forceinline__ Tile tile_of(const MmaArgs& a, const Extent& ext, int item, int t) {
  Tile x;
  x.which = 0;
  x.split = 0;
  x.n = N_TILE;
  if constexpr (MODE == PRODUCT) {
    x.which = item >= ext.first_items;
    const Part& p = a.part[x.which];
    const int i = item - (x.which ? ext.first_items : 0);
    const int k_blocks = p.planes * (p.a_mn ? ext.row_k_blocks : p.k_blocks);
    const int nt = i % p.n_tiles, rest = i / p.n_tiles;
    x.split = rest % p.splits;
    x.m0 = rest / p.splits * M_TILE;
    x.n0 = nt * p.n_step;
    if (p.n_step < N_TILE || p.n_total - x.n0 <= N_TILE / 2) x.n = N_TILE / 2;
    x.k0 = static_cast<int32_t>(static_cast<int64_t>(k_blocks) * x.split / p.splits);
    x.k1 = static_cast<int32_t>(static_cast<int64_t>(k_blocks) * (x.split + 1) / p.splits);
  } else if constexpr (is_few<MODE>()) {
    x.n = FEW_ROWS;
    x.m0 = t * M_TILE;  // classes
    x.n0 = 0;
    x.k0 = 0;
    x.k1 = a.k_blocks;
  } else if constexpr (MODE == NARROW) {
    x.n = NARROW_COLS;
    x.m0 = item * M_TILE;
    x.n0 = 0;
    x.k0 = t * NARROW_K;
    x.k1 = a.k_blocks < x.k0 + NARROW_K ? a.k_blocks : x.k0 + NARROW_K;
  } else {
    x.m0 = item % ext.row_blocks * M_TILE;
    x.n0 = t * N_TILE;
    x.k0 = 0;
    x.k1 = a.k_blocks;
  }
  return x;
}
// the column tiles (NARROW: runs along k) [t0, t1) of an item
template <int MODE>
__device__ __forceinline__ void range_of(const MmaArgs& a, const Extent& ext, int item, int* t0, int* t1) {
  if constexpr (MODE == FEW_STATS) {
    *t0 = static_cast<int>(static_cast<int64_t>(a.col_tiles) * item / a.slices);
    *t1 = static_cast<int>(static_cast<int64_t>(a.col_tiles) * (item + 1) / a.slices);
  } else if constexpr (MODE == FEW_GRAD) {
    *t0 = item;
    *t1 = item + 1;
  } else if constexpr (MODE == STATS) {
    const int slice = item / ext.row_blocks;
    *t0 = static_cast<int>(static_cast<int64_t>(a.col_tiles) * slice / ext.slices);
    *t1 = static_cast<int>(static_cast<int64_t>(a.col_tiles) * (slice + 1) / ext.slices);
  } else if constexpr (MODE == NARROW) {
    *t0 = 0;
    *t1 = (a.k_blocks + NARROW_K - 1) / NARROW_K;
  } else if constexpr (MODE == GRAD) {
    *t0 = item / ext.row_blocks;
    *t1 = *t0 + 1;
  } else {
    *t0 = 0;
    *t1 = 1;
  }
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e^(v - base) for 32 values, in pairs: packed additions and multiplications halve what stands beside the 16 ex2 a clock and SM.
// (A share of the exponentials as polynomials on the multiply-add units does not help.)  The difference comes first and is exact, or
// nearly, where it counts: the largest logit of a row gives exactly one, so its loss is never negative.  v log2(e) - rn(base log2(e))
// in one operation would be off by 2^-24 |base| in each exponent, and so would be the loss.
__device__ __forceinline__ void exp_pairs(const uint32_t (&v)[32], float base, uint64_t (&e)[16]) {
  const uint64_t scale2 = two(LOG2E, LOG2E), minus2 = two(-base, -base);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float lo, hi;
    split2(mul2(add2(two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), minus2), scale2), &lo, &hi);
    e[i] = two(ex2(lo), ex2(hi));
  }
}

// Running maximum of one row and the sum of e^(s - top)
struct RowSum {
  float top = -INFINITY, total = 0.0f;
  __device__ __forceinline__ void add(uint32_t (&v)[32], int valid) {
    if (valid < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i >= valid) v[i] = __float_as_uint(-INFINITY);
    }
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max_or_nan(at(v, i), at(v, i + 4));
#pragma unroll
    for (int i = 8; i < 32; ++i) m[i & 3] = max_or_nan(m[i & 3], at(v, i));
    const float now = max_or_nan(max_or_nan(max_or_nan(m[0], m[1]), max_or_nan(m[2], m[3])), top);
    // nothing but minus infinity so far: the exponential must not see their difference
    const float base = now == -INFINITY ? 0.0f : now;
    uint64_t e[16];
    exp_pairs(v, base, e);
#pragma unroll
    for (int i = 4; i < 16; ++i) e[i & 3] = add2(e[i & 3], e[i]);
    float lo, hi;
    split2(add2(add2(e[0], e[1]), add2(e[2], e[3])), &lo, &hi);
    total = total * ex2((top - base) * LOG2E) + (lo + hi);  // (0 while top is minus infinity)
    top = now;
  }
  static __device__ __forceinline__ float at(const uint32_t (&v)[32], int i) { return __uint_as_float(v[i]); }
};

__device__ __forceinline__ float pick(const uint32_t (&bits)[32], int at) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i == at) r = bits[i];
  return __uint_as_float(r);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}
template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t v, float* lo, float* hi) {
  if constexpr (BF16) {
    *lo = __uint_as_float(v << 16);
    *hi = __uint_as_float(v & 0xffff0000u);
  } else {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v));
    *lo = t.x;
    *hi = t.y;
  }
}
__device__ __forceinline__ void st_shared(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// G is scaled so that its largest possible value, max |dloss|, becomes 2^15, and the products' results are scaled back.  float16:
// probabilities down to 2^-29 of it stay normal numbers.  Both types: the entries that weigh most, those of targets with a small
// probability, stand just below a power of two, where rounding to the type is off least (half as far as just above one: 275 rows
// with weights between half and three halves of 1 / 275 gave gradients 1.57 times as far off as their own rounding without it).
__device__ __forceinline__ float grad_factor(const float* largest, int count, int lane, bool inverse) {
  float m = 0.0f;
  for (int i = lane; i < count; i += 32) m = fmaxf(m, largest[i]);
  m = __uint_as_float(__reduce_max_sync(FULL_MASK, __float_as_uint(m)));
  m = m > 0.0f ? fminf(fmaxf(m, 1e-30f), 1e30f) : 1.0f;
  return inverse ? m * (1.0f / 32768.0f) : 32768.0f / m;
}

template <int MODE, bool BF16>
__global__ void __launch_bounds__(MMA_THREADS, 1) __cluster_dims__(2, 1, 1) ce_mma_kernel(const __grid_constant__ MmaArgs a) {
  constexpr int STAGES = stages<MODE>();
  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging = smem + STAGES * STAGE_BYTES;
  const uint32_t words = staging + (is_stats<MODE>() || is_few<MODE>() ? 0 : EPILOGUE_WARPS * STAGING_BYTES);
  const uint32_t full = words, empty = full + 8 * STAGES, acc_full = empty + 8 * STAGES, acc_empty = acc_full + 16, tmem_word = acc_empty + 16;
  volatile int32_t* dead = reinterpret_cast<volatile int32_t*>(smem_raw + (tmem_word + 8 - smem_addr(smem_raw)));
  const uint32_t joined = tmem_word + 16;  // a barrier for each of JOINS
  JoinRows* join_rows = reinterpret_cast<JoinRows*>(smem_raw + (words + 256 - smem_addr(smem_raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(acc_full + 8 * i, 1);
      bar_init(acc_empty + 8 * i, 2 * EPILOGUE_WARPS);
    }
    for (int i = 0; i < JOINS; ++i) bar_init(joined + 8 * i, EPILOGUE_WARPS);
    *dead = 0;
    bar_init_fence();
  }
  if (warp == 2) tmem_alloc(tmem_word, TMEM_COLS);
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_word) : "memory");
  pdl_enter();
  const Extent ext = extent_of<MODE>(a);

  bool ok = true;  // this thread's waits have all ended well
  if (warp == 0 && lane == 0) {
    // ---- fetch: this CTA's rows of A and its half of B
    fence_async_global();  // operands that ordinary stores of an earlier launch wrote
    int st = 0;
    uint32_t phase = 0;
    for (int item = pair; ok && item < ext.items; item += pairs) {
      int t0, t1;
      range_of<MODE>(a, ext, item, &t0, &t1);
      for (int t = t0; ok && t < t1; ++t) {
        const Tile x = tile_of<MODE>(a, ext, item, t);
        const CUtensorMap *ma = &a.a[x.which], *mb = &a.b[x.which];
        const bool a_mn = MODE == PRODUCT && a.part[x.which].a_mn;
        const uint32_t bytes = 2 * A_BYTES + x.n * (K_TILE * 2);  // of both CTAs
        const int32_t m = x.m0 + static_cast<int32_t>(rank) * M_CTA, n = x.n0 + static_cast<int32_t>(rank) * (x.n / 2);
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (!(ok = !*dead && bar_wait(empty + 8 * st, phase ^ 1))) break;
          const uint32_t to = smem + st * STAGE_BYTES, bar = in_cta(full + 8 * st, 0);
          if (rank == 0) bar_expect(full + 8 * st, bytes);
          // two planes: their blocks take turns, so that the other operand's block comes out of L2 the second time
          const bool alternate = MODE == PRODUCT && a.part[x.which].planes == 2;
          const int32_t k = (alternate ? kb >> 1 : kb) * K_TILE, plane = alternate && (kb & 1) ? a.part[x.which].plane_rows : 0;
          if (a_mn) {
            load_box(to, ma, m, k + plane, bar);
            load_box(to + BOX_BYTES, ma, m + 64, k + plane, bar);
          } else {
            load_box(to, ma, k, m + plane, bar);
          }
          if (MODE == PRODUCT) {
            load_box(to + A_BYTES, mb, n, k, bar);
            if (x.n == N_TILE) load_box(to + A_BYTES + BOX_BYTES, mb, n + 64, k, bar);
          } else {
            load_box(to + A_BYTES, mb, k, n, bar);
          }
          if (++st == STAGES) st = 0, phase ^= 1;
        }
      }
    }
    if (!ok) {
      // this CTA's copies still in flight land within microseconds; nobody will read them, but they must not outlive the CTA
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- products
    int st = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    for (int item = pair; ok && item < ext.items; item += pairs) {
      int t0, t1;
      range_of<MODE>(a, ext, item, &t0, &t1);
      for (int t = t0; ok && t < t1; ++t) {
        const Tile x = tile_of<MODE>(a, ext, item, t);
        const bool a_mn = MODE == PRODUCT && a.part[x.which].a_mn;
        constexpr bool b_mn = MODE == PRODUCT;
        const uint32_t idesc = mma_desc(BF16, a_mn, b_mn, M_TILE, x.n);
        const uint32_t d = tmem + buf * N_TILE;
        if (!(ok = !*dead && bar_wait(acc_empty + 8 * buf, acc_phase ^ 1))) break;
        fence_after();
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (!(ok = !*dead && bar_wait(full + 8 * st, phase))) break;
          fence_after();
          const uint32_t sa = smem + st * STAGE_BYTES, sb = sa + A_BYTES;
          const uint64_t da = smem_desc(sa, a_mn ? BOX_BYTES : 16, 1024), db = smem_desc(sb, b_mn ? BOX_BYTES : 16, 1024);
          // 16 of k: 32 bytes of every row (K-major) or 16 rows of 128 bytes (MN-major), in units of 16 bytes
          const uint32_t step_a = a_mn ? 128 : 2, step_b = b_mn ? 128 : 2;
#pragma unroll
          for (int k = 0; k < K_TILE / 16; ++k) mma(d, da + k * step_a, db + k * step_b, idesc, kb > x.k0 || k > 0);
          mma_commit(empty + 8 * st);
          if (++st == STAGES) st = 0, phase ^= 1;
        }
        if (!ok) break;
        mma_commit(acc_full + 8 * buf);
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
    }
  } else if (is_few<MODE>() && warp >= FIRST_EPILOGUE_WARP) {
    // ---- finished accumulators, classes by rows: a lane has one class of the tile, the warp eight rows
    const int quarter = warp & 3, group = (warp - FIRST_EPILOGUE_WARP) >> 2, r0 = group * FEW_EACH;
    const uint32_t from0 = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + r0;
    const uint32_t free_bar = in_cta(acc_empty, 0);
    int buf = 0;
    uint32_t acc_phase = 0;
    const float factor = MODE == FEW_GRAD ? grad_factor(a.largest, a.largest_count, lane, false) : 1.0f;
    int32_t word[FEW_EACH];
    float grad[FEW_EACH], lse[FEW_EACH], hit[FEW_EACH];
#pragma unroll
    for (int r = 0; r < FEW_EACH; ++r) {
      word[r] = -1;
      grad[r] = lse[r] = hit[r] = 0.0f;
      if (r0 + r < ext.rows) {
        bool wrong;
        word[r] = MODE == FEW_GRAD || a.word != nullptr ? a.word[r0 + r] : target_word(a.target, a.ids64, r0 + r, a.V, a.ignore_index, &wrong);
        if (MODE == FEW_GRAD) {
          grad[r] = a.dloss[r0 + r] * factor;
          lse[r] = a.lse[r0 + r];
          if (a.hit != nullptr) hit[r] = a.hit[r0 + r];
        }
      }
    }
    for (int item = pair; ok && item < ext.items; item += pairs) {
      int t0, t1;
      range_of<MODE>(a, ext, item, &t0, &t1);
      float top[FEW_EACH], total[FEW_EACH];  // of this lane's classes
#pragma unroll
      for (int r = 0; r < FEW_EACH; ++r) top[r] = -INFINITY, total[r] = 0.0f;
      for (int t = t0; t < t1; ++t) {
        ok = !*dead && bar_wait(acc_full + 8 * buf, acc_phase);
        ok = __all_sync(FULL_MASK, ok);
        if (!ok) break;
        fence_after();
        uint32_t bits[FEW_EACH];
        tmem_read8(from0 + buf * N_TILE, bits);
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_in(free_bar + 8 * buf);
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
        const int32_t c = t * M_TILE + static_cast<int32_t>(rank) * M_CTA + quarter * 32 + lane;  // FEW_GRAD: of the piece
        if (c >= a.V) continue;
#pragma unroll
        for (int r = 0; r < FEW_EACH; ++r) {
          if (r0 + r >= a.n) break;  // (the same for all lanes)
          const float v = __uint_as_float(bits[r]);
          if constexpr (MODE == FEW_STATS) {
            if (c == word[r]) a.target_logit[r0 + r] = v;
            const float d = v - top[r], e = ex2(-fabsf(d) * LOG2E);
            if (v > top[r]) {
              total[r] = total[r] * e + 1.0f;  // (0 * 0 + 1 for the first)
              top[r] = v;
            } else if (v != -INFINITY) {
              total[r] += e;  // (a NaN goes this way and stays)
            }
          } else {
            float g = 0.0f;
            if (word[r] >= 0) {
              g = ex2((v - lse[r]) * LOG2E);
              if (c + a.v0 == word[r]) g = a.hit != nullptr ? hit[r] : g - 1.0f;
              g *= grad[r];
            }
            const uint32_t hi = pack2<BF16>(g, 0.0f);
            const int64_t at = static_cast<int64_t>(r0 + r) * a.low_pitch + c;
            a.g[at] = static_cast<uint16_t>(hi);
            if (a.low != nullptr) {
              float back, none;
              unpack2<BF16>(hi, &back, &none);
              a.low[at] = static_cast<uint16_t>(pack2<BF16>(g - back, 0.0f));
            }
          }
        }
      }
      if (MODE == FEW_STATS && ok) {
        // one pair for the warp's lanes, in an order that is always the same
#pragma unroll
        for (int r = 0; r < FEW_EACH; ++r) {
          float m = top[r];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, o));
          float s = m == -INFINITY ? total[r] : total[r] * ex2((top[r] - m) * LOG2E);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL_MASK, s, o);
          if (lane == 0 && r0 + r < ext.rows) {
            const int64_t at = (static_cast<int64_t>(r0 + r) * a.slices + item) * FEW_PARTS + static_cast<int64_t>(rank) * 4 + quarter;
            a.top[at] = m;
            a.total[at] = s;
          }
        }
      }
    }
  } else if (!is_few<MODE>() && warp >= FIRST_EPILOGUE_WARP) {
    // ---- finished accumulators: a warp reads the 32 lanes (rows) that its number allows, and a quarter of the columns
    constexpr int COLS = MODE == NARROW ? NARROW_COLS / COL_GROUPS : GROUP_COLS;
    const int quarter = warp & 3, group = (warp - FIRST_EPILOGUE_WARP) >> 2, c0 = group * COLS;
    const uint32_t from0 = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c0;
    const uint32_t stage_at = staging + (warp - FIRST_EPILOGUE_WARP) * STAGING_BYTES;
    const uint32_t free_bar = in_cta(acc_empty, 0);
    int buf = 0;
    uint32_t acc_phase = 0;
    float factor = 1.0f;
    if (!is_stats<MODE>()) factor = grad_factor(a.largest, a.largest_count, lane, MODE == PRODUCT);
    // what a row brings along; GRAD's next row is asked for a tile ahead
    const int32_t my_row = static_cast<int32_t>(rank) * M_CTA + quarter * 32 + lane;
    int32_t next_word = -1;
    float next_grad = 0.0f, next_lse = 0.0f, next_hit = 0.0f;
    auto ask = [&](int item) {
      const int32_t row = tile_of<MODE>(a, ext, item, 0).m0 + my_row;
      next_word = -1;
      if (item >= ext.items || row >= ext.rows) return;
      bool wrong;
      next_word = MODE == GRAD || a.word != nullptr ? a.word[row] : target_word(a.target, a.ids64, row, a.V, a.ignore_index, &wrong);
      if (MODE == GRAD) {
        next_grad = a.dloss[row];
        next_lse = a.lse[row];
        if (a.hit != nullptr) next_hit = a.hit[row];
      }
    };
    if (MODE != PRODUCT) ask(pair);
    int round = 0;  // items so far
    for (int item = pair; ok && item < ext.items; item += pairs, ++round) {
      JoinRows* join = may_join<MODE>() && a.loss_out != nullptr ? join_rows + round % JOINS : nullptr;
      const int in_cta_row = quarter * 32 + lane;
      int t0, t1;
      range_of<MODE>(a, ext, item, &t0, &t1);
      RowSum sum;
      uint32_t logits[MODE == NARROW ? 32 : 1];
      const int32_t word = next_word;
      const float grad = next_grad * factor, lse = next_lse, hit = next_hit;
      if (MODE != PRODUCT) ask(item + pairs);
      for (int t = t0; t < t1; ++t) {
        const Tile x = tile_of<MODE>(a, ext, item, t);
        const int32_t row = x.m0 + my_row;
        ok = !*dead && bar_wait(acc_full + 8 * buf, acc_phase);
        ok = __all_sync(FULL_MASK, ok);
        if (!ok) break;
        fence_after();
        // a narrow tile has nothing for half of the warps, a block that is not full nothing for those behind its last row
        const int32_t last_row = is_stats<MODE>() ? ext.rows : MODE == GRAD ? static_cast<int32_t>(a.n) : a.part[x.which].m_total;
        const int chunks = c0 < x.n && row - lane < last_row ? COLS / 32 : 0;
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c) {
          if (c < chunks) {
            uint32_t now[32];
            tmem_load32(from0 + buf * N_TILE + c * 32, now);
            tmem_wait(now);
            if (c + 1 == chunks) {
              fence_before();
              __syncwarp();
              if (lane == 0) bar_arrive_in(free_bar + 8 * buf);
            }
            const int32_t col = x.n0 + c0 + c * 32;  // first of the 32
            if constexpr (MODE == NARROW) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                logits[i] = t == t0 ? now[i] : __float_as_uint(__uint_as_float(logits[i]) + __uint_as_float(now[i]));
              if (t + 1 == t1) {
                const uint32_t at = static_cast<uint32_t>(word - col);
                if (at < 32u && word >= 0) *(join ? &join->target[in_cta_row] : &a.target_logit[row]) = pick(logits, static_cast<int>(at));
                if (col < a.V) sum.add(logits, static_cast<int32_t>(a.V) - col);
              }
            } else if constexpr (MODE == STATS) {
              const int32_t left = static_cast<int32_t>(a.V) - col;
              const uint32_t at = static_cast<uint32_t>(word - col);
              if (at < 32u && word >= 0) *(join ? &join->target[in_cta_row] : &a.target_logit[row]) = pick(now, static_cast<int>(at));
              if (left > 0) sum.add(now, left);
            } else if constexpr (MODE == GRAD) {
              uint64_t e[16];
              exp_pairs(now, lse, e);
              const uint64_t grad2 = two(grad, grad);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float lo, hi;
                split2(mul2(e[i], grad2), &lo, &hi);
                now[2 * i] = __float_as_uint(lo);
                now[2 * i + 1] = __float_as_uint(hi);
              }
              const uint32_t at = static_cast<uint32_t>(word - a.v0 - col);
              if (at < 32u && word >= 0) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (i == static_cast<int>(at)) now[i] = __float_as_uint(a.hit != nullptr ? grad * hit : __uint_as_float(now[i]) - grad);
              }
              if (word < 0) {
#pragma unroll
                for (int i = 0; i < 32; ++i) now[i] = 0;
              }
            }
            if constexpr (!is_stats<MODE>()) {
              const int kind = MODE == GRAD ? static_cast<int>(OUT_TYPED) : a.part[x.which].out_kind;
              const bool typed = kind == OUT_TYPED || kind == OUT_TYPED_ODD;
              if (MODE == PRODUCT) {
#pragma unroll
                for (int i = 0; i < 32; ++i) now[i] = __float_as_uint(__uint_as_float(now[i]) * factor);
              }
              // two chunks of 16-bit values fill the buffer, one of 32-bit values does
              if (!typed || (c & 1) == 0) {
                if (lane == 0) store_wait_read<0>();
                __syncwarp();
              }
              const uint32_t at_row = stage_at + lane * 128;
              if (typed) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  uint32_t p[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    p[i] = pack2<BF16>(__uint_as_float(now[j * 8 + i * 2]), __uint_as_float(now[j * 8 + i * 2 + 1]));
                  st_shared(at_row + (((c & 1) * 4 + j) ^ (lane & 7)) * 16, p[0], p[1], p[2], p[3]);
                  if (MODE == GRAD && a.low != nullptr) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                      float hi0, hi1;
                      unpack2<BF16>(p[i], &hi0, &hi1);
                      p[i] = pack2<BF16>(__uint_as_float(now[j * 8 + i * 2]) - hi0, __uint_as_float(now[j * 8 + i * 2 + 1]) - hi1);
                    }
                    if (row < a.n) *reinterpret_cast<uint4*>(a.low + row * a.low_pitch + col + j * 8) = uint4{p[0], p[1], p[2], p[3]};
                  }
                }
              } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  st_shared(at_row + (j ^ (lane & 7)) * 16, now[j * 4], now[j * 4 + 1], now[j * 4 + 2], now[j * 4 + 3]);
              }
              if (!typed || (c & 1) == 1) {
                const int32_t first = typed ? col - 32 : col, row0 = row - lane;
                if (kind == OUT_TYPED_ODD) {
                  // rows that do not begin at 16-byte boundaries: element by element, a row at a time
                  __syncwarp();
                  const Part& p = a.part[x.which];
                  for (int r = 0; r < 32 && row0 + r < p.m_total; ++r) {
#pragma unroll
                    for (int e = lane; e < 64; e += 32) {
                      uint16_t bits;
                      asm volatile("ld.shared.b16 %0, [%1];"
                                   : "=h"(bits)
                                   : "r"(stage_at + r * 128 + (((e >> 3) ^ (r & 7)) * 16) + (e & 7) * 2)
                                   : "memory");
                      if (first + e < p.n_total)
                        static_cast<uint16_t*>(p.odd)[static_cast<int64_t>(row0 + r) * p.n_total + first + e] = bits;
                    }
                  }
                  __syncwarp();
                } else {
                  fence_async_smem();
                  __syncwarp();
                  if (lane == 0) {
                    const CUtensorMap* to = &a.out[x.which];
                    const int32_t y = MODE == PRODUCT && !typed ? static_cast<int32_t>(x.split * a.part[x.which].split_rows) + row0 : row0;
                    if (kind == OUT_F32_ADD) add_box(to, first, y, stage_at);
                    else store_box(to, first, y, stage_at);
                    store_commit();
                  }
                }
              }
            }
          }
        }
        if (chunks == 0 && lane == 0) bar_arrive_in(free_bar + 8 * buf);
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
      if (may_join<MODE>() && ok && join != nullptr) {
        join->sum[group][in_cta_row] = float2{sum.top, sum.total};
        __syncwarp();
        if (lane == 0) bar_arrive(joined + 8 * (round % JOINS));
        if (group == 0) {
          ok = !*dead && bar_wait(joined + 8 * (round % JOINS), (round / JOINS) & 1);
          ok = __all_sync(FULL_MASK, ok);
          if (!ok) break;
          const int32_t row = item * M_TILE + my_row;
          float m = -INFINITY, s = 0.0f;
#pragma unroll
          for (int g = 0; g < COL_GROUPS; ++g) m = fmaxf(m, join->sum[g][in_cta_row].x);
          const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
          for (int g = 0; g < COL_GROUPS; ++g) s += join->sum[g][in_cta_row].y * expf(join->sum[g][in_cta_row].x - base);
          if (row < ext.rows) {
            bool wrong = false;
            if (a.word == nullptr) target_word(a.target, a.ids64, row, a.V, a.ignore_index, &wrong);
            if (wrong) raise_status(a.status, DGS_ERR_RANGE);
            const float l = logf(s);
            a.lse_out[row] = word >= 0 ? base + l : 0.0f;
            a.loss_out[row] = word >= 0 ? (base - join->target[in_cta_row]) + l : 0.0f;
          }
        }
      } else if (is_stats<MODE>() && ok) {
        const int32_t row = item % ext.row_blocks * M_TILE + static_cast<int32_t>(rank) * M_CTA + quarter * 32 + lane;
        const int64_t at = static_cast<int64_t>(row) * (ext.slices * COL_GROUPS) + item / ext.row_blocks * COL_GROUPS + group;
        if (row < ext.rows) {
          a.top[at] = sum.top;
          a.total[at] = sum.total;
        }
      }
    }
    if (!is_stats<MODE>() && lane == 0) store_wait_all();
  }
  if (!ok) {
    *dead = 1;
    raise_status(a.status, DGS_ERR_CUDA);
  }
  __syncwarp();
  __syncthreads();
  fence_before();
  cluster_sync();  // the pair's products, copies and arrivals are over
  fence_after();
  if (warp == 2) tmem_free(tmem, TMEM_COLS);
}

// The weight's rows, `pitch` elements apart (rows of an odd length cannot be fetched by TMA where they lie).  A lane makes eight
// elements out of the two aligned 16-byte words that hold them; words that reach over the matrix's first or last byte are read
// element by element.
__device__ __forceinline__ uint4 eight_elements(const uint16_t* from, int count, uintptr_t first, uintptr_t end) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(from), word = at & ~uintptr_t(15);
  const uint32_t skip = static_cast<uint32_t>(at - word) >> 1;  // elements in front of the first
  if (word >= first && word + (skip ? 32 : 16) <= end) {
    const uint4 a = *reinterpret_cast<const uint4*>(word);
    uint32_t v[8] = {a.x, a.y, a.z, a.w, 0, 0, 0, 0};
    if (skip) {
      const uint4 b = *reinterpret_cast<const uint4*>(word + 16);
      v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    // whole words first, then the odd element
    if (skip & 4) {
#pragma unroll
      for (int i = 0; i < 6; ++i) v[i] = i + 2 < 8 ? v[i + 2] : 0;
    }
    if (skip & 2) {
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = v[i + 1];
    }
    if (skip & 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __funnelshift_r(v[i], v[i + 1], 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 2 * i + 1 < count ? v[i] : 2 * i < count ? v[i] & 0xffffu : 0u;
    return uint4{v[0], v[1], v[2], v[3]};
  }
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = 2 * i < count ? from[2 * i] : 0u, hi = 2 * i + 1 < count ? from[2 * i + 1] : 0u;
    v[i] = lo | (hi << 16);
  }
  return uint4{v[0], v[1], v[2], v[3]};
}

__global__ void __launch_bounds__(256) ce_pack_weight_kernel(const uint16_t* __restrict__ weight, const int64_t stride, const int64_t V,
                                                             const int D, const int pitch, uint16_t* __restrict__ packed) {
  pdl_enter();
  const uintptr_t first = reinterpret_cast<uintptr_t>(weight), end = reinterpret_cast<uintptr_t>(weight + (V - 1) * stride + D);
  const int chunks = pitch / 8;
  const int64_t all = V * chunks, step = static_cast<int64_t>(gridDim.x) * 256;
  // (row and chunk are carried along: a division of 64 bits for every eight elements would cost more than moving them)
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, row = i / chunks;
  int chunk = static_cast<int>(i - row * chunks);
  const int64_t step_rows = step / chunks;
  const int step_chunks = static_cast<int>(step - step_rows * chunks);
#pragma unroll 4
  for (; i < all; i += step) {
    const int left = D - chunk * 8;
    *reinterpret_cast<uint4*>(packed + row * pitch + chunk * 8) =
        eight_elements(weight + row * stride + chunk * 8, left < 8 ? left : 8, first, end);
    row += step_rows;
    chunk += step_chunks;
    if (chunk >= chunks) {
      chunk -= chunks;
      ++row;
    }
  }
}

// dW for one or two rows of few columns and many classes: no product to speak of but the writing of dW, which tiles of the tensor
// core pass through their accumulators, 256 x 256 values for 64 of k of which one or two count.  A thread keeps the rows' values of
// VEC columns and takes CLASSES classes at a time: a load of G a row and plane, sums in 32 bits, stores side by side.  Forward and
// backward, one row against 831 627 classes: 80 columns 311 -> 272 us (30 of it this kernel, 4.5 TB/s; the product for dh that is
// left takes 150), 75 columns 485 -> 397, 256 columns 417 -> 397; two rows: 75 columns 493 -> 421, 256 columns 417 -> 420.  With
// eight rows it loses (80 columns 333 -> 363), and below some 50 000 classes the launch costs more than it saves (2 000 classes
// 28 -> 30); against 140 000 one row of 80 goes from 78 to 73.
constexpr int FEW_WEIGHT = 2, FEW_WEIGHT_THREADS = 256;
constexpr int64_t FEW_WEIGHT_CLASSES = int64_t(1) << 17;
struct FewWeightArgs {
  const uint16_t* rows;  // packed
  int64_t pitch;
  const uint16_t* g;
  int64_t g_pitch;
  int32_t n, D, across;  // across: threads that share a class
  int64_t width;                 // classes of the piece
  uint16_t* out;
  const float* largest;
  int32_t largest_count;
};

template <bool BF16, int VEC, int ROWS>
__global__ void __launch_bounds__(FEW_WEIGHT_THREADS, 2) ce_few_weight_kernel(const __grid_constant__ FewWeightArgs a) {
  constexpr int CLASSES = VEC == 1 ? 8 : 4;
  pdl_enter();
  const float factor = grad_factor(a.largest, a.largest_count, threadIdx.x & 31, true);
  const int group = threadIdx.x / a.across, groups = FEW_WEIGHT_THREADS / a.across;
  const int col = threadIdx.x % a.across * VEC;
  if (group >= groups) return;
  float h[ROWS][VEC];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float unused;
      h[i][e] = 0.0f;
      if (i < a.n) unpack2<BF16>(a.rows[i * a.pitch + col + e], &h[i][e], &unused);
    }
  for (int64_t v = (static_cast<int64_t>(blockIdx.x) * groups + group) * CLASSES; v < a.width;
       v += static_cast<int64_t>(gridDim.x) * groups * CLASSES) {
    uint32_t both[ROWS][2][CLASSES / 2];  // of two planes, all under way at once
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // (G's rows have room for whole tiles: nothing is read behind them)
        const uint16_t* from = a.g + (static_cast<int64_t>(q) * a.n + i) * a.g_pitch + v;
        if constexpr (CLASSES == 8) {
          const uint4 x = i < a.n ? *reinterpret_cast<const uint4*>(from) : uint4{0, 0, 0, 0};
          both[i][q][0] = x.x, both[i][q][1] = x.y, both[i][q][2] = x.z, both[i][q][3] = x.w;
        } else {
          const uint2 x = i < a.n ? *reinterpret_cast<const uint2*>(from) : uint2{0, 0};
          both[i][q][0] = x.x, both[i][q][1] = x.y;
        }
      }
    }
    float acc[CLASSES][VEC] = {};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
#pragma unroll
      for (int k = 0; k < CLASSES; k += 2) {
        float high[2], low[2];
        unpack2<BF16>(both[i][0][k / 2], &high[0], &high[1]);
        unpack2<BF16>(both[i][1][k / 2], &low[0], &low[1]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          acc[k][e] = fmaf(high[0] + low[0], h[i][e], acc[k][e]);
          acc[k + 1][e] = fmaf(high[1] + low[1], h[i][e], acc[k + 1][e]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < CLASSES; ++k) {
      if (v + k < a.width) {
        uint16_t* to = a.out + (v + k) * a.D + col;
        if constexpr (VEC == 1) {
          *to = static_cast<uint16_t>(pack2<BF16>(acc[k][0] * factor, 0.0f));
        } else {
          *reinterpret_cast<uint2*>(to) =
              uint2{pack2<BF16>(acc[k][0] * factor, acc[k][1] * factor), pack2<BF16>(acc[k][2] * factor, acc[k][3] * factor)};
        }
      }
    }
  }
}

template <bool BF16>
int few_weight(FewWeightArgs a, cudaStream_t s) {
  const bool fours = a.D % 4 == 0 && aligned_to(a.out, 8);
  const int classes = fours ? 4 : 8;
  a.across = a.D / (fours ? 4 : 1);  // (D <= N_TILE)
  const int64_t need = tiles(a.width, FEW_WEIGHT_THREADS / a.across * classes), most = static_cast<int64_t>(sm_count()) * 16;
  const dim3 grid(static_cast<unsigned>(need < most ? need : most));
  auto kernel = a.n == 1 ? fours ? ce_few_weight_kernel<BF16, 4, 1> : ce_few_weight_kernel<BF16, 1, 1>
                         : fours ? ce_few_weight_kernel<BF16, 4, 2> : ce_few_weight_kernel<BF16, 1, 2>;
  DGS_CUDA_TRY(launch_training(kernel, grid, FEW_WEIGHT_THREADS, 0, s, a));
  return DGS_OK;
}

// ---- host side -----------------------------------------------------------------------------------------------------
struct MmaPlan {
  int64_t pitch, row_blocks, col_tiles, slices, pairs;
  int64_t piece, splits, dpitch;
  int64_t planes;  // of G
  bool one_piece, compact, dh_first, few, few_weight;
  size_t packed, word, slot, live, counts, weight, target_logit, top, total, dloss, lse, hit, largest, g, dh;
  size_t forward_bytes, backward_bytes;
};

// How often dh's tiles are cut along the classes, and whether they come before dW's: the launch deals its items to the pairs in
// turn, and the cut is the one whose busiest pair has the least to do, in blocks of K_TILE plus what an item costs besides.
int64_t splits_for(int64_t row_blocks, int64_t d_tiles, int64_t dh_k, int64_t dw_tiles, int64_t dw_k, int64_t pairs, bool* dh_first) {
  constexpr int64_t kItem = 6, kMostSplits = 64;
  int64_t best = 1, least = INT64_MAX;
  *dh_first = true;
  // (1 to 8, then steps of an eighth to a quarter: this is worked out on every call)
  for (int64_t s = 1; s <= kMostSplits && (s == 1 || (s * 4 <= dh_k && row_blocks * d_tiles * s <= 32 * pairs)); s += s < 8 ? 1 : s < 16 ? 2 : s < 32 ? 4 : 8) {
    const int64_t count[2] = {row_blocks * d_tiles * s, dw_tiles * d_tiles}, cost[2] = {tiles(dh_k, s) + kItem, dw_k + kItem};
    for (int first = 0; first < 2; ++first) {
      const int64_t n0 = count[first], n1 = count[1 - first], c0 = cost[first], c1 = cost[1 - first];
      // the first r0 pairs have one item of the first kind more than the others; those of the second kind begin where these ended,
      // and r1 pairs, the next ones round the circle, have one more of them
      const int64_t r0 = n0 % pairs, r1 = n1 % pairs;
      const int64_t more = r0 + r1 > pairs ? c0 + c1 : r0 > 0 && (r1 == 0 || c0 > c1) ? c0 : r1 > 0 ? c1 : 0;
      const int64_t most = n0 / pairs * c0 + n1 / pairs * c1 + more;
      if (most < least) {
        least = most;
        best = s;
        *dh_first = first == 0;
      }
    }
  }
  return best;
}

// Whether the rows without a valid target are left out of the products.  That takes a launch more, and dh leaves by way of its
// 32-bit form to be spread over the call's rows.  Forward / forward and backward, no row ignored and 30 % of them, in us:
//   4 099 x 203 x 30 011 (2.5e10)  not compact 67 / 278 and 66 / 273,  compact 70 / 286 and 54 / 222
//   2 048 x 256 x 20 000 (1.0e10)  not compact 25 / 102 and 25 / 101,  compact 32 / 114 and 28 / 96
bool worth_compacting(int64_t n, int64_t D, int64_t V) {
  return static_cast<double>(n) * static_cast<double>(D) * static_cast<double>(V) >= 2e10 && n <= (int64_t(1) << 22);
}

MmaPlan make_plan(int64_t n, int64_t D, int64_t V) {
  MmaPlan p{};
  p.pairs = sm_count() / 2;
  p.pitch = up(D, 8);
  p.row_blocks = tiles(n, M_TILE);
  p.col_tiles = tiles(V, N_TILE);
  p.few = n <= FEW_ROWS && V > NARROW_COLS;
  p.slices = !p.few ? slices_for(p.row_blocks, p.col_tiles, p.pairs) : p.col_tiles < p.pairs ? p.col_tiles : p.pairs;
  // as many column tiles as PIECE_BYTES allow, rounded down to full rounds of the GRAD launch
  p.planes = two_planes(n, D, V) ? 2 : 1;
  int64_t piece_tiles = PIECE_BYTES / 2 / (p.planes * n) / N_TILE;
  if (piece_tiles < 1) piece_tiles = 1;
  if (piece_tiles >= p.col_tiles) {
    piece_tiles = p.col_tiles;
  } else if (p.row_blocks * piece_tiles >= p.pairs) {
    const int64_t rounds = p.row_blocks * piece_tiles / p.pairs, full = rounds * p.pairs / p.row_blocks;
    if (full > 0) piece_tiles = full;
  }
  p.piece = piece_tiles * N_TILE;
  p.one_piece = p.piece >= V;
  p.dpitch = up(D, 4);
  p.compact = worth_compacting(n, D, V);
  p.few_weight = n <= FEW_WEIGHT && n * D <= N_TILE && V >= FEW_WEIGHT_CLASSES && p.planes == 2 && !p.compact;
  p.splits = splits_for(p.row_blocks, tiles(D, N_TILE), p.planes * tiles(p.piece, K_TILE), p.few_weight ? 0 : piece_tiles, p.planes * tiles(n, K_TILE),
                        p.pairs, &p.dh_first);
  Layout l;
  p.packed = l.take(n * p.pitch * 2);
  p.word = l.take(n * 4);
  if (p.compact) {
    p.slot = l.take(n * 4);
    p.live = l.take(8);
    p.counts = l.take(tiles(n, CE_COUNT_ROWS) * 4);
  }
  if (D % 8 != 0) p.weight = l.take(V * p.pitch * 2);
  const Layout common = l;
  p.target_logit = l.take(n * 4);
  // (compact: the number of slices follows the number of rows, which is not known here; but blocks * slices <= kMostRounds * pairs
  // unless there is one slice)
  const int64_t most = p.few ? n * p.slices * FEW_PARTS : (p.compact ? n + kMostRounds * p.pairs * M_TILE : n * p.slices) * COL_GROUPS;
  p.top = l.take(most * 4);
  p.total = l.take(most * 4);
  p.forward_bytes = l.bytes;
  l = common;
  p.dloss = l.take(n * 4);
  p.lse = l.take(n * 4);
  p.hit = l.take(n * 4);
  p.largest = l.take(ce_pack_ctas(n) * 4);
  p.g = l.take(p.planes * n * p.piece * 2);
  if (!(p.one_piece && p.splits == 1 && !p.compact)) p.dh = l.take(p.splits * p.row_blocks * M_TILE * p.dpitch * 4);
  p.backward_bytes = l.bytes;
  return p;
}

template <int MODE, bool BF16>
int launch(const MmaArgs& a, int64_t pairs, cudaStream_t s) {
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> allowed[kMaxDevices] = {};
  auto kernel = ce_mma_kernel<MODE, BF16>;
  int dev = 0;
  DGS_CUDA_TRY(cudaGetDevice(&dev));
  DGS_REQUIRE(dev >= 0 && dev < kMaxDevices, DGS_ERR_UNSUPPORTED, "cross entropy: device ordinal %d", dev);
  if (!allowed[dev].load(std::memory_order_acquire)) {
    DGS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<MODE>())));
    allowed[dev].store(true, std::memory_order_release);
  }
  const int64_t used = a.items < pairs ? a.items : pairs;
  DGS_CUDA_TRY(launch_training(kernel, dim3(static_cast<unsigned>(2 * used)), MMA_THREADS, smem_bytes<MODE>(), s, a));
  return DGS_OK;
}
template <int MODE>
int launch(const MmaArgs& a, int64_t pairs, int32_t dtype, cudaStream_t s) {
  return dtype == DGS_BF16 ? launch<MODE, true>(a, pairs, s) : launch<MODE, false>(a, pairs, s);
}

// the weight as TMA can fetch it
struct Weight {
  const uint16_t* p;
  int64_t stride;
};
int fetchable_weight(const CeProblem& q, const MmaPlan& p, Weight* w, cudaStream_t s) {
  *w = Weight{static_cast<const uint16_t*>(q.weight), q.V == 1 ? p.pitch : q.weight_stride};
  if (aligned_to(w->p, 16) && w->stride % 8 == 0) return DGS_OK;
  DGS_REQUIRE(q.D % 8 != 0, DGS_ERR_INVALID, "linear_cross_entropy: rows of %lld 16-bit elements must begin at 16-byte boundaries",
              static_cast<long long>(q.D));
  uint16_t* packed = reinterpret_cast<uint16_t*>(q.ws + p.weight);
  const int64_t need = tiles(q.V * (p.pitch / 8), 256), most = static_cast<int64_t>(sm_count()) * 8;
  DGS_CUDA_TRY(launch_training(ce_pack_weight_kernel, dim3(static_cast<unsigned>(need < most ? need : most)), 256, 0, s, w->p,
                               q.weight_stride, q.V, static_cast<int>(q.D), static_cast<int>(p.pitch), packed));
  *w = Weight{packed, p.pitch};
  return DGS_OK;
}

}  // namespace

size_t ce_mma_forward_bytes(int64_t n, int64_t D, int64_t V) { return make_plan(n, D, V).forward_bytes; }
size_t ce_mma_backward_bytes(int64_t n, int64_t D, int64_t V) { return make_plan(n, D, V).backward_bytes; }

static CePacked packed_rows(const CeProblem& q, const MmaPlan& p) {
  CePacked r{};
  r.rows = q.ws + p.packed;
  r.pitch = p.pitch;
  r.word = reinterpret_cast<int32_t*>(q.ws + p.word);
  r.compact = p.compact;
  if (p.compact) {
    r.slot = reinterpret_cast<int32_t*>(q.ws + p.slot);
    r.live = reinterpret_cast<int32_t*>(q.ws + p.live);
    r.counts = reinterpret_cast<int32_t*>(q.ws + p.counts);
    r.block_rows = M_TILE;
    r.col_tiles = static_cast<int32_t>(p.col_tiles);
    r.slots = static_cast<int32_t>(p.pairs);
  }
  return r;
}

int ce_mma_forward(const CeProblem& q, float* loss, float* lse, cudaStream_t s) {
  const MmaPlan p = make_plan(q.n, q.D, q.V);
  CePacked r = packed_rows(q, p);
  // A row's statistics depend on that row alone: rows that TMA can fetch need no packing (what an ignored row holds ends there)
  const bool where_they_lie = !p.compact && aligned_to(q.hidden, 16) && (q.n == 1 ? q.D : q.hidden_stride) % 8 == 0;
  if (!where_they_lie) {
    if (int rc = ce_pack(q, r, nullptr, nullptr, nullptr, s)) return rc;
  }
  Weight w;
  if (int rc = fetchable_weight(q, p, &w, s)) return rc;
  MmaArgs a{};
  const bool narrow = !p.few && q.V <= NARROW_COLS;
  const void* rows = where_they_lie ? q.hidden : r.rows;
  const int64_t pitch = !where_they_lie ? p.pitch : q.n == 1 ? q.D : q.hidden_stride;
  if (int rc = make_map(p.few ? &a.b[0] : &a.a[0], rows, q.dtype, q.D, q.n, pitch, K_TILE, p.few ? FEW_ROWS / 2 : M_CTA)) return rc;
  if (int rc = make_map(p.few ? &a.a[0] : &a.b[0], w.p, q.dtype, q.D, q.V, w.stride, K_TILE, p.few ? M_CTA : narrow ? NARROW_COLS / 2 : N_TILE / 2))
    return rc;
  a.items = static_cast<int32_t>(p.row_blocks * p.slices);
  a.col_tiles = static_cast<int32_t>(p.col_tiles);
  a.slices = static_cast<int32_t>(p.slices);
  a.k_blocks = static_cast<int32_t>(tiles(q.D, K_TILE));
  a.n = q.n;
  a.V = q.V;
  a.live = r.live;
  a.word = where_they_lie ? nullptr : r.word;
  a.target = q.target;
  a.ids64 = q.ids64;
  a.ignore_index = q.ignore_index;
  a.target_logit = reinterpret_cast<float*>(q.ws + p.target_logit);
  a.top = reinterpret_cast<float*>(q.ws + p.top);
  a.total = reinterpret_cast<float*>(q.ws + p.total);
  a.status = q.status;
  const bool join_there = p.slices == 1 && !p.compact && !p.few;
  if (join_there) {
    a.loss_out = loss;
    a.lse_out = lse;
  }
  if (int rc = p.few    ? launch<FEW_STATS>(a, p.pairs, q.dtype, s)
               : narrow ? launch<NARROW>(a, p.pairs, q.dtype, s)
                        : launch<STATS>(a, p.pairs, q.dtype, s))
    return rc;
  if (join_there) return DGS_OK;
  return ce_join(q, a.top, a.total, p.few ? FEW_PARTS : COL_GROUPS, p.slices, p.few ? nullptr : r.live, a.word, r.slot, a.target_logit, loss, lse, s);
}

int ce_mma_backward(const CeProblem& q, const float* dloss, const float* lse, const float* loss, void* dhidden, void* dweight, cudaStream_t s) {
  const MmaPlan p = make_plan(q.n, q.D, q.V);
  CePacked r = packed_rows(q, p);
  r.dloss = reinterpret_cast<float*>(q.ws + p.dloss);
  r.lse = reinterpret_cast<float*>(q.ws + p.lse);
  r.largest = reinterpret_cast<float*>(q.ws + p.largest);
  r.hit = loss != nullptr ? reinterpret_cast<float*>(q.ws + p.hit) : nullptr;
  if (int rc = ce_pack(q, r, dloss, lse, loss, s)) return rc;
  const void* packed = r.rows;
  Weight w;
  if (int rc = fetchable_weight(q, p, &w, s)) return rc;
  uint16_t* g = reinterpret_cast<uint16_t*>(q.ws + p.g);
  float* dh = reinterpret_cast<float*>(q.ws + p.dh);
  // results whose rows begin at 16-byte boundaries leave by TMA
  const bool dh_direct = p.one_piece && p.splits == 1 && !p.compact, even = q.D % 8 == 0;
  for (int64_t v0 = 0; v0 < q.V; v0 += p.piece) {
    const int64_t width = q.V - v0 < p.piece ? q.V - v0 : p.piece;
    const uint16_t* wp = w.p + v0 * w.stride;
    MmaArgs a{};
    if (int rc = make_map(p.few ? &a.b[0] : &a.a[0], packed, q.dtype, q.D, q.n, p.pitch, K_TILE, p.few ? FEW_ROWS / 2 : M_CTA)) return rc;
    if (int rc = make_map(p.few ? &a.a[0] : &a.b[0], wp, q.dtype, q.D, width, w.stride, K_TILE, p.few ? M_CTA : N_TILE / 2)) return rc;
    if (int rc = make_map(&a.out[0], g, q.dtype, width, q.n, p.piece, 64, 32)) return rc;
    a.low = p.planes == 2 ? g + q.n * p.piece : nullptr;
    a.low_pitch = p.piece;
    a.g = g;
    a.col_tiles = static_cast<int32_t>(tiles(width, N_TILE));
    a.items = static_cast<int32_t>(p.row_blocks) * a.col_tiles;
    a.k_blocks = static_cast<int32_t>(tiles(q.D, K_TILE));
    a.n = q.n;
    a.V = width;
    a.v0 = static_cast<int32_t>(v0);
    a.live = r.live;
    a.word = r.word;
    a.dloss = r.dloss;
    a.lse = r.lse;
    a.hit = r.hit;
    a.largest = r.largest;
    a.largest_count = static_cast<int32_t>(ce_pack_ctas(q.n));
    a.status = q.status;
    if (int rc = p.few ? launch<FEW_GRAD>(a, p.pairs, q.dtype, s) : launch<GRAD>(a, p.pairs, q.dtype, s)) return rc;

    MmaArgs m{};
    // half as wide tiles where that gives more pairs something to do (1 024 rows of 256 against 172 classes: 5 tiles of 256)
    const int64_t wide = tiles(q.D, N_TILE) * (p.row_blocks * p.splits + tiles(width, M_TILE));
    const int32_t n_step = 2 * wide <= p.pairs ? N_TILE / 2 : N_TILE, d_tiles = static_cast<int32_t>(tiles(q.D, n_step));
    const bool dw_there = dweight != nullptr && !p.few_weight;
    const int both = dhidden != nullptr && dw_there, at_dh = both && !p.dh_first, at_dw = both && p.dh_first;
    int64_t dh_items = 0, dw_items = 0;
    if (dhidden != nullptr) {
      Part& t = m.part[at_dh];
      t.a_mn = 0;
      t.planes = static_cast<int32_t>(p.planes);
      t.plane_rows = static_cast<int32_t>(q.n);
      t.n_tiles = d_tiles;
      t.n_step = n_step;
      t.k_blocks = static_cast<int32_t>(tiles(width, K_TILE));
      // (the first piece has work for every split; a narrow last one adds to as many as it has)
      const int64_t k_all = p.planes * t.k_blocks;
      t.splits = static_cast<int32_t>(p.splits < k_all ? p.splits : k_all);
      dh_items = p.row_blocks * d_tiles * t.splits;
      t.n_total = static_cast<int32_t>(q.D);
      t.m_total = static_cast<int32_t>(q.n);
      t.split_rows = p.row_blocks * M_TILE;
      t.out_kind = !dh_direct ? (v0 > 0 ? OUT_F32_ADD : OUT_F32_STORE) : even && aligned_to(dhidden, 16) ? OUT_TYPED : OUT_TYPED_ODD;
      t.odd = dhidden;
      if (int rc = make_map(&m.a[at_dh], g, q.dtype, width, p.planes * q.n, p.piece, K_TILE, M_CTA)) return rc;
      if (int rc = make_map(&m.b[at_dh], wp, q.dtype, q.D, width, w.stride, 64, K_TILE)) return rc;
      if (t.out_kind == OUT_TYPED) {
        if (int rc = make_map(&m.out[at_dh], dhidden, q.dtype, q.D, q.n, q.D, 64, 32)) return rc;
      } else if (t.out_kind != OUT_TYPED_ODD) {
        if (int rc = make_map(&m.out[at_dh], dh, DGS_F32, q.D, p.splits * t.split_rows, p.dpitch, 32, 32)) return rc;
      }
    }
    if (dw_there) {
      Part& t = m.part[at_dw];
      t.a_mn = 1;
      t.planes = static_cast<int32_t>(p.planes);
      t.plane_rows = static_cast<int32_t>(q.n);
      t.n_tiles = d_tiles;
      t.n_step = n_step;
      t.splits = 1;
      t.k_blocks = static_cast<int32_t>(tiles(q.n, K_TILE));
      dw_items = tiles(width, M_TILE) * d_tiles;
      t.n_total = static_cast<int32_t>(q.D);
      t.m_total = static_cast<int32_t>(width);
      uint16_t* to = static_cast<uint16_t*>(dweight) + v0 * q.D;
      t.out_kind = even && aligned_to(dweight, 16) ? OUT_TYPED : OUT_TYPED_ODD;
      t.odd = to;
      if (int rc = make_map(&m.a[at_dw], g, q.dtype, width, p.planes * q.n, p.piece, 64, K_TILE)) return rc;
      if (int rc = make_map(&m.b[at_dw], packed, q.dtype, q.D, q.n, p.pitch, 64, K_TILE)) return rc;
      if (t.out_kind == OUT_TYPED) {
        if (int rc = make_map(&m.out[at_dw], to, q.dtype, q.D, width, q.D, 64, 32)) return rc;
      }
    }
    m.parts = 1 + both;
    m.items = static_cast<int32_t>(dh_items + dw_items);
    m.n = q.n;
    m.live = r.live;
    m.largest = r.largest;
    m.largest_count = a.largest_count;
    m.status = q.status;
    if (m.items > 0)
      if (int rc = launch<PRODUCT>(m, p.pairs, q.dtype, s)) return rc;
    if (dweight != nullptr && p.few_weight) {
      const FewWeightArgs f{static_cast<const uint16_t*>(packed), p.pitch, g, p.piece, static_cast<int32_t>(q.n),
                            static_cast<int32_t>(q.D), 0, width, static_cast<uint16_t*>(dweight) + v0 * q.D, r.largest, a.largest_count};
      if (int rc = q.dtype == DGS_BF16 ? few_weight<true>(f, s) : few_weight<false>(f, s)) return rc;
    }
  }
  if (dhidden != nullptr && !dh_direct) return ce_sum(dh, p.splits, q.n, q.D, p.row_blocks * M_TILE, p.dpitch, r.slot, dhidden, q.dtype, s);
  return DGS_OK;
}

}  // namespace dgs
