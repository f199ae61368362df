// Softmax attention of packed sequences: queries rows [q_offsets[s], q_offsets[s + 1]), keys and values rows of k_offsets; query head
// a reads key head a / (heads / kv_heads); with `causal` query i of Lq sees the keys j <= i + Lk - Lq.
//
//   x_ij = scale q_i.k_j,  lse_i = log sum_j exp x_ij,  p_ij = exp(x_ij - lse_i),  o_i = sum_j p_ij v_j    (no key: o = 0, lse = -inf)
//   dv_j = sum_i p_ij do_i,  e_ij = do_i.v_j,  delta_i = sum_j p_ij e_ij,  ds_ij = p_ij (e_ij - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i   (over all queries and heads that read j)
//
// This file: the plan of a call, and the rows of sequences with few queries (a seed over its sampled neighbours, a read-out over
// a graph) and of 32-bit operands, on the CUDA cores; sequences of ATTN_TILE_QUERIES queries and more in 16 bits (of fewer over many pairs,
// attn_in_tiles) are tiles on the tensor cores (attention_mma.cu).  Nothing is added by atomics: the same call gives the same bits.  How the
// lanes of a warp share a row follows from the call's keys a sequence on average, so in another batch a row's sums may have another order.
#include <type_traits>

#include "attention.h"

namespace dgs {
namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_ONE_CTA = 2048;  // sequences up to which one CTA makes the plan and clears its counts itself
constexpr int ROW_WARPS = 8;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ---- plan -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t offset_at(const void* p, int32_t wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Tiles in order of their work: a bucket for each quarter of a power of two of steps, the heaviest first
constexpr int PLAN_BUCKETS = 128;
__device__ __forceinline__ int bucket_of(int steps) {
  const int top = 31 - __clz(steps | 1), quarter = top >= 2 ? (steps >> (top - 2)) & 3 : 0;
  return PLAN_BUCKETS - 1 - (top * 4 + quarter);
}
__device__ __forceinline__ int tiles_of(int rows, int tile) { return (rows + tile - 1) / tile; }

// the n-th tile of queries (`rows` each), or of keys
__device__ __forceinline__ AttnTile query_tile(const AttnArgs& a, const AttnSeq& e, int n) {
  AttnTile t{};
  const int at = n * a.q_tile_rows;
  t.row = e.q0 + at;
  t.rows = min(a.q_tile_rows, e.q_len - at);
  t.other = e.k0;
  t.others = e.k_len;
  t.seen = a.causal ? at + 1 + e.k_len - e.q_len : e.k_len;
  const int last = a.causal ? min(e.k_len, t.seen + t.rows - 1) : e.k_len;
  t.steps = last > 0 ? tiles_of(last, ATTN_TILE) : 0;
  return t;
}
__device__ __forceinline__ AttnTile key_tile(const AttnArgs& a, const AttnSeq& e, int n) {
  AttnTile t{};
  const int at = n * ATTN_TILE, first = a.causal ? min(e.q_len, max(0, at - (e.k_len - e.q_len))) : 0;
  t.row = e.k0 + at;
  t.rows = min(ATTN_TILE, e.k_len - at);
  t.other = e.q0 + first;
  t.others = e.q_len - first;
  t.seen = a.causal ? at - (e.k_len - e.q_len) - first : INT32_MIN / 2;
  t.steps = tiles_of(t.others, ATTN_TILE);
  return t;
}

// A warp for each sequence: its place, whose its rows are, the parts of rows with many keys, the tiles of long ones.
__global__ __launch_bounds__(PLAN_THREADS) void attn_plan_kernel(const __grid_constant__ AttnArgs a, int32_t backward, int32_t alone) {
  __shared__ int bucket[2][PLAN_BUCKETS];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (alone && blockIdx.x == 0) {
    if (threadIdx.x < ATTN_COUNTS) a.counts[threadIdx.x] = 0;
    if (threadIdx.x < 2) a.norms[threadIdx.x] = 0.0f;
    if (threadIdx.x < 2 * PLAN_BUCKETS) bucket[threadIdx.x / PLAN_BUCKETS][threadIdx.x % PLAN_BUCKETS] = 0;
    __syncthreads();
  }
  // Where one CTA makes the lists, the others write whose the rows are.  Each warp reads the offsets of up to 32 sequences at once and then
  // takes them in turn.
  const bool lists = !alone || blockIdx.x == 0, maps = !alone || blockIdx.x > 0;
  const int ctas = alone ? (lists ? 1 : gridDim.x - 1) : gridDim.x, cta = alone && !lists ? blockIdx.x - 1 : blockIdx.x;
  const int warps = ctas * (PLAN_THREADS / 32), batch = min(32, (a.seqs + warps - 1) / warps);
  int tiles = 0, single = 0, several = 0;  // sequences of each kind
  for (int s0 = (cta * (PLAN_THREADS / 32) + warp) * batch; s0 < a.seqs; s0 += warps * batch) {
    const int mine = s0 + lane;
    AttnSeq own{0, 0, 0, 0};
    if (lane < batch && mine < a.seqs) {
      const int64_t q0 = offset_at(a.q_offsets, a.offsets64, mine), q1 = offset_at(a.q_offsets, a.offsets64, mine + 1);
      const int64_t k0 = offset_at(a.k_offsets, a.offsets64, mine), k1 = offset_at(a.k_offsets, a.offsets64, mine + 1);
      if (q0 >= 0 && q0 <= q1 && q1 <= a.n_q && k0 >= 0 && k0 <= k1 && k1 <= a.n_k)
        own = {static_cast<int32_t>(q0), static_cast<int32_t>(q1 - q0), static_cast<int32_t>(k0), static_cast<int32_t>(k1 - k0)};
      else
        raise_status(a.status, DGS_ERR_RANGE), several = 1;
      if (lists) a.seq[mine] = own;
      if (attn_in_tiles(a, own)) tiles = 1;
      else if (attn_is_single(a, own)) single = 1;
      else several = 1;
    }
    for (int n = 0; n < batch && s0 + n < a.seqs; ++n) {
      const int s = s0 + n;
      const AttnSeq e{__shfl_sync(FULL_MASK, own.q0, n), __shfl_sync(FULL_MASK, own.q_len, n), __shfl_sync(FULL_MASK, own.k0, n),
                      __shfl_sync(FULL_MASK, own.k_len, n)};
      if (maps) {
        for (int i = lane; i < e.q_len; i += 32) a.q_seq[e.q0 + i] = s;
        if (backward)
          for (int i = lane; i < e.k_len; i += 32) a.k_seq[e.k0 + i] = s;
        if (!lists) continue;
      }
      if (attn_in_tiles(a, e)) {
        const int nq = tiles_of(e.q_len, a.q_tile_rows), nk = backward ? tiles_of(e.k_len, ATTN_TILE) : 0;
        if (alone) {  // counted first, placed below
          for (int i = lane; i < nq; i += 32) atomicAdd(&bucket[0][bucket_of(query_tile(a, e, i).steps)], 1);
          for (int i = lane; i < nk; i += 32) atomicAdd(&bucket[1][bucket_of(key_tile(a, e, i).steps)], 1);
          continue;
        }
        int at[2] = {0, 0};
        if (lane < 2) at[0] = atomicAdd(&a.counts[lane ? ATTN_N_K_TILES : ATTN_N_Q_TILES], lane ? nk : nq);
        at[1] = __shfl_sync(FULL_MASK, at[0], 1);
        at[0] = __shfl_sync(FULL_MASK, at[0], 0);
        // (the bounds are of the sizes; offsets that overlap may get beyond them)
        for (int i = lane; i < nq && at[0] + i < a.q_tile_bound; i += 32) a.q_tiles[at[0] + i] = query_tile(a, e, i);
        for (int i = lane; i < nk && at[1] + i < a.k_tile_bound; i += 32) a.k_tiles[at[1] + i] = key_tile(a, e, i);
      } else if (attn_is_split(a, e) && e.q_len > 0) {
        const int parts = (e.k_len + ATTN_SPLIT_KEYS - 1) / ATTN_SPLIT_KEYS, all = parts * e.q_len;
        int first = 0;
        if (lane == 0) first = atomicAdd(&a.counts[ATTN_N_SPLITS], all);
        first = __shfl_sync(FULL_MASK, first, 0);
        for (int i = lane; i < all; i += 32) {
          const int row = i / parts, part = i - row * parts;
          if (first + i >= a.split_bound) break;
          a.splits[first + i] = make_int4(e.q0 + row, part * ATTN_SPLIT_KEYS, first + row * parts, parts);
          for (int c = 0; c < a.kv_heads; ++c) a.arrived[static_cast<int64_t>(first + i) * a.kv_heads + c] = 0;
        }
      }
    }
  }
  if (!lists) return;
  // which kinds there are: kernels for the others leave at once
  const unsigned kinds = __reduce_or_sync(FULL_MASK, (tiles ? 1u << ATTN_HAS_TILES : 0u) | (single ? 1u << ATTN_HAS_SINGLE : 0u) | (several ? 1u << ATTN_HAS_SEVERAL : 0u));
  if (lane == 0 && kinds != 0) atomicOr(&a.counts[ATTN_KINDS], static_cast<int>(kinds));
  if (!alone || !a.tiles) return;
  __syncthreads();
  if (warp < 2) {  // where each bucket begins
    int carry = 0;
    for (int b = lane; b < PLAN_BUCKETS; b += 32) {
      const int n = bucket[warp][b];
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(FULL_MASK, sum, o);
        if (lane >= o) sum += up;
      }
      bucket[warp][b] = carry + sum - n;
      carry += __shfl_sync(FULL_MASK, sum, 31);
    }
    if (lane == 0) a.counts[warp ? ATTN_N_K_TILES : ATTN_N_Q_TILES] = carry;
  }
  __syncthreads();
  for (int s0 = warp * batch; s0 < a.seqs; s0 += warps * batch) {
    AttnSeq own{0, 0, 0, 0};
    if (lane < batch && s0 + lane < a.seqs) own = a.seq[s0 + lane];
    for (unsigned todo = __ballot_sync(FULL_MASK, attn_in_tiles(a, own)); todo != 0; todo &= todo - 1) {
      const int n = __ffs(todo) - 1;
      const AttnSeq e{__shfl_sync(FULL_MASK, own.q0, n), __shfl_sync(FULL_MASK, own.q_len, n), __shfl_sync(FULL_MASK, own.k0, n),
                      __shfl_sync(FULL_MASK, own.k_len, n)};
      for (int i = lane; i < tiles_of(e.q_len, a.q_tile_rows); i += 32) {
        const AttnTile t = query_tile(a, e, i);
        const int at = atomicAdd(&bucket[0][bucket_of(t.steps)], 1);
        if (at < a.q_tile_bound) a.q_tiles[at] = t;
      }
      if (!backward) continue;
      for (int i = lane; i < tiles_of(e.k_len, ATTN_TILE); i += 32) {
        const AttnTile t = key_tile(a, e, i);
        const int at = atomicAdd(&bucket[1][bucket_of(t.steps)], 1);
        if (at < a.k_tile_bound) a.k_tiles[at] = t;
      }
    }
  }
}

__device__ __forceinline__ float ex2(float x) {  // exp2 within two units in the last place, results below 2^-126 flushed to 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---- rows ------------------------------------------------------------------------------------------------------------
// A row of DP elements lies in G lanes, VEC elements each.  A warp holds 32 / G of them side by side: `side` key heads of one key (which
// lie side by side in memory too), and where there are fewer heads than that, several keys.
template <typename T>
constexpr int vec_of() {
  return 16 / static_cast<int>(sizeof(T));
}
template <typename T, int DP>
constexpr int lanes_of() {
  return DP / vec_of<T>();
}

template <typename T, int DP>
struct Lanes {
  static constexpr int G = lanes_of<T, DP>(), SLOTS = 32 / G;
  int side, blocks;          // key heads side by side, and how many times as many there are
  int vec, head, key, keys;  // this lane's elements, its head of those side by side, its key; keys at once
  bool in_d;
  __device__ __forceinline__ Lanes(const AttnArgs& a, int heads_side_by_side) : side(heads_side_by_side) {
    const int lane = threadIdx.x & 31, slot = lane / G;
    blocks = (a.kv_heads + side - 1) / side;
    vec = lane % G;
    head = slot & (side - 1);
    key = slot / side;
    keys = SLOTS / side;
    in_d = vec * vec_of<T>() < a.d;
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void load_row(const T* p, bool there, float (&v)[VEC]) {
  if (there) {
    load_vec<T, VEC>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
  }
}
// two elements an instruction
template <int VEC>
__device__ __forceinline__ float dot(const float (&a)[VEC], const float (&b)[VEC]) {
  uint64_t s = mul2(two(a[0], a[1]), two(b[0], b[1]));
#pragma unroll
  for (int e = 2; e < VEC; e += 2) s = fma2(two(a[e], a[e + 1]), two(b[e], b[e + 1]), s);
  float lo, hi;
  split2(s, &lo, &hi);
  return lo + hi;
}
template <int VEC>
__device__ __forceinline__ void add_scaled(float by, const float (&x)[VEC], float (&sum)[VEC]) {
  const uint64_t by2 = two(by, by);
#pragma unroll
  for (int e = 0; e < VEC; e += 2) split2(fma2(by2, two(x[e], x[e + 1]), two(sum[e], sum[e + 1])), &sum[e], &sum[e + 1]);
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  return v;
}

// Keys j0, j0 + step, .. (U times as many as lie side by side at once) of one row: running maximum (of log2 values), sum and weighted values
// of R heads.
template <typename T, int DP, int R, int U>
__device__ __forceinline__ void forward_keys(const T* k, int64_t k_row, const T* v, int64_t v_row, int j0, int j1, int step, const Lanes<T, DP>& w,
                                             bool in, const float (&q)[R][vec_of<T>()], float (&m)[R], float (&l)[R], float (&acc)[R][vec_of<T>()]) {
  constexpr int VEC = vec_of<T>(), G = lanes_of<T, DP>();
  for (int j = j0; j < j1; j += step) {
    Vec<T, VEC> kr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = j + u * w.keys + w.key;
      const bool there = at < j1 && in;
      kr[u] = there ? *reinterpret_cast<const Vec<T, VEC>*>(k + at * k_row) : Vec<T, VEC>{};
      vr[u] = there ? *reinterpret_cast<const Vec<T, VEC>*>(v + at * v_row) : Vec<T, VEC>{};
    }
    float x[R][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) kf[e] = to_float<T>(kr[u].v[e]);
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][u] = group_sum<G>(dot<VEC>(q[r], kf));
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j + u * w.keys + w.key >= j1) x[r][u] = -INFINITY;
        top = fmaxf(top, x[r][u]);
      }
      const float ref = top == -INFINITY ? 0.0f : top, scale = ex2(m[r] - ref);
      m[r] = top;
      l[r] *= scale;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[r][u] = ex2(x[r][u] - ref);
        l[r] += x[r][u];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[r][e] *= scale;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float vf[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) vf[e] = to_float<T>(vr[u].v[e]);
#pragma unroll
      for (int r = 0; r < R; ++r) add_scaled<VEC>(x[r][u], vf, acc[r]);
    }
  }
}

// the lanes that hold the same elements of other keys joined: (m, l, acc) each
template <int VEC>
__device__ __forceinline__ void join_keys(int first, float& m, float& l, float (&acc)[VEC]) {
  for (int o = first; o < 32; o <<= 1) {
    const float m2 = __shfl_xor_sync(FULL_MASK, m, o), l2 = __shfl_xor_sync(FULL_MASK, l, o);
    const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top;
    const float s1 = ex2(m - ref), s2 = ex2(m2 - ref);
    l = l * s1 + l2 * s2;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = acc[e] * s1 + __shfl_xor_sync(FULL_MASK, acc[e], o) * s2;
    m = top;
  }
}
template <int VEC>
__device__ __forceinline__ void add_keys(int first, float (&v)[VEC]) {
  for (int o = first; o < 32; o <<= 1)
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] += __shfl_xor_sync(FULL_MASK, v[e], o);
}

// The sequence of a row, or none (a row outside of all of them); again: the tiles left the row to be made again
__device__ __forceinline__ AttnSeq sequence_of(const AttnArgs& a, const int32_t* map, int row, bool key, bool* found, bool* again) {
  const int word = map[row], s = word & ~ATTN_AGAIN;
  AttnSeq e{0, 0, 0, 0};
  *found = false;
  *again = (word & ATTN_AGAIN) != 0;
  if (s < a.seqs) {
    e = a.seq[s];
    const int at = row - (key ? e.k0 : e.q0);
    *found = at >= 0 && at < (key ? e.k_len : e.q_len);
  }
  return e;
}

// keys that a query sees
__device__ __forceinline__ int keys_seen(const AttnArgs& a, const AttnSeq& e, int row) {
  if (!a.causal) return e.k_len;
  const int n = row - e.q0 + 1 + e.k_len - e.q_len;
  return n < 0 ? 0 : n < e.k_len ? n : e.k_len;
}

template <typename T, int R>
__device__ __forceinline__ void load_heads(const AttnView& x, int row, int head0, int heads, int vec, bool in, float by, float (&q)[R][vec_of<T>()]) {
  constexpr int VEC = vec_of<T>();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    load_row<T, VEC>(static_cast<const T*>(x.p) + row * x.row + (head0 + r) * x.head + vec * VEC, in && r < heads, q[r]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) q[r][e] *= by;
  }
}

// Rows that a kernel looks at: all, or, where every sequence is another kernel's, those outside of all sequences.
struct Range {
  int rows, skip_at, skip;
  __device__ __forceinline__ int row(int i) const { return i < skip_at ? i : i + skip; }
};
__device__ __forceinline__ Range range_of(const AttnArgs& a, bool key) {
  const int n = key ? a.n_k : a.n_q;
  if (a.seqs == 0 || (a.counts[ATTN_KINDS] & (1 << ATTN_HAS_SEVERAL | 1 << ATTN_HAS_AGAIN)) != 0) return {n, n, 0};
  // (the plan found all offsets in order)
  const void* p = key ? a.k_offsets : a.q_offsets;
  const int first = static_cast<int>(offset_at(p, a.offsets64, 0)), skip = static_cast<int>(offset_at(p, a.offsets64, a.seqs)) - first;
  return {n - skip, first, skip};
}

// Rows a.rows_at_once at a time: whose they are is looked up side by side, a lane a row; `f` gets those that `mine` names, one after another.
template <typename Mine, typename F>
__device__ __forceinline__ void each_row(const AttnArgs& a, int64_t task, int64_t tasks_step, const Range& range, int blocks, const int32_t* map,
                                         bool key, const Mine& mine, const F& f) {
  const int lane = threadIdx.x & 31, rows = range.rows;
  const int64_t all = static_cast<int64_t>((rows + a.rows_at_once - 1) / a.rows_at_once) * blocks;
  for (; task < all; task += tasks_step) {
    const int batch = static_cast<int>(task / blocks), block = static_cast<int>(task - static_cast<int64_t>(batch) * blocks);
    const int at = batch * a.rows_at_once + lane;
    bool found = false, take = false, again;
    AttnSeq e{0, 0, 0, 0};
    if (lane < a.rows_at_once && at < rows) {
      e = sequence_of(a, map, range.row(at), key, &found, &again);
      take = mine(e, found, again);
    }
    if (!found) e = AttnSeq{0, 0, 0, 0};
    for (unsigned todo = __ballot_sync(FULL_MASK, take); todo != 0; todo &= todo - 1) {
      const int n = __ffs(todo) - 1;
      const AttnSeq x{__shfl_sync(FULL_MASK, e.q0, n), __shfl_sync(FULL_MASK, e.q_len, n), __shfl_sync(FULL_MASK, e.k0, n),
                      __shfl_sync(FULL_MASK, e.k_len, n)};
      f(range.row(batch * a.rows_at_once + n), block, x);
    }
  }
}

// What a CTA's warps found of a row's part, one head side by side after another: [warp][head][DP values, ..]
template <typename T, int DP, int FLOATS>
struct Shared {
  float v[ROW_WARPS][Lanes<T, DP>::SLOTS][FLOATS];
};

// the last part of a row to be there: true for the CTA that takes all of them
__device__ __forceinline__ bool last_part(const AttnArgs& a, const int4& it, int block, bool* flag) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    *flag = atomicAdd(&a.arrived[static_cast<int64_t>(it.z) * a.kv_heads + block], 1u) + 1 == static_cast<uint32_t>(it.w);
  __syncthreads();
  const bool last = *flag;
  if (last) __threadfence();
  return last;
}

// Forward.  Rows with up to ATTN_SPLIT_FROM keys: a warp each, for all the key heads side by side.  SPLIT: CTAs take the parts of rows with
// many keys; the last part of a row to be there joins them in their order.  Bound by HBM where every query has keys of its own: what is
// under way is many warps with few keys each for short rows (60 000 seeds of 7.5 keys: 144 us with 32 warps an SM and two keys against 169 with
// 16 and four when that was chosen, 127 now), more keys a warp for long ones.
template <typename T, int DP, int R, bool SPLIT>
__global__ __launch_bounds__(ROW_WARPS * 32, R == 1 && !SPLIT ? 4 : 2) void attn_rows_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int VEC = vec_of<T>(), G = lanes_of<T, DP>(), U = R == 2 ? 4 : 2, SPLIT_U = R == 1 ? 4 : 2;
  pdl_enter();
  const int warp = threadIdx.x >> 5, group = a.heads / a.kv_heads;
  const Lanes<T, DP> w(a, SPLIT ? a.split_side : a.side);
  const int blocks = w.blocks;
  if constexpr (SPLIT) {
    __shared__ Shared<T, DP, DP + 2> shared;
    __shared__ bool flag;
    const int split_ctas = gridDim.x;
    const int floats = a.d + 2, n = min(a.counts[ATTN_N_SPLITS], a.split_bound);
    for (int64_t t = blockIdx.x; t < static_cast<int64_t>(n) * blocks; t += split_ctas) {
      const int item = static_cast<int>(t / blocks), block = static_cast<int>(t - static_cast<int64_t>(item) * blocks);
      const int4 it = a.splits[item];
      bool found, again;
      const AttnSeq e = sequence_of(a, a.q_seq, it.x, false, &found, &again);
      const int c = block * w.side + w.head, j0 = it.y, j1 = min(found ? keys_seen(a, e, it.x) : 0, j0 + ATTN_SPLIT_KEYS);
      const bool in = w.in_d && c < a.kv_heads;
      const T* k = static_cast<const T*>(a.k.p) + e.k0 * a.k.row + c * a.k.head + w.vec * VEC;
      const T* v = static_cast<const T*>(a.v.p) + e.k0 * a.v.row + c * a.v.head + w.vec * VEC;
      for (int h0 = 0; h0 < group; h0 += R) {
        const int heads = min(R, group - h0);
        float q[R][VEC], m[R], l[R], acc[R][VEC];
        load_heads<T, R>(a.q, it.x, c * group + h0, heads, w.vec, in, a.scale * LOG2E, q);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          m[r] = -INFINITY;
          l[r] = 0.0f;
#pragma unroll
          for (int x = 0; x < VEC; ++x) acc[r][x] = 0.0f;
        }
        forward_keys<T, DP, R, SPLIT_U>(k, a.k.row, v, a.v.row, j0 + warp * w.keys * SPLIT_U, j1, ROW_WARPS * w.keys * SPLIT_U, w, in, q, m, l, acc);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          join_keys<VEC>(w.side * G, m[r], l[r], acc[r]);
          if (r >= heads) continue;  // (the same for all threads)
          __syncthreads();           // `shared` may be written again
          if (w.key == 0) {
            float* to = shared.v[warp][w.head];
#pragma unroll
            for (int x = 0; x < VEC; ++x) to[w.vec * VEC + x] = acc[r][x];
            if (w.vec == 0) to[DP] = m[r], to[DP + 1] = l[r];
          }
          __syncthreads();
          // the warps' parts, an element a thread
          for (int i = threadIdx.x; i < w.side * (a.d + 1); i += ROW_WARPS * 32) {
            const int hs = i / (a.d + 1), x = i - hs * (a.d + 1), at = x < a.d ? x : DP + 1, kv = block * w.side + hs;
            if (kv >= a.kv_heads) continue;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int y = 0; y < ROW_WARPS; ++y) top = fmaxf(top, shared.v[y][hs][DP]);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int y = 0; y < ROW_WARPS; ++y) sum += shared.v[y][hs][at] * ex2(shared.v[y][hs][DP] - ref);
            float* part = a.parts + (static_cast<int64_t>(item) * a.heads + kv * group + h0 + r) * floats;
            part[x < a.d ? x : a.d + 1] = sum;
            if (x == 0) part[a.d] = top;
          }
        }
      }
      if (last_part(a, it, block, &flag) && found) {
        const int lane = threadIdx.x & 31, first = block * w.side * group, all = min(a.heads - first, w.side * group);
        for (int h = warp; h < all; h += ROW_WARPS) {
          const int head = first + h;
          const float* part = a.parts + (static_cast<int64_t>(it.z) * a.heads + head) * floats;
          const int64_t apart = static_cast<int64_t>(a.heads) * floats;
          float top = -INFINITY;
          for (int p = lane; p < it.w; p += 32) top = fmaxf(top, __ldcg(part + p * apart + a.d));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
          const float ref = top == -INFINITY ? 0.0f : top;
          float l = 0.0f, acc[DP / 32];
#pragma unroll
          for (int x = 0; x < DP / 32; ++x) acc[x] = 0.0f;
#pragma unroll 4
          for (int p = 0; p < it.w; ++p) {
            const float by = ex2(__ldcg(part + p * apart + a.d) - ref);
            l += __ldcg(part + p * apart + a.d + 1) * by;
#pragma unroll
            for (int x = 0; x < DP / 32; ++x)
              if (x * 32 + lane < a.d) acc[x] += __ldcg(part + p * apart + x * 32 + lane) * by;
          }
          const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // (nan stays nan)
#pragma unroll
          for (int x = 0; x < DP / 32; ++x)
            if (x * 32 + lane < a.d)
              static_cast<T*>(a.out)[(static_cast<int64_t>(it.x) * a.heads + head) * a.d + x * 32 + lane] = from_float<T>(acc[x] * inv);
          if (lane == 0) a.lse[static_cast<int64_t>(head) * a.n_q + it.x] = l == 0.0f ? -INFINITY : (top + log2f(l)) * LN2;
        }
      }
      __syncthreads();  // `flag` may be written again
    }
    return;
  }
  each_row(
      a, static_cast<int64_t>(blockIdx.x) * ROW_WARPS + warp, static_cast<int64_t>(gridDim.x) * ROW_WARPS, Range{a.n_q, a.n_q, 0}, blocks, a.q_seq, false,
      [&](const AttnSeq& e, bool found, bool again) { return !found || again || !(attn_in_tiles(a, e) || attn_is_split(a, e)); },
      [&](int row, int block, const AttnSeq& e) {
        const int seen = keys_seen(a, e, row), c = block * w.side + w.head;
        const bool in = w.in_d && c < a.kv_heads;
        const T* k = static_cast<const T*>(a.k.p) + e.k0 * a.k.row + c * a.k.head + w.vec * VEC;
        const T* v = static_cast<const T*>(a.v.p) + e.k0 * a.v.row + c * a.v.head + w.vec * VEC;
        for (int h0 = 0; h0 < group; h0 += R) {
          const int heads = min(R, group - h0);
          float q[R][VEC], m[R], l[R], acc[R][VEC];
          load_heads<T, R>(a.q, row, c * group + h0, heads, w.vec, in && seen > 0, a.scale * LOG2E, q);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[r][x] = 0.0f;
          }
          forward_keys<T, DP, R, U>(k, a.k.row, v, a.v.row, 0, seen, w.keys * U, w, in, q, m, l, acc);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            join_keys<VEC>(w.side * G, m[r], l[r], acc[r]);
            if (!(w.key == 0 && in && r < heads)) continue;
            const int head = c * group + h0 + r;
            const float inv = l[r] > 0.0f ? 1.0f / l[r] : (l[r] == 0.0f ? 0.0f : l[r]);
            float o[VEC];
#pragma unroll
            for (int x = 0; x < VEC; ++x) o[x] = acc[r][x] * inv;
            store_vec<T, VEC>(static_cast<T*>(a.out) + (static_cast<int64_t>(row) * a.heads + head) * a.d + w.vec * VEC, o);
            if (w.vec == 0) a.lse[static_cast<int64_t>(head) * a.n_q + row] = l[r] == 0.0f ? -INFINITY : (m[r] + log2f(l[r])) * LN2;
          }
        }
      });
}

// ---- backward --------------------------------------------------------------------------------------------------------
// log2-sum-exp of a row; a row that had no finite score has no weights
__device__ __forceinline__ float reference_of(const AttnArgs& a, int head, int row, bool there) {
  const float lse = there ? a.lse[static_cast<int64_t>(head) * a.n_q + row] * LOG2E : 0.0f;
  return lse == -INFINITY ? INFINITY : lse;
}

// Sequences of one query and few keys (a seed over its neighbours): nobody else reads these keys, so a warp a query gives all three
// gradients.  delta = sum_j p_j e_j of values in 32 bits has to be there before the first slope, so the keys are gone over twice: for dv and
// delta, then for dk.  (do.o of an `out` rounded to 16 bits, which would be there at once, is off most where few keys are averaged: it left dq of two
// keys 1.95 times as far off as rounding the exact one does, 2 to 6 times where v and do have a common mean.)  Weights and e are held in
// shared memory in between, HELD / side / R keys of them, all that most rows have; others, and those of three and four heads (which a bound of 128
// registers leaves little room), are made again.  ONCE: dq = scale (sum p e k - delta sum p k) out of the first pass, else out of the second, which
// reads K again.  Bound by HBM and by what is under way.  Backward calls, us, 60 000 seeds of up to 15 keys, 4 heads of 64: bfloat16 299, float16 308,
// float32 416; 2 key heads 240; 5 000 of 100 to 400 keys, 8 heads: bfloat16 1 042 (1 302 without ONCE), float32 2 217.
template <typename T, int DP, int R>
__global__ __launch_bounds__(ROW_WARPS * 32, R == 1 ? 3 : 2) void attn_single_backward_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int VEC = vec_of<T>(), G = lanes_of<T, DP>(), U = 2, SLOTS = Lanes<T, DP>::SLOTS;
  constexpr bool ONCE = R == 2 || (R == 1 && sizeof(T) == 2);
  constexpr int HELD = R <= 2 ? 512 : 1, HELD_STEPS = R <= 2 ? HELD / (U * SLOTS * R) : 0;
  __shared__ float2 held[ROW_WARPS][HELD];
  pdl_enter();
  if ((a.counts[ATTN_KINDS] >> ATTN_HAS_SINGLE & 1) == 0) return;
  const int warp = threadIdx.x >> 5, group = a.heads / a.kv_heads, blocks = (a.kv_heads + a.side - 1) / a.side;
  const Lanes<T, DP> w(a, a.side);
  float2* const mine = held[warp] + (threadIdx.x & 31) / G * R;
  each_row(
      a, static_cast<int64_t>(blockIdx.x) * ROW_WARPS + warp, static_cast<int64_t>(gridDim.x) * ROW_WARPS, Range{a.n_q, a.n_q, 0}, blocks,
      a.q_seq, false,
      [&](const AttnSeq& e, bool found, bool) { return found && !attn_in_tiles(a, e) && attn_is_single(a, e); },
      [&](int row, int block, const AttnSeq& e) {
        const int seen = e.k_len, c = block * w.side + w.head;  // (the one query sees all keys, causal or not)
        const bool in = w.in_d && c < a.kv_heads;
        const T* k = static_cast<const T*>(a.k.p) + e.k0 * a.k.row + c * a.k.head + w.vec * VEC;
        const T* v = static_cast<const T*>(a.v.p) + e.k0 * a.v.row + c * a.v.head + w.vec * VEC;
        const int64_t to = (static_cast<int64_t>(e.k0) * a.kv_heads + c) * a.d + w.vec * VEC, to_row = static_cast<int64_t>(a.kv_heads) * a.d;
        float q[R][VEC], g[R][VEC], ref[R], delta[R], dq[R][VEC], pk[ONCE ? R : 1][VEC];
        load_heads<T, R>(a.q, row, c * group, group, w.vec, in && seen > 0, 1.0f, q);
        load_heads<T, R>(a.dout, row, c * group, group, w.vec, in && seen > 0, 1.0f, g);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          ref[r] = reference_of(a, c * group + r, row, in && seen > 0 && r < group);
          delta[r] = 0.0f;
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            dq[r][x] = 0.0f;
            if (ONCE) pk[r][x] = 0.0f;
          }
        }
        const auto rows_of = [&](const T* p, int64_t p_row, int j, Vec<T, VEC> (&x)[U]) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int at = j + u * w.keys + w.key;
            x[u] = at < seen && in ? *reinterpret_cast<const Vec<T, VEC>*>(p + at * p_row) : Vec<T, VEC>{};
          }
        };
        const auto floats_of = [&](const Vec<T, VEC>& x, float (&f)[VEC]) {
          if constexpr (R == 1 && sizeof(T) == 2) {  // (kept in their place: moved ahead of one another they take more registers than there are)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(&x.v[i]);
              if constexpr (std::is_same_v<T, __half>) {
                asm volatile("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
                             : "=f"(f[i]), "=f"(f[i + 1])
                             : "r"(w));
              } else {
                uint32_t lo, hi;
                asm volatile("shl.b32 %0, %2, 16;\n\tand.b32 %1, %2, 0xffff0000;" : "=r"(lo), "=r"(hi) : "r"(w));
                f[i] = __uint_as_float(lo), f[i + 1] = __uint_as_float(hi);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = to_float<T>(x.v[i]);
          }
        };
        // a weight and e = do.v
        const auto pair = [&](int r, int at, const float (&kf)[VEC], const float (&vf)[VEC]) {
          const float x = group_sum<G>(dot<VEC>(q[r], kf)) * (a.scale * LOG2E), y = group_sum<G>(dot<VEC>(g[r], vf));
          return make_float2(at < seen && r < group ? ex2(x - ref[r]) : 0.0f, y);
        };
        __syncwarp();  // (the row before has read what it held)
        for (int j = 0, step = 0; j < seen; j += w.keys * U, ++step) {
          Vec<T, VEC> kr[U], vr[U];
          rows_of(k, a.k.row, j, kr);
          rows_of(v, a.v.row, j, vr);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int at = j + u * w.keys + w.key;
            float kf[VEC], vf[VEC], dv[VEC];
            floats_of(kr[u], kf);
            floats_of(vr[u], vf);
#pragma unroll
            for (int x = 0; x < VEC; ++x) dv[x] = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              const float2 pe = pair(r, at, kf, vf);
              delta[r] = fmaf(pe.x, pe.y, delta[r]);
              add_scaled<VEC>(pe.x, g[r], dv);
              if constexpr (ONCE) {
                add_scaled<VEC>(pe.x * pe.y, kf, dq[r]);
                add_scaled<VEC>(pe.x, kf, pk[r]);
              }
              if (HELD_STEPS > 0 && w.vec == 0 && step < HELD_STEPS) mine[(step * U + u) * SLOTS * R + r] = pe;
            }
            if (a.dk != nullptr && at < seen && in) store_vec<T, VEC>(static_cast<T*>(a.dv) + to + at * to_row, dv);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float one[1] = {delta[r]};
          add_keys<1>(w.side * G, one);
          delta[r] = one[0];
        }
        __syncwarp();
        if (!ONCE || a.dk != nullptr) {
          for (int j = 0, step = 0; j < seen; j += w.keys * U, ++step) {
            Vec<T, VEC> kr[U], vr[U];
            const bool again = HELD_STEPS == 0 || step >= HELD_STEPS;
            if (!ONCE || again) rows_of(k, a.k.row, j, kr);
            if (again) rows_of(v, a.v.row, j, vr);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int at = j + u * w.keys + w.key;
              float kf[VEC], dk[VEC];
              if (!ONCE || again) floats_of(kr[u], kf);
#pragma unroll
              for (int x = 0; x < VEC; ++x) dk[x] = 0.0f;
#pragma unroll
              for (int r = 0; r < R; ++r) {
                float2 pe;
                if (again) {
                  float vf[VEC];
                  floats_of(vr[u], vf);
                  pe = pair(r, at, kf, vf);
                } else {
                  pe = mine[(step * U + u) * SLOTS * R + r];
                }
                const float ds = pe.x * (pe.y - delta[r]) * a.scale;
                add_scaled<VEC>(ds, q[r], dk);
                if constexpr (!ONCE) add_scaled<VEC>(ds, kf, dq[r]);
              }
              if (a.dk != nullptr && at < seen && in) store_vec<T, VEC>(static_cast<T*>(a.dk) + to + at * to_row, dk);
            }
          }
        }
        if (a.dq == nullptr) return;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if constexpr (ONCE) {
#pragma unroll
            for (int x = 0; x < VEC; ++x) dq[r][x] = a.scale * fmaf(-delta[r], pk[r][x], dq[r][x]);
          }
          add_keys<VEC>(w.side * G, dq[r]);
          if (w.key == 0 && in && r < group)
            store_vec<T, VEC>(static_cast<T*>(a.dq) + (static_cast<int64_t>(row) * a.heads + c * group + r) * a.d + w.vec * VEC, dq[r]);
        }
      });
}

// Over some keys of one row, for R heads: sum p e k, sum p k (so that dq = scale (the first - delta times the second) takes one pass) and
// sum p e = delta.
template <typename T, int DP, int R>
__device__ __forceinline__ void backward_keys(const T* k, int64_t k_row, const T* v, int64_t v_row, int j0, int j1, int step, const Lanes<T, DP>& w,
                                              bool in, const float (&q)[R][vec_of<T>()], const float (&g)[R][vec_of<T>()], const float (&ref)[R],
                                              float (&pek)[R][vec_of<T>()], float (&pk)[R][vec_of<T>()], float (&delta)[R]) {
  constexpr int VEC = vec_of<T>(), G = lanes_of<T, DP>(), U = 2;
  for (int j = j0; j < j1; j += step) {
    Vec<T, VEC> kr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = j + u * w.keys + w.key;
      const bool there = at < j1 && in;
      kr[u] = there ? *reinterpret_cast<const Vec<T, VEC>*>(k + at * k_row) : Vec<T, VEC>{};
      vr[u] = there ? *reinterpret_cast<const Vec<T, VEC>*>(v + at * v_row) : Vec<T, VEC>{};
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[VEC], vf[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        kf[e] = to_float<T>(kr[u].v[e]);
        vf[e] = to_float<T>(vr[u].v[e]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float x = group_sum<G>(dot<VEC>(q[r], kf)), e = group_sum<G>(dot<VEC>(g[r], vf));
        const float p = j + u * w.keys + w.key < j1 ? ex2(x - ref[r]) : 0.0f;
        delta[r] = fmaf(p, e, delta[r]);
        add_scaled<VEC>(p * e, kf, pek[r]);
        add_scaled<VEC>(p, kf, pk[r]);
      }
    }
  }
}

// dq and delta of the rows of other sequences, in the shape of attn_rows_kernel
template <typename T, int DP, int R, bool SPLIT>
__global__ __launch_bounds__(ROW_WARPS * 32, 2) void attn_rows_dq_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int VEC = vec_of<T>(), G = lanes_of<T, DP>(), U = 2;
  pdl_enter();
  const int warp = threadIdx.x >> 5, group = a.heads / a.kv_heads;
  const Lanes<T, DP> w(a, SPLIT ? a.split_side : a.side);
  const int blocks = w.blocks;
  float q[R][VEC], g[R][VEC], ref[R], pek[R][VEC], pk[R][VEC], delta[R];
  const auto begin = [&](int row, int head, int heads, bool in) {
    load_heads<T, R>(a.q, row, head, heads, w.vec, in, a.scale * LOG2E, q);
    load_heads<T, R>(a.dout, row, head, heads, w.vec, in, 1.0f, g);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ref[r] = reference_of(a, head + r, row, in && r < heads);
      delta[r] = 0.0f;
#pragma unroll
      for (int x = 0; x < VEC; ++x) pek[r][x] = pk[r][x] = 0.0f;
    }
  };
  const auto add = [&](int r) {
    add_keys<VEC>(w.side * G, pek[r]);
    add_keys<VEC>(w.side * G, pk[r]);
    float one[1] = {delta[r]};
    add_keys<1>(w.side * G, one);
    delta[r] = one[0];
  };
  if constexpr (SPLIT) {
    __shared__ Shared<T, DP, 2 * DP + 1> shared;
    __shared__ bool flag;
    const int split_ctas = gridDim.x;
    const int floats = 2 * a.d + 1, n = min(a.counts[ATTN_N_SPLITS], a.split_bound);
    for (int64_t t = blockIdx.x; t < static_cast<int64_t>(n) * blocks; t += split_ctas) {
      const int item = static_cast<int>(t / blocks), block = static_cast<int>(t - static_cast<int64_t>(item) * blocks);
      const int4 it = a.splits[item];
      bool found, again;
      const AttnSeq e = sequence_of(a, a.q_seq, it.x, false, &found, &again);
      const int c = block * w.side + w.head, j0 = it.y, j1 = min(found ? keys_seen(a, e, it.x) : 0, j0 + ATTN_SPLIT_KEYS);
      const bool in = w.in_d && c < a.kv_heads;
      const T* k = static_cast<const T*>(a.k.p) + e.k0 * a.k.row + c * a.k.head + w.vec * VEC;
      const T* v = static_cast<const T*>(a.v.p) + e.k0 * a.v.row + c * a.v.head + w.vec * VEC;
      for (int h0 = 0; h0 < group; h0 += R) {
        const int heads = min(R, group - h0);
        begin(it.x, c * group + h0, heads, in && j1 > 0);
        backward_keys<T, DP, R>(k, a.k.row, v, a.v.row, j0 + warp * w.keys * U, j1, ROW_WARPS * w.keys * U, w, in, q, g, ref, pek, pk, delta);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          add(r);
          if (r >= heads) continue;  // (the same for all threads)
          __syncthreads();           // `shared` may be written again
          if (w.key == 0) {
            float* to = shared.v[warp][w.head];
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
              to[w.vec * VEC + x] = pek[r][x];
              to[DP + w.vec * VEC + x] = pk[r][x];
            }
            if (w.vec == 0) to[2 * DP] = delta[r];
          }
          __syncthreads();
          for (int i = threadIdx.x; i < w.side * floats; i += ROW_WARPS * 32) {
            const int hs = i / floats, x = i - hs * floats, at = x < a.d ? x : x < 2 * a.d ? DP + x - a.d : 2 * DP, kv = block * w.side + hs;
            if (kv >= a.kv_heads) continue;
            float sum = 0.0f;
#pragma unroll
            for (int y = 0; y < ROW_WARPS; ++y) sum += shared.v[y][hs][at];
            a.parts[(static_cast<int64_t>(item) * a.heads + kv * group + h0 + r) * floats + x] = sum;
          }
        }
      }
      if (last_part(a, it, block, &flag) && found) {
        const int lane = threadIdx.x & 31, first = block * w.side * group, all = min(a.heads - first, w.side * group);
        for (int h = warp; h < all; h += ROW_WARPS) {
          const int head = first + h;
          const float* part = a.parts + (static_cast<int64_t>(it.z) * a.heads + head) * floats;
          const int64_t apart = static_cast<int64_t>(a.heads) * floats;
          float sum = 0.0f, ek[DP / 32], pk1[DP / 32];
#pragma unroll
          for (int x = 0; x < DP / 32; ++x) ek[x] = pk1[x] = 0.0f;
#pragma unroll 4
          for (int p = 0; p < it.w; ++p) {
            sum += __ldcg(part + p * apart + 2 * a.d);
#pragma unroll
            for (int x = 0; x < DP / 32; ++x)
              if (x * 32 + lane < a.d) {
                ek[x] += __ldcg(part + p * apart + x * 32 + lane);
                pk1[x] += __ldcg(part + p * apart + a.d + x * 32 + lane);
              }
          }
#pragma unroll
          for (int x = 0; x < DP / 32; ++x)
            if (x * 32 + lane < a.d && a.dq != nullptr)
              static_cast<T*>(a.dq)[(static_cast<int64_t>(it.x) * a.heads + head) * a.d + x * 32 + lane] =
                  from_float<T>(a.scale * fmaf(-sum, pk1[x], ek[x]));
          if (lane == 0) a.delta[static_cast<int64_t>(head) * a.n_q + it.x] = sum;
        }
      }
      __syncthreads();  // `flag` may be written again
    }
    return;
  }
  each_row(
      a, static_cast<int64_t>(blockIdx.x) * ROW_WARPS + warp, static_cast<int64_t>(gridDim.x) * ROW_WARPS, range_of(a, false), blocks, a.q_seq, false,
      [&](const AttnSeq& e, bool found, bool again) {
        return !found || again || !(attn_in_tiles(a, e) || attn_is_split(a, e) || attn_is_single(a, e));
      },
      [&](int row, int block, const AttnSeq& e) {
        const int seen = keys_seen(a, e, row), c = block * w.side + w.head;
        const bool in = w.in_d && c < a.kv_heads;
        const T* k = static_cast<const T*>(a.k.p) + e.k0 * a.k.row + c * a.k.head + w.vec * VEC;
        const T* v = static_cast<const T*>(a.v.p) + e.k0 * a.v.row + c * a.v.head + w.vec * VEC;
        for (int h0 = 0; h0 < group; h0 += R) {
          const int heads = min(R, group - h0), head = c * group + h0;
          begin(row, head, heads, in && seen > 0);
          backward_keys<T, DP, R>(k, a.k.row, v, a.v.row, 0, seen, w.keys * U, w, in, q, g, ref, pek, pk, delta);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            add(r);
            if (!(w.key == 0 && in && r < heads)) continue;
            float dq[VEC];
#pragma unroll
            for (int x = 0; x < VEC; ++x) dq[x] = a.scale * fmaf(-delta[r], pk[r][x], pek[r][x]);
            if (a.dq != nullptr)
              store_vec<T, VEC>(static_cast<T*>(a.dq) + (static_cast<int64_t>(row) * a.heads + head + r) * a.d + w.vec * VEC, dq);
            if (w.vec == 0) a.delta[static_cast<int64_t>(head + r) * a.n_q + row] = delta[r];
          }
        }
      });
}

// dk and dv of the keys of other sequences: a slot of lanes for each key row and key head, over the queries that see it, the heads of its group R
// at a time.  Keys that no sequence holds get zeros.
template <typename T, int DP, int R>
__global__ __launch_bounds__(ROW_WARPS * 32, 2) void attn_rows_dkv_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int VEC = vec_of<T>(), G = lanes_of<T, DP>();
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.heads / a.kv_heads, blocks = (a.kv_heads + a.side - 1) / a.side;
  const Lanes<T, DP> w(a, a.side);
  const Range range = range_of(a, true);
  const int64_t all = static_cast<int64_t>((range.rows + a.rows_at_once - 1) / a.rows_at_once) * blocks;
  for (int64_t task = static_cast<int64_t>(blockIdx.x) * ROW_WARPS + warp; task < all; task += static_cast<int64_t>(gridDim.x) * ROW_WARPS) {
    const int batch = static_cast<int>(task / blocks), block = static_cast<int>(task - static_cast<int64_t>(batch) * blocks);
    const int begin = batch * a.rows_at_once, mine = begin + lane;
    bool found = false, take = false, again;
    AttnSeq own{0, 0, 0, 0};
    if (lane < a.rows_at_once && mine < range.rows) {
      own = sequence_of(a, a.k_seq, range.row(mine), true, &found, &again);
      take = !found || again || !(attn_in_tiles(a, own) || attn_is_single(a, own));
      if (!found) own = AttnSeq{0, 0, 0, 0};
    }
    unsigned todo = __ballot_sync(FULL_MASK, take);
    while (todo != 0) {
      // as many of them as lie side by side
      int n = -1;
      for (int i = 0; i < w.keys && todo != 0; ++i, todo &= todo - 1)
        if (i == w.key) n = __ffs(todo) - 1;
      const int from = n < 0 ? 0 : n, row = range.row(begin + from), c = block * w.side + w.head;
      const AttnSeq e{__shfl_sync(FULL_MASK, own.q0, from), __shfl_sync(FULL_MASK, own.q_len, from), __shfl_sync(FULL_MASK, own.k0, from),
                      __shfl_sync(FULL_MASK, own.k_len, from)};
      const bool here = n >= 0 && c < a.kv_heads, in = here && w.in_d;
      const int first = a.causal ? max(0, row - e.k0 - (e.k_len - e.q_len)) : 0;  // query that sees this key first
      const int queries = here ? max(0, e.q_len - first) : 0;
      const int most = __reduce_max_sync(FULL_MASK, queries);
      float k[VEC], v[VEC], dk[VEC], dv[VEC];
      load_row<T, VEC>(static_cast<const T*>(a.k.p) + row * a.k.row + c * a.k.head + w.vec * VEC, in && queries > 0, k);
      load_row<T, VEC>(static_cast<const T*>(a.v.p) + row * a.v.row + c * a.v.head + w.vec * VEC, in && queries > 0, v);
#pragma unroll
      for (int x = 0; x < VEC; ++x) dk[x] = dv[x] = 0.0f;
      for (int i = 0; i < most; ++i) {
        const bool on = i < queries;
        const int at = e.q0 + first + (on ? i : 0);
        for (int h0 = 0; h0 < group; h0 += R) {
          const int heads = min(R, group - h0), head = c * group + h0;
          float q[R][VEC], g[R][VEC], ref[R], delta[R];
          load_heads<T, R>(a.q, at, head, heads, w.vec, in && on, 1.0f, q);
          load_heads<T, R>(a.dout, at, head, heads, w.vec, in && on, 1.0f, g);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            ref[r] = reference_of(a, head + r, at, here && on && r < heads);
            delta[r] = here && on && r < heads ? a.delta[static_cast<int64_t>(head + r) * a.n_q + at] : 0.0f;
          }
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float x = group_sum<G>(dot<VEC>(q[r], k)) * (a.scale * LOG2E), y = group_sum<G>(dot<VEC>(g[r], v));
            const float p = on && r < heads ? ex2(x - ref[r]) : 0.0f, ds = p * (y - delta[r]);
            add_scaled<VEC>(p, g[r], dv);
            add_scaled<VEC>(ds, q[r], dk);
          }
        }
        // what is not a number stays so: long sequences made again after a step that went wrong altogether end here (4 causal ones of 8 192 tokens,
        // forward and backward: 5.1 ms of numbers, 7.7 with q and v all nan, 370 without this; 95 with one nan, in the first value)
        if ((i & 31) == 31) {
          bool gone = true;
#pragma unroll
          for (int x = 0; x < VEC; ++x) gone &= dk[x] != dk[x] && dv[x] != dv[x];
          if (__all_sync(FULL_MASK, gone || !in)) break;
        }
      }
      if (!in) continue;
#pragma unroll
      for (int x = 0; x < VEC; ++x) dk[x] *= a.scale;
      const int64_t to = (static_cast<int64_t>(row) * a.kv_heads + c) * a.d + w.vec * VEC;
      store_vec<T, VEC>(static_cast<T*>(a.dk) + to, dk);
      store_vec<T, VEC>(static_cast<T*>(a.dv) + to, dv);
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct Layout {
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};

// whether sequences may go to the tensor cores (a scale that is not positive, which no model has, stays on the CUDA cores: the tiles take the largest
// score for the largest weight)
bool has_tiles(const dgs_attention& p) {
  return p.dtype != DGS_F32 && p.n_q >= ATTN_FEW_QUERIES && p.n_k > 0 && p.seqs > 0 && p.scale > 1e-30f;
}

// Parts that rows with many keys can have, whatever the offsets: k keys are ceil(k / ATTN_SPLIT_KEYS) <= k / ATTN_SPLIT_KEYS + 1 parts for each of a
// sequence's queries.  Where many sequences are just long enough, keys are the bound: 2 parts for ATTN_SPLIT_KEYS + 1 of them is the most (as
// 1 for ATTN_SPLIT_FROM + 1 nearly is), and with tiles, which take ATTN_FEW_QUERIES and more over up to ATTN_MANY_KEYS, 5 for ATTN_MANY_KEYS + 1.
// (none, and no launch for them, where all keys together are too few for one: whether a row is split is a matter of its own keys alone)
int64_t split_bound(const dgs_attention& p) {
  if (p.n_k <= ATTN_SPLIT_FROM) return 0;
  static_assert(2 * (ATTN_SPLIT_FROM + 1) >= ATTN_SPLIT_KEYS + 1 && ATTN_MANY_KEYS == 4 * ATTN_SPLIT_KEYS, "parts of a key");
  const int64_t queries = p.n_q < ATTN_SPLIT_QUERIES ? p.n_q : ATTN_SPLIT_QUERIES;
  const int64_t longest = p.n_k / (ATTN_SPLIT_FROM + 1), some = ATTN_SPLIT_QUERIES * (longest < p.seqs ? longest : p.seqs);
  const int64_t by_rows = queries * (p.n_k / ATTN_SPLIT_KEYS) + (p.n_q < some ? p.n_q : some);
  const bool tiles = has_tiles(p);
  const int64_t few = tiles && queries >= ATTN_FEW_QUERIES ? ATTN_FEW_QUERIES - 1 : queries;
  int64_t by_keys = few * 2 * p.n_k / (ATTN_SPLIT_KEYS + 1);
  if (tiles && by_keys < queries * 5 * p.n_k / (ATTN_MANY_KEYS + 1)) by_keys = queries * 5 * p.n_k / (ATTN_MANY_KEYS + 1);
  return by_rows < by_keys ? by_rows : by_keys;
}

// Workspace of a call; `base` == nullptr: its size alone
int64_t lay_out(const dgs_attention& p, bool backward, char* base, AttnArgs* a) {
  Layout l;
  a->split_bound = static_cast<int32_t>(split_bound(p));
  const int64_t floats = backward ? 2 * p.d + 1 : p.d + 2;
  auto at = [&](int64_t bytes) { return base + l.take(bytes); };
  a->counts = reinterpret_cast<int32_t*>(at(ATTN_COUNTS * 4));
  a->norms = reinterpret_cast<float*>(at(8));
  a->seq = reinterpret_cast<AttnSeq*>(at(p.seqs * static_cast<int64_t>(sizeof(AttnSeq))));
  a->q_seq = reinterpret_cast<int32_t*>(at(p.n_q * 4));
  a->k_seq = reinterpret_cast<int32_t*>(at(backward ? p.n_k * 4 : 0));
  a->splits = reinterpret_cast<int4*>(at(int64_t(16) * a->split_bound));
  a->arrived = reinterpret_cast<uint32_t*>(at(int64_t(4) * a->split_bound * p.kv_heads));
  a->parts = reinterpret_cast<float*>(at(int64_t(4) * a->split_bound * p.heads * floats));
  a->delta = reinterpret_cast<float*>(at(backward ? int64_t(4) * p.heads * p.n_q : 0));
  a->tiles = has_tiles(p);
  // forward, a CTA's two tiles of queries: the same rows of two heads that share their keys, or neighbouring rows
  a->head_pairs = p.heads / p.kv_heads % 2 == 0;
  a->q_tile_rows = backward || a->head_pairs ? ATTN_TILE : 2 * ATTN_TILE;
  // tiles, whatever the offsets: rows / tile + 1 for each of the sequences that can be that long
  const int64_t longest = p.n_q / ATTN_FEW_QUERIES, some = a->tiles ? (longest < p.seqs ? longest : p.seqs) : 0;
  a->q_tile_bound = static_cast<int32_t>(a->tiles ? p.n_q / a->q_tile_rows + some : 0);
  a->k_tile_bound = static_cast<int32_t>(a->tiles && backward ? p.n_k / ATTN_TILE + some : 0);
  a->q_tiles = reinterpret_cast<AttnTile*>(at(a->q_tile_bound * static_cast<int64_t>(sizeof(AttnTile))));
  a->k_tiles = reinterpret_cast<AttnTile*>(at(a->k_tile_bound * static_cast<int64_t>(sizeof(AttnTile))));
  a->lse2 = reinterpret_cast<float*>(at(a->tiles && backward ? int64_t(4) * p.heads * p.n_q : 0));
  return l.bytes;
}

int check(const char* who, const dgs_attention* p) {
  DGS_REQUIRE(p != nullptr, DGS_ERR_INVALID, "%s: null argument", who);
  const int esz = dtype_bytes(p->dtype);
  DGS_REQUIRE(esz != 0, DGS_ERR_UNSUPPORTED, "%s: element type %d", who, p->dtype);
  DGS_REQUIRE(p->n_q >= 0 && p->n_k >= 0 && p->seqs >= 0 && p->n_q < (int64_t(1) << 30) && p->n_k < (int64_t(1) << 30), DGS_ERR_INVALID,
              "%s: %lld query rows, %lld key rows, %d sequences", who, static_cast<long long>(p->n_q), static_cast<long long>(p->n_k), p->seqs);
  DGS_REQUIRE(p->heads >= 1 && p->kv_heads >= 1 && p->heads % p->kv_heads == 0 && p->heads <= 65535, DGS_ERR_INVALID,
              "%s: %d query heads over %d key heads", who, p->heads, p->kv_heads);
  const int vec = 16 / esz;
  DGS_REQUIRE(p->d >= vec && p->d <= ATTN_MAX_D && p->d % vec == 0, DGS_ERR_UNSUPPORTED,
              "%s: heads of %d elements (multiples of %d up to %d)", who, p->d, vec, ATTN_MAX_D);
  DGS_REQUIRE(p->q_row % vec == 0 && p->q_head % vec == 0 && p->k_row % vec == 0 && p->k_head % vec == 0 && p->v_row % vec == 0 &&
                  p->v_head % vec == 0 && aligned_to(p->q, 16) && aligned_to(p->k, 16) && aligned_to(p->v, 16),
              DGS_ERR_INVALID, "%s: heads must begin at 16-byte boundaries", who);
  const auto apart = [](int64_t stride, int64_t n) { return stride > 0 || n <= 1; };
  DGS_REQUIRE(apart(p->q_row, p->n_q) && apart(p->q_head, p->heads) && apart(p->k_row, p->n_k) && apart(p->k_head, p->kv_heads) &&
                  apart(p->v_row, p->n_k) && apart(p->v_head, p->kv_heads),
              DGS_ERR_INVALID, "%s: strides must be positive", who);
  DGS_REQUIRE(p->scale - p->scale == 0.0f, DGS_ERR_INVALID, "%s: scale must be a finite number", who);
  DGS_REQUIRE((p->n_q == 0 || p->q != nullptr) && (p->n_k == 0 || (p->k != nullptr && p->v != nullptr)) &&
                  p->q_offsets != nullptr && p->k_offsets != nullptr,
              DGS_ERR_INVALID, "%s: null argument", who);
  DGS_REQUIRE(split_bound(*p) < (int64_t(1) << 27), DGS_ERR_INVALID, "%s: too many rows", who);
  return DGS_OK;
}

AttnArgs arguments(const dgs_attention& p) {
  AttnArgs a{};
  a.q = {p.q, p.q_row, p.q_head};
  a.k = {p.k, p.k_row, p.k_head};
  a.v = {p.v, p.v_row, p.v_head};
  a.q_offsets = p.q_offsets;
  a.k_offsets = p.k_offsets;
  a.offsets64 = p.ids64;
  a.seqs = p.seqs;
  a.n_q = static_cast<int32_t>(p.n_q);
  a.n_k = static_cast<int32_t>(p.n_k);
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.d = p.d;
  a.causal = p.causal != 0;
  a.singles = p.n_q <= 2 * static_cast<int64_t>(p.seqs) && p.heads <= ATTN_SINGLE_GROUP * p.kv_heads;
  a.scale = p.scale;
  a.wait_limit = wait_limit();
  return a;
}

int launch_plan(const AttnArgs& a, bool backward, cudaStream_t s) {
  const bool one = a.seqs <= PLAN_ONE_CTA;
  if (!one) {
    DGS_CUDA_TRY(cudaMemsetAsync(a.counts, 0, ATTN_COUNTS * 4, s));
    DGS_CUDA_TRY(cudaMemsetAsync(a.norms, 0, 8, s));
  }
  // (one CTA: and others for the maps, a warp for every sequence or two)
  const int64_t each = (static_cast<int64_t>(a.seqs) + PLAN_THREADS / 32 - 1) / (PLAN_THREADS / 32);
  const int64_t ctas = one ? 1 + (each < 32 ? each < 1 ? 1 : each : 32) : each, most = 2 * static_cast<int64_t>(sm_count());
  DGS_CUDA_TRY(launch_training(attn_plan_kernel, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), PLAN_THREADS, 0, s, a,
                               static_cast<int32_t>(backward), static_cast<int32_t>(one)));
  return DGS_OK;
}

// f.run<T, DP, R>() with the elements of a head filled up to DP, R heads of a group at once (MOST of them at most)
template <typename T, int DP, int MOST, typename F>
int with_heads(const AttnArgs& a, const F& f) {
  const int group = a.heads / a.kv_heads;
  if (group == 1) return f.template run<T, DP, 1>();
  if (group == 2 || MOST == 2) return f.template run<T, DP, 2>();
  return f.template run<T, DP, MOST>();
}
template <typename T, int MOST, typename F>
int with_width(const AttnArgs& a, const F& f) {
  return a.d <= 32 ? with_heads<T, 32, MOST>(a, f) : a.d <= 64 ? with_heads<T, 64, MOST>(a, f) : with_heads<T, 128, MOST>(a, f);
}
template <int MOST, typename F>
int with_type(int32_t dtype, const AttnArgs& a, const F& f) {
  return dtype == DGS_F32    ? with_width<float, MOST>(a, f)
         : dtype == DGS_BF16 ? with_width<__nv_bfloat16, MOST>(a, f)
                             : with_width<__half, MOST>(a, f);
}

int split_ctas(const AttnArgs& a) {
  const int64_t tasks = static_cast<int64_t>(a.split_bound) * a.kv_heads, most = static_cast<int64_t>(sm_count()) * 4;
  return static_cast<int>(tasks < most ? tasks : most);
}
// CTAs for so many rows: enough to fill the SMs, which then take the rows in turn
unsigned row_ctas(const AttnArgs& a, int64_t rows) {
  const int64_t blocks = (a.kv_heads + a.side - 1) / a.side, tasks = (rows + a.rows_at_once - 1) / a.rows_at_once * blocks;
  const int64_t need = (tasks + ROW_WARPS - 1) / ROW_WARPS, most = static_cast<int64_t>(sm_count()) * 16;
  return static_cast<unsigned>(need < most ? need : most);
}
// how the lanes of a warp are shared out, and how many rows a warp looks up at once: more where there are rows enough for all warps
template <typename T, int DP>
AttnArgs with_lanes(AttnArgs a, int64_t rows, bool keys = false) {
  a.split_side = 1;
  while (a.split_side < a.kv_heads && a.split_side < 32 / lanes_of<T, DP>()) a.split_side *= 2;
  a.side = a.n_k <= static_cast<int64_t>(ATTN_FEW_KEYS) * a.seqs ? a.split_side : 1;
  // (eight where rows are short; two, or a key for each slot of a warp, where they may take long)
  const int64_t warps = static_cast<int64_t>(sm_count()) * 32;
  const int most = a.side > 1 ? 8 : keys ? 32 / lanes_of<T, DP>() : 2;
  a.rows_at_once = keys && a.side == 1 ? most : 1;
  while (a.rows_at_once < most && rows >= warps * 2 * a.rows_at_once) a.rows_at_once *= 2;
  return a;
}

struct RowsForward {
  const AttnArgs& a;
  cudaStream_t s;
  template <typename T, int DP, int R>
  int run() const {
    const AttnArgs b = with_lanes<T, DP>(a, a.n_q);
    if (const int ctas = split_ctas(b)) DGS_CUDA_TRY(launch_training(attn_rows_kernel<T, DP, R, true>, dim3(ctas), ROW_WARPS * 32, 0, s, b));
    DGS_CUDA_TRY(launch_training(attn_rows_kernel<T, DP, R, false>, dim3(row_ctas(b, b.n_q)), ROW_WARPS * 32, 0, s, b));
    return DGS_OK;
  }
};
struct RowsSingle {
  const AttnArgs& a;
  cudaStream_t s;
  template <typename T, int DP, int R>
  int run() const {
    const AttnArgs b = with_lanes<T, DP>(a, a.n_q);
    DGS_CUDA_TRY(launch_training(attn_single_backward_kernel<T, DP, R>, dim3(row_ctas(b, b.n_q)), ROW_WARPS * 32, 0, s, b));
    return DGS_OK;
  }
};
struct RowsBackward {
  const AttnArgs& a;
  cudaStream_t s;
  template <typename T, int DP, int R>
  int run() const {
    const AttnArgs b = with_lanes<T, DP>(a, a.n_q);
    if (const int ctas = split_ctas(b)) DGS_CUDA_TRY(launch_training(attn_rows_dq_kernel<T, DP, R, true>, dim3(ctas), ROW_WARPS * 32, 0, s, b));
    DGS_CUDA_TRY(launch_training(attn_rows_dq_kernel<T, DP, R, false>, dim3(row_ctas(b, b.n_q)), ROW_WARPS * 32, 0, s, b));
    return DGS_OK;
  }
};
struct KeysBackward {
  const AttnArgs& a;
  cudaStream_t s;
  template <typename T, int DP, int R>
  int run() const {
    const AttnArgs b = with_lanes<T, DP>(a, a.n_k, true);
    DGS_CUDA_TRY(launch_training(attn_rows_dkv_kernel<T, DP, R>, dim3(row_ctas(b, b.n_k)), ROW_WARPS * 32, 0, s, b));
    return DGS_OK;
  }
};

}  // namespace
}  // namespace dgs

using namespace dgs;

extern "C" size_t dgs_attention_workspace_bytes(const dgs_attention* p, int32_t backward) {
  if (p == nullptr || p->n_q < 0 || p->n_k < 0 || p->seqs < 0 || p->heads < 1 || p->kv_heads < 1 || p->d < 1) return 0;
  AttnArgs a{};
  return static_cast<size_t>(lay_out(*p, backward != 0, nullptr, &a));
}

extern "C" int dgs_attention_forward(const dgs_attention* p, void* out, float* lse, void* workspace, size_t workspace_bytes,
                                     int32_t* status, dgs_stream_t stream) {
  if (int rc = check("attention", p)) return rc;
  if (p->n_q == 0) return DGS_OK;
  DGS_REQUIRE(out != nullptr && lse != nullptr && aligned_to(out, 16), DGS_ERR_INVALID, "attention: out (16-byte aligned) and lse are needed");
  const size_t need = dgs_attention_workspace_bytes(p, 0);
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "attention: workspace of %zu bytes, 256-byte aligned, is needed", need);
  AttnArgs a = arguments(*p);
  lay_out(*p, false, static_cast<char*>(workspace), &a);
  a.out = out;
  a.lse = lse;
  a.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = launch_plan(a, false, s)) return rc;
  if (a.tiles)
    if (int rc = attn_tiles_forward(a, p->dtype, s)) return rc;
  return with_type<4>(p->dtype, a, RowsForward{a, s});
}

extern "C" int dgs_attention_backward(const dgs_attention* p, const void* dout, int64_t dout_row, int64_t dout_head, const void* out,
                                      const float* lse, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                      int32_t* status, dgs_stream_t stream) {
  if (int rc = check("attention_backward", p)) return rc;
  DGS_REQUIRE((dk == nullptr) == (dv == nullptr), DGS_ERR_INVALID, "attention_backward: the gradients of keys and values come together");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t esz = dtype_bytes(p->dtype), kv = static_cast<size_t>(p->n_k) * p->kv_heads * p->d * esz;
  if (p->n_q == 0) {
    if (dk != nullptr && kv != 0) {
      DGS_CUDA_TRY(cudaMemsetAsync(dk, 0, kv, s));
      DGS_CUDA_TRY(cudaMemsetAsync(dv, 0, kv, s));
    }
    return DGS_OK;
  }
  if (dq == nullptr && dk == nullptr) return DGS_OK;
  const int64_t vec = 16 / static_cast<int64_t>(esz);
  DGS_REQUIRE(dout != nullptr && out != nullptr && lse != nullptr && aligned_to(dout, 16) && aligned_to(out, 16) && aligned_to(dq, 16) &&
                  aligned_to(dk, 16) && aligned_to(dv, 16) && dout_row % vec == 0 && dout_head % vec == 0 && (dout_row > 0 || p->n_q == 1) &&
                  (dout_head > 0 || p->heads == 1),
              DGS_ERR_INVALID, "attention_backward: dout, out, lse and gradients must be there, heads must begin at 16-byte boundaries");
  const size_t need = dgs_attention_workspace_bytes(p, 1);
  DGS_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned_to(workspace, 256), DGS_ERR_INVALID,
              "attention_backward: workspace of %zu bytes, 256-byte aligned, is needed", need);
  AttnArgs a = arguments(*p);
  lay_out(*p, true, static_cast<char*>(workspace), &a);
  a.dout = {dout, dout_row, dout_head};
  a.out = const_cast<void*>(out);
  a.lse = const_cast<float*>(lse);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.status = status;
  if (int rc = launch_plan(a, true, s)) return rc;
  if (a.tiles)
    if (int rc = attn_tiles_backward(a, p->dtype, s)) return rc;
  if (a.singles)
    if (int rc = with_type<4>(p->dtype, a, RowsSingle{a, s})) return rc;
  if (int rc = with_type<2>(p->dtype, a, RowsBackward{a, s})) return rc;
  return a.dk == nullptr || a.n_k == 0 ? DGS_OK : with_type<4>(p->dtype, a, KeysBackward{a, s});
}
