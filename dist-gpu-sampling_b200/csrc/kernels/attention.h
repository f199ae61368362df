// What the kernels of packed attention share (attention.cu: the plan, rows on the CUDA cores, entry points; attention_mma.cu: tiles
// on the tensor cores).  Not part of the C ABI.
#pragma once
#include "train_common.cuh"

namespace dgs {

// Rows of one sequence; a sequence whose offsets are not in order has none.
struct AttnSeq {
  int32_t q0, q_len, k0, k_len;
};

// A tile of query rows (all heads take it), or of key rows with the query rows that see them.
struct __align__(16) AttnTile {
  int32_t row, rows;           // the tile's rows
  int32_t other, others;       // first row and number of the rows on the other side: the keys; the queries that see one of the keys
  int32_t seen;                // causal: keys of `others` that the tile's first query sees (may be negative); key tiles: the tile's first key as the
                               // first of `others` counts the keys that it sees (key j of the tile is seen by query i if j + seen <= i)
  int32_t steps;               // tiles on the other side
  int32_t pad[2];
};

struct AttnView {
  const void* p;
  int64_t row, head;  // strides in elements
};

struct AttnArgs {
  AttnView q, k, v, dout;
  const void *q_offsets, *k_offsets;
  int32_t offsets64;
  int32_t seqs, n_q, n_k, heads, kv_heads, d, causal;
  int32_t tiles, singles;  // whether long sequences go to the tensor cores, single queries to a kernel of their own
  float scale;
  // results: contiguous rows of `heads` (`kv_heads`) times d elements; lse and delta [heads, n_q]
  void* out;
  float* lse;
  void *dq, *dk, *dv;
  // workspace
  AttnSeq* seq;                 // [seqs]
  int32_t *q_seq, *k_seq;       // the sequence of a row (ATTN_AGAIN beside it); only entries whose sequence holds the row mean anything
  int32_t* counts;              // ATTN_COUNTS words
  int4* splits;                 // {row, first key, index of the row's first part, parts}
  uint32_t* arrived;            // parts that are there, one word for each part (the first of a row's is used) and key head
  float* parts;                 // [part][heads][part_floats]
  AttnTile *q_tiles, *k_tiles;  // heaviest first where one CTA makes the plan
  float *delta, *lse2;  // [heads, n_q]; lse in powers of two, as the tiles' backward pass takes it
  float* norms;                 // [2] the largest row norms of dout and v (as they are ordered, through unsigned words)
  int32_t* status;
  uint64_t wait_limit;  // of a wait, in nanoseconds
  int32_t split_bound, q_tile_bound, k_tile_bound, q_tile_rows, head_pairs;
  // rows on the CUDA cores: key heads side by side in a warp (and in those of a split row), rows that it looks up at once
  int32_t side, split_side, rows_at_once;
};

enum { ATTN_N_SPLITS = 0, ATTN_N_Q_TILES = 1, ATTN_N_K_TILES = 2, ATTN_KINDS = 3, ATTN_COUNTS = 8 };
enum { ATTN_HAS_TILES = 0, ATTN_HAS_SINGLE = 1, ATTN_HAS_SEVERAL = 2, ATTN_HAS_AGAIN = 3 };  // bits of the word ATTN_KINDS

// A row of a causal tile whose result is not a number although it may have to be one: a pair that is masked has the weight 0, and 0 times what is
// not finite is not a number.  The rows' kernels, which come after the tiles' and read what a row sees alone, make it again.
constexpr int32_t ATTN_AGAIN = INT32_MIN;

constexpr int ATTN_MAX_D = 128;
// keys from which a CTA takes a row instead of a warp.  8 heads on 2, width 64, bf16, us forward / backward with 256 and with 512 here: 2 000
// rows of 500 keys 287 / 1 650 and 185 / 702, one row of 500 keys 25 / 38 and 38 / 114; with 1 024, when a warp took its keys once backward: one
// row of 1 000 keys 36 / 54 and 68 / 153
constexpr int ATTN_SPLIT_FROM = 512;
constexpr int ATTN_SPLIT_KEYS = 1024;  // so many of them at a time
constexpr int ATTN_SPLIT_QUERIES = 16; // (with more queries there are warps enough)
constexpr int ATTN_TILE = 128;         // rows of a tile of keys, and of queries
constexpr int ATTN_TILE_QUERIES = 24;  // queries from which a sequence goes to the tensor cores whatever its keys, ...
constexpr int ATTN_FEW_QUERIES = 8;    // ... or from which it does with so many pairs, unless there are keys enough to be split
constexpr int ATTN_TILE_PAIRS = 576, ATTN_MANY_KEYS = 4096;
constexpr int ATTN_FEW_KEYS = 24;      // keys a sequence on average up to which a warp takes key heads side by side, beyond it takes keys

__host__ __device__ inline bool attn_many_keys(const AttnSeq& s) {
  return s.k_len > ATTN_SPLIT_FROM && s.q_len <= ATTN_SPLIT_QUERIES && (s.q_len < ATTN_FEW_QUERIES || s.k_len > ATTN_MANY_KEYS);
}
__host__ __device__ inline bool attn_in_tiles(const AttnArgs& a, const AttnSeq& s) {
  if (!a.tiles || s.k_len == 0 || s.q_len < ATTN_FEW_QUERIES) return false;
  return s.q_len >= ATTN_TILE_QUERIES || (!attn_many_keys(s) && static_cast<int64_t>(s.q_len) * s.k_len >= ATTN_TILE_PAIRS);
}
__host__ __device__ inline bool attn_is_split(const AttnArgs& a, const AttnSeq& s) {
  return s.k_len > ATTN_SPLIT_FROM && s.q_len <= ATTN_SPLIT_QUERIES && !attn_in_tiles(a, s);
}
// one query over a few keys: its backward pass is one kernel (whose registers hold so many heads of a group), where most sequences are so
constexpr int ATTN_SINGLE_GROUP = 4;
__host__ __device__ inline bool attn_is_single(const AttnArgs& a, const AttnSeq& s) {
  return a.singles && s.q_len == 1 && s.k_len <= ATTN_SPLIT_FROM;
}

// attention_mma.cu: the sequences that attn_in_tiles names, after the plan
int attn_tiles_forward(const AttnArgs& a, int32_t dtype, cudaStream_t s);
int attn_tiles_backward(const AttnArgs& a, int32_t dtype, cudaStream_t s);

}  // namespace dgs
