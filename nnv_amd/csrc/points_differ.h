// Differential attention of points: what the forward and the backward kernels share.
//
//   S_m = scale q_m k_m^T,  lse_m = log sum over the keys that a query sees of exp(S_m),  P_m = exp(S_m - lse_m)     (maps m = 0, 1)
//   o_m = P_m v,  o = o_0 - w o_1                                                     (w: one per head; v has twice the values of q_m)
//   D_m = rowsum(do o_m),  dP = do v^T (one for both maps),  dS_0 = P_0 (dP - D_0),  dS_1 = -w P_1 (dP - D_1)
//   dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dv = (P_0 - w P_1)^T do,  dw = -sum of D_1
//
// Rows, and how the products follow one another, are as in points_attend.h: row r of (sequence, key/value head) is query r % queries of the
// group's head r / queries.  Of the values of lse, D and the partial results there is one for each map and row: (sequence, key/value head, map, row) of the
// kernels' own, while the caller's lse lies as (sequence, head, map, query).
//
// A causal row sees the keys in front of n - queries + query + 1, n the sequence's length; rows of a tile differ in it, and the first
// rows of a sequence shorter than the queries see none.
#pragma once
#include "points_attend.h"

namespace nnvhip {

struct DifferArgs : AttendArgs {   // (its lse is the caller's; scale, masks and the views as there, with 2 heads of q and k)
  const void* weights;
  int wide_weights, causal;
  void* second;                    // dense, or null
  void* dweights;
  float* info;                     // [sequence, key/value head][kInfos][info_rows]: see RowInfo
  int info_rows;                   // rows, rounded up to kInfoRows
  float* dots;                     // D of 16-bit tensors as the kernel of dq finds it, [split][sequence, key/value head][map][row]; else null
};

// What the gradients of keys need of a row, as arrays over the rows of a key/value head that a tile's transfer takes as they lie: the exponents' offsets of both
// maps (infinite for rows without keys, and behind the last one), D of both, the weight with its sign turned, and how many keys the row sees.
enum RowInfo { kOffset0, kOffset1, kDelta0, kDelta1, kWeight, kSees, kInfos };
constexpr int kInfoRows = 64;
// Of 16-bit tensors, whose o and second are rounded, D of a block of rows that see up to so many keys is found by going through the keys twice: what D of rounded values leaves in dq is large
// where keys are few (in bf16 a causal call of 64 x 16 has dq 1.4 times as far off as its rounding, 1000 x 1000 1.07, not causal 1.01), and for long rows going twice would take
// the gradients of 4096 x 4096, 16 heads of 64, 1081 us instead of 865.
constexpr int kTwice = 256;
__device__ __forceinline__ float* info_at(const DifferArgs& a, int64_t bkv, int64_t r, int which) { return a.info + (bkv * kInfos + which) * a.info_rows + r; }

__device__ __forceinline__ int64_t map_row_at(const TokenView& t, const DifferArgs& a, int b, int kv, int64_t r, int map) {
  const int64_t g = (uint32_t)r / (uint32_t)a.queries, i = r - g * a.queries;
  return b * t.b + i * t.t + (2 * (kv * (int64_t)a.group + g) + map) * t.h;
}
__device__ __forceinline__ int64_t lse_at(const DifferArgs& a, int b, int kv, int64_t r, int map) {
  const int64_t g = (uint32_t)r / (uint32_t)a.queries, i = r - g * a.queries;
  return ((b * (int64_t)a.kv_heads * a.group + kv * (int64_t)a.group + g) * 2 + map) * a.queries + i;
}
// the first map's row in dq, and a row of o, second: dense tensors
__device__ __forceinline__ int64_t dense_map_row_at(const DifferArgs& a, int b, int kv, int64_t r, int map) {
  const int64_t g = (uint32_t)r / (uint32_t)a.queries, i = r - g * a.queries;
  return ((b * (int64_t)a.queries + i) * a.kv_heads * a.group * 2 + (kv * (int64_t)a.group + g) * 2 + map) * a.head;
}
__device__ __forceinline__ int64_t wide_row_at(const DifferArgs& a, int b, int kv, int64_t r) { return dense_map_row_at(a, b, kv, r, 0); }
__device__ __forceinline__ int64_t own_row(const DifferArgs& a, int64_t bkv, int64_t r, int map) { return (bkv * 2 + map) * a.rows + r; }
__device__ __forceinline__ int64_t own_rows(const DifferArgs& a) { return (int64_t)a.batch * a.kv_heads * 2 * a.rows; }

template <typename T>
__device__ __forceinline__ float weight_of(const DifferArgs& a, int head) {
  return a.wide_weights ? ((const float*)a.weights)[head] : to_f(((const T*)a.weights)[head]);
}
__device__ __forceinline__ int head_of_row(const DifferArgs& a, int kv, int64_t r) {
  return kv * a.group + (int)((uint32_t)r / (uint32_t)a.queries);
}

// keys that row r sees, of the n that count
__device__ __forceinline__ int seen_by(const DifferArgs& a, int64_t r, int n) {
  if (!a.causal) return n;
  const int i = (int)((uint32_t)r % (uint32_t)a.queries);
  return max(0, n - a.queries + i + 1);
}
// the most keys, and the fewest, that one of the rows first ... last sees
__device__ __forceinline__ int most_seen(const DifferArgs& a, int64_t first, int64_t last, int n) {
  if (!a.causal) return n;
  const uint32_t q = (uint32_t)a.queries;
  return (uint32_t)first / q != (uint32_t)last / q ? n : seen_by(a, last, n);
}
__device__ __forceinline__ int fewest_seen(const DifferArgs& a, int64_t first, int64_t last, int n) {
  if (!a.causal) return n;
  const uint32_t q = (uint32_t)a.queries;
  return (uint32_t)first / q != (uint32_t)last / q ? max(0, n - a.queries + 1) : seen_by(a, first, n);
}
// The first tile of `size` rows, from tile t on, of which a row may see key `key`: causal rows in front of a head's row i_min do not.  (Behind the last: a
// number of no tile.)
__device__ __forceinline__ int next_row_tile(const DifferArgs& a, int t, int size, int i_min) {
  if (i_min <= 0) return t;
  const int64_t first = (int64_t)t * size;
  if (first >= a.rows) return t;
  const uint32_t q = (uint32_t)a.queries, g = (uint32_t)first / q, i = (uint32_t)first - g * q;
  if (i + size > q || (int)(i + size) > i_min) return t;   // reaches into the next head, or to i_min
  return (int)(((int64_t)g * q + i_min) / size);           // (of this head: i_min is one of its rows)
}

// The x-th tile of rows that blocks take, of those of a key/value head.  Causal: those that see most keys first, of all heads of the group, so that the
// short ones fill what is left at the end.
__device__ __forceinline__ int row_tile_of(const DifferArgs& a, int x) {
  const int each = a.row_tiles / a.group;   // tiles of a head, about
  return a.causal && x < each * a.group ? x % a.group * each + each - 1 - x / a.group : x;
}
// Where the tiles of `size` rows of a split of a block over keys begin, of those of which a row may see one of its keys, from a head's row i_min on: all splits
// get as many such rows.  (8 x 2552 x 640 causal, 4 / 2 heads of 32, five splits: with as many tiles each, 20 of one had rows that see a key, of another none.)
__device__ __forceinline__ int first_row_tile(const DifferArgs& a, int split, int size, int i_min) {
  const uint32_t splits = a.splits, q = a.queries, skipped = min(max(i_min, 0), a.queries), each = q - skipped;
  if (split == 0 || each == 0) return 0;
  if (split == a.splits) return (int)((a.rows + size - 1) / size);
  const uint32_t all = each * a.group, at = all / splits * split + all % splits * split / splits, head = at / each;
  return (int)((head * q + skipped + (at - head * each)) / (uint32_t)size);
}
// Blocks of the kernels over keys.  Causal: a tile of early keys is seen by most rows, one of late keys by few, and a block takes one of either (and
// where their number is odd, one block the middle one alone).  Not where the tiles are few, or few of the keys are hidden from any row (8 x 16 x 504, 2 heads
// of 96: 29 us, in pairs 49; 2 x 4096 x 4096, 16 / 4 heads of 64: 650, in pairs 430).
__host__ __device__ inline int key_blocks_of(int key_tiles, int64_t queries, int64_t keys, bool causal) {
  return causal && key_tiles >= 6 && queries >= keys / 2 ? (key_tiles + 1) / 2 : key_tiles;
}
__device__ __forceinline__ int key_blocks_of(const DifferArgs& a) { return key_blocks_of(a.key_tiles, a.queries, a.keys, a.causal); }

// Where a block works: (sequence, key/value head) and one of `each` blocks of it.  Blocks are dealt to the 8 XCDs in turn, and those of a key/value head
// go to one, whose L2 then holds its keys; sequences go by length, the longest first, so that short blocks fill what is left at the end.
// (8 x 577 x 1000 by length, 12 heads of 40, 480 blocks: in the order of their numbers 64 us, two of the longest one after the other.)
struct BlockPlace {
  int b, kv, x;
};
__device__ __forceinline__ BlockPlace block_place(const DifferArgs& a, uint32_t id, uint32_t each) {   // (a grid has fewer blocks than 2^23)
  const uint32_t groups = (uint32_t)a.batch * a.kv_heads, whole = groups / 8 * 8 * each;
  uint32_t group, x;
  if (id < whole) {
    group = id / 8 / each * 8 + id % 8;
    x = id / 8 % each;
  } else {
    group = groups / 8 * 8 + (id - whole) / each;
    x = (id - whole) % each;
  }
  BlockPlace p{(int)(group / (uint32_t)a.kv_heads), (int)(group % (uint32_t)a.kv_heads), (int)x};
  if (a.lengths != nullptr && a.batch <= 64 && a.batch > 1) {   // the sequence of that rank
    const int lane = threadIdx.x & 63, mine = lane < a.batch ? min(max(a.lengths[lane], 0), a.keys) : -1;
    int rank = 0;
    for (int j = 0; j < a.batch; ++j) {
      const int other = __builtin_amdgcn_readlane(mine, j);
      rank += other > mine || (other == mine && j < lane);
    }
    p.b = __builtin_ctzll(__ballot(lane < a.batch && rank == p.b));
  }
  return p;
}

// store_four where sizes are multiples of four: no code for what is behind the last one (of which the 16-bit kernels had more than of all else, and
// fetched it from memory where they run for a few microseconds)
template <typename T>
__device__ __forceinline__ void put_four(T* row, int d, int size, const float (&f)[4]) {
  if (d >= size) return;
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = from_f<T>(f[i]);
  __builtin_memcpy(row + d, t, sizeof(t));
}

// low bits of a word of 32 (or 64) keys: those in front of `seen`
__device__ __forceinline__ uint32_t first_bits(int seen) { return seen >= 32 ? ~0u : seen <= 0 ? 0u : (1u << seen) - 1; }

int differ_args(const char* what, const nnvhip_differ_args* d, bool backward, DifferArgs* a);

// lse of a row as the exponent's offset in powers of two; a row without keys takes no part (exp2(s - inf) = 0), one with missing values does
__device__ __forceinline__ float offset_of(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// Which template takes a head size: chunks of 16 values of a map's head, of 32 of v's.
#define DIFFER_BY_HEAD(CALL, T, ...)                \
  do {                                              \
    if (a.head <= 32) CALL<T, 2>(__VA_ARGS__);      \
    else if (a.head <= 48) CALL<T, 3>(__VA_ARGS__); \
    else if (a.head <= 64) CALL<T, 4>(__VA_ARGS__); \
    else if (a.head <= 80) CALL<T, 5>(__VA_ARGS__); \
    else if (a.head <= 96) CALL<T, 6>(__VA_ARGS__); \
    else CALL<T, 8>(__VA_ARGS__);                   \
  } while (0)
#define DIFFER_BY_TYPE(type, CALL, ...)                                             \
  do {                                                                              \
    if ((type) == NNVHIP_TYPE_F32) DIFFER_BY_HEAD(CALL, float, __VA_ARGS__);        \
    else if ((type) == NNVHIP_TYPE_BF16) DIFFER_BY_HEAD(CALL, bf16_t, __VA_ARGS__); \
    else DIFFER_BY_HEAD(CALL, f16_t, __VA_ARGS__);                                  \
  } while (0)

// Tiles of 32 rows in LDS for the kernels with f32 products: a row is the two maps' parts (16 CH values each) and the wide one (32 CH).  Four floats more a
// row, so that the 16-byte reads of one column of 16 rows, and the reads of 16 columns of rows 4 apart, meet every bank once.
template <int CH>
struct F32Tile {
  static constexpr int ROWS = 32, LD = 64 * CH + 4, FLOATS = ROWS * LD;
};
// 32 rows on their way there: NT threads, four values of PER places each.  FOUR: the head is a multiple of 4.
template <typename T, int CH, int NT, bool FOUR>
struct TripleAhead {
  static constexpr int PER = 512 * CH / NT;
  RawFour<T> r[PER];
  // map(j, m), wide(j): pointers of row j's parts, of rows that exist
  template <class Map, class Wide>
  __device__ __forceinline__ void load(Map map, Wide wide, int head, int tid) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = p * NT + tid, j = at / (16 * CH), c = at % (16 * CH), m = c >= 4 * CH;
      const bool third = c >= 8 * CH;
      const T* row = third ? wide(j) : map(j, m);
      const int d = 4 * (third ? c - 8 * CH : c - m * 4 * CH), size = third ? 2 * head : head;
      if constexpr (FOUR) r[p].load(row, d, size);
      else r[p].load_any(row, d, size);
    }
  }
  // rows whose bit of `valid` is not set are zeros, as is what lies behind the head
  __device__ __forceinline__ void store(float* tile, uint32_t valid, int head, int tid) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = p * NT + tid, j = at / (16 * CH), c = at % (16 * CH), m = c >= 4 * CH;
      const bool third = c >= 8 * CH;
      const int d = 4 * (third ? c - 8 * CH : c - m * 4 * CH), size = third ? 2 * head : head;
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = (valid >> j & 1) && d + i < size ? r[p][i] : 0.0f;
      __builtin_memcpy(tile + j * F32Tile<CH>::LD + 4 * c, f, 16);
    }
  }
};

// Products on v_mfma_f32_16x16x4_f32.  Lane l holds column l % 16 of a product and its rows 4 (l / 16) + i; as operands, row or column l % 16 and index
// l / 16 of the summed four.  So a product's registers are the right operand of the next one as they stand, if its left operand takes the
// summed rows in that order, and a row's values are taken four at a time: 16 c + 4 (l / 16) + j in step 4 c + j.
__device__ __forceinline__ float4_t mfma4(float x, float y, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0); }

// s[k] = the products over N chunks of 16 values of the tile's rows 16 k + l % 16 (at: the tile, at the lane's row and 4 (l / 16) of the part) with a column's
// values f
template <int CH, int N>
__device__ __forceinline__ void f32_over_head(const float* at, const float (&f)[N][4], float4_t (&s)[2]) {
  constexpr int LD = F32Tile<CH>::LD;
#pragma unroll
  for (int k = 0; k < 2; ++k) s[k] = float4_t{0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < N; ++c) {
    float x[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) __builtin_memcpy(x[k], at + 16 * k * LD + 16 * c, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) s[k] = mfma4(x[k][j], f[c][j], s[k]);
  }
}
// acc[d] += the products over the tile's 32 rows of its columns 16 d + l % 16 (at: the tile, at row 4 (l / 16) and column l % 16 of the part) with p
template <int CH, int N>
__device__ __forceinline__ void f32_over_rows(const float* at, const float4_t (&p)[2], float4_t (&acc)[N]) {
  constexpr int LD = F32Tile<CH>::LD;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int d = 0; d < N; ++d) acc[d] = mfma4(at[(16 * k + j) * LD + 16 * d], p[k][j], acc[d]);
}
// a column's values, as f32_over_head takes them
template <typename T, int N>
__device__ __forceinline__ void f32_operands(const T* row, int q4, int size, bool there, float (&f)[N][4]) {
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const Four x = load_four(row, 16 * c + 4 * q4, size, there);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[c][j] = x.v[j];
  }
}
template <int N>
__device__ __forceinline__ void f32_zero(float4_t (&acc)[N]) {
#pragma unroll
  for (int d = 0; d < N; ++d) acc[d] = float4_t{0, 0, 0, 0};
}
template <bool FOUR, typename T, int N>
__device__ __forceinline__ void f32_store(T* row, const float4_t (&acc)[N], float by, int q4, int size) {
#pragma unroll
  for (int d = 0; d < N; ++d) {
    const float f[4] = {acc[d][0] * by, acc[d][1] * by, acc[d][2] * by, acc[d][3] * by};
    if constexpr (FOUR) put_four(row, 16 * d + 4 * q4, size, f);
    else store_four(row, 16 * d + 4 * q4, size, f);
  }
}
// which of the 8 keys (or rows) 16 k + 4 q4 + i of 32 a lane's registers are
__device__ __forceinline__ bool f32_bit(uint32_t word, int k, int i, int q4) { return word >> (16 * k + 4 * q4 + i) & 1; }

// over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quarters_max(float x) { return fmaxf(fmaxf(x, __shfl_xor(x, 16, 64)), fmaxf(__shfl_xor(x, 32, 64), __shfl_xor(x, 48, 64))); }
__device__ __forceinline__ float quarters_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

}  // namespace nnvhip
