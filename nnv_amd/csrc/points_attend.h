// Attention of points to another sequence's states: what the forward and the backward kernels share.
//
//   S = scale q k^T,  lse = log sum over the keys that count of exp(S),  P = exp(S - lse),  o = P v
//   D = rowsum(do o),  dS = P (do v^T - D),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T do
//
// Rows.  The heads / kv_heads heads that share keys and values are taken as more rows of one product: row r of (sequence b,
// key/value head) is query r % queries of the group's head r / queries.  A tile of keys then serves all of them, a
// single token of a group of heads fills a tile as far as the group goes, and the gradients of shared keys and values are sums
// over rows like any other.  lse, D and the partial results are indexed by (b, key/value head, row), which is the
// (b, head, query) order of the caller's lse.
//
// Every product is formed so that what comes out of one is what the next one takes in.  The 32x32 matrix instructions
// leave lane l column l % 32 and rows 8 (i / 4) + 4 (l / 32) + i % 4 (i = 0 .. 15) of a product, and take as right operand
// column l % 32 and a slice of the summed index.  So the scores are formed transposed, S^T = k q^T: a lane holds 16 keys of one
// query, row sums and largest values need one exchange with lane l ^ 32, and P^T is the right operand of o^T = v^T P^T as it
// stands, if the left operand takes its keys in the same order.
#pragma once
#include "points.h"

#include <algorithm>

namespace nnvhip {

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef float float4_t __attribute__((ext_vector_type(4)));

struct TokenView {   // batch x tokens x heads x head, the last index dense
  const void* p;
  int64_t b, t, h;   // strides in elements
};

struct AttendArgs {
  TokenView q, k, v, o, go;   // go: the gradient of o
  void* out;                  // o of the forward pass, dense
  void *dq, *dk, *dv;         // dense
  float* lse;                 // batch x heads x queries
  const int32_t* lengths;     // batch, or null
  const uint8_t* mask;        // batch x keys, or null
  int64_t mask_b, mask_k;
  int batch, queries, keys, kv_heads, group, head;
  int64_t rows;               // group * queries, below 2^31
  float scale;
  int row_tiles, key_tiles, splits;
  float* delta;               // D, batch x heads x queries
  float* part;                // partial results of the splits
  float* part_lse;
};

__device__ __forceinline__ int keys_that_count(const AttendArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
}
__device__ __forceinline__ bool key_counts(const AttendArgs& a, int b, int key, int n) {
  return key < n && (a.mask == nullptr || a.mask[b * a.mask_b + key * a.mask_k] != 0);
}
// The same as a number that is zero where the key does not count: a mask's byte as it was loaded, so that nothing waits for it
// before it is used.
__device__ __forceinline__ int key_word(const AttendArgs& a, int b, int key, int n) {
  if (a.mask == nullptr) return key < n;
  return a.mask[b * a.mask_b + min(key, n - 1) * a.mask_k] & (key < n ? 0xff : 0);
}
// offset of row r of (b, kv) in a token view
__device__ __forceinline__ int64_t row_at(const TokenView& t, const AttendArgs& a, int b, int kv, int64_t r) {
  const int64_t g = (uint32_t)r / (uint32_t)a.queries, i = r - g * a.queries;
  return b * t.b + i * t.t + (kv * (int64_t)a.group + g) * t.h;
}
// ... and in a dense tensor of that shape
__device__ __forceinline__ int64_t dense_row_at(const AttendArgs& a, int b, int kv, int64_t r) {
  const int64_t g = (uint32_t)r / (uint32_t)a.queries, i = r - g * a.queries;
  return ((b * (int64_t)a.queries + i) * a.kv_heads * a.group + kv * (int64_t)a.group + g) * a.head;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// the row of a 32x32 product that register i of a lane's half h holds
__device__ __forceinline__ int product_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

struct Four {
  float v[4];
};
// four elements at d, d + 1, ... of a row of `head`; those that do not exist, and all of them if !there, are zero
template <typename T>
__device__ __forceinline__ Four load_four(const T* row, int d, int head, bool there) {
  Four f;
  if (there && d + 4 <= head) {
    T t[4];
    __builtin_memcpy(t, row + d, sizeof(t));
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = to_f(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = there && d + i < head ? to_f(row[d + i]) : 0.0f;
  }
  return f;
}
template <typename T>
__device__ __forceinline__ void store_four(T* row, int d, int head, const float (&f)[4]) {
  if (d + 4 <= head) {
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = from_f<T>(f[i]);
    __builtin_memcpy(row + d, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < head) row[d + i] = from_f<T>(f[i]);
  }
}

constexpr int kWaveRows = 32;  // rows of a wave's tile on either side
constexpr int64_t kMostBlocks = (int64_t(1) << 23) - 1;   // of up to 512 threads: a grid has fewer than 2^32

// Four elements as the words they are loaded as (see Pack): what is asked for a tile ahead is taken apart, and found not to
// count, when it is stored, so that nothing waits for it before.  For the same reason no lane takes another way than its neighbours: what lies
// behind the head is read from the head's end, and zero when it is stored.
template <typename T>
struct RawFour {
  unsigned w[sizeof(T)];
  __device__ __forceinline__ void load(const T* row, int d, int head) {   // head is a multiple of 4
    __builtin_memcpy(w, row + min(d, head - 4), 4 * sizeof(T));
  }
  __device__ __forceinline__ void load_any(const T* row, int d, int head) {
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = row[min(d + i, head - 1)];
    __builtin_memcpy(w, t, sizeof(t));
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return to_f(__builtin_bit_cast(T, w[i]));
    else return to_f(__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1)))));
  }
};

// 32 rows of a token view on their way to LDS: NT threads, four values of PER rows each.  FOUR: the head is a multiple of 4.
template <typename T, int DP, int NT, bool FOUR>
struct RowsAhead {
  static constexpr int PER = kWaveRows * DP / 4 / NT;
  RawFour<T> r[PER];
  struct Words {   // what says of the same rows whether they count
    int w[PER];
    template <class Word>
    __device__ __forceinline__ void load(Word word_of, int tid) {
#pragma unroll
      for (int p = 0; p < PER; ++p) w[p] = word_of((p * NT + tid) / (DP / 4));
    }
  };
  // row(j): pointer of row j, one that exists
  template <class Row>
  __device__ __forceinline__ void load(Row row, int head, int tid) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = p * NT + tid, j = at / (DP / 4), d = at % (DP / 4) * 4;
      if constexpr (FOUR) r[p].load(row(j), d, head);
      else r[p].load_any(row(j), d, head);
    }
  }
  // to(j, d, f): takes the values d .. d + 3 of row j; those of a row for which counts(word) is false are zero
  template <class To, class Counts>
  __device__ __forceinline__ void store(To to, const Words& words, Counts counts, int head, int tid) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = p * NT + tid, j = at / (DP / 4), d = at % (DP / 4) * 4;
      const bool ok = counts(words.w[p]);
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = ok && d + i < head ? r[p][i] : 0.0f;
      to(j, d, f);
    }
  }
};

// The arguments of the kernels from the caller's; what it checks, it reports as `what`.
int attend_args(const char* what, const nnvhip_attention* d, bool backward, AttendArgs* a);
// Over how many blocks one axis of `tiles` tiles is split where there are `blocks` blocks without: the number for which the rounds of
// `slots` blocks that the chip holds, times the tiles of a block and what starting one costs, take least, the joining of what
// they leave (where there is any) counted in.  No split gets fewer than `least` tiles.  For 144 blocks of 19 tiles in 512 slots: 3.
inline int split_of(int64_t blocks, int64_t tiles, int64_t least, int64_t slots, int64_t start, int64_t join) {
  if (blocks <= 0) return 1;
  int64_t best = 1, cost = ceil_div(blocks, slots) * (tiles + start);
  for (int64_t s = 2; s <= std::min<int64_t>(tiles / least, 256) && blocks * s <= 4 * slots; ++s) {
    const int64_t c = ceil_div(blocks * s, slots) * (ceil_div(tiles, s) + start) + join;
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return (int)best;
}

#define ATTEND_BY_HEAD(CALL, T, ...)                 \
  do {                                               \
    if (a.head <= 32) CALL<T, 32>(__VA_ARGS__);      \
    else if (a.head <= 64) CALL<T, 64>(__VA_ARGS__); \
    else if (a.head <= 96) CALL<T, 96>(__VA_ARGS__); \
    else CALL<T, 128>(__VA_ARGS__);                  \
  } while (0)
#define ATTEND_BY_TYPE(type, CALL, ...)                                        \
  do {                                                                         \
    if ((type) == NNVHIP_TYPE_F32) ATTEND_BY_HEAD(CALL, float, __VA_ARGS__);   \
    else if ((type) == NNVHIP_TYPE_BF16) ATTEND_BY_HEAD(CALL, bf16_t, __VA_ARGS__); \
    else ATTEND_BY_HEAD(CALL, f16_t, __VA_ARGS__);                             \
  } while (0)

}  // namespace nnvhip
