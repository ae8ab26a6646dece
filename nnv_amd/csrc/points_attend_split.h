// f32 products on the bf16 matrix instructions.  Cut into three pieces of 8 significant bits, an f32 is exactly
//   x = x0 + x1 + x2,   x0 = x rounded to bf16, x1 = x - x0 rounded to bf16, x2 = the rest (8 bits, by then),
// each a bf16, x1 no more than 2^-8 of x and x2 2^-17.  Of the nine products of two such numbers the six largest are formed, exactly, and
// added up in f32; the three left out are below 2^-24 of the result, what an f32 product's rounding is, and of either sign.  (Cut off instead of
// rounded, they are up to 2^-7 and 2^-15 and have its sign: up to 2^-21 is left out, 0.7 of 2^-24 on the mean, always towards zero.)  Six products of
// 32x32x16 take 192 cycles; the f32 instructions (32x32x2) take 512 for the same.
//
// An infinity's first piece is all of it, and its products with the other's small pieces are NaN where those are zero.  So a score that is not finite by its
// first product is that; and the weights that meet values have their pieces cut off, so that none is below zero, and raised to the smallest number at
// least (cut_weights).  (Asked for only where a tile holds an infinity: 120 us for 4 x 1024 x 1024, 16 heads of 64, as always.  The gradients of
// what meets an infinity are infinite or NaN, with or without: there it would take 4 % of the time.)
//
// Numbers of 16 bits have two pieces (a bf16 one, an f16 two, of 8 and 3 bits): four products are all of theirs.  Two pieces of a softmax's
// weight, 16 bits, are five more than the result keeps: three products with those.  (The gradients of 3 x 2304 x 302, 48 heads of 80, 12 for keys, in f16: 690 us;
// with three pieces half as much again.)
#pragma once
#include "points_attend16.h"

namespace nnvhip {

typedef half8<bf16_t> piece8;
template <typename T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : 2;

__device__ __forceinline__ unsigned upper_halves(float a, float b) {   // of a in the lower half of the word, of b in the upper one
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302);
}
__device__ __forceinline__ float cut(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u); }
__device__ __forceinline__ unsigned rounded_halves(float a, float b) {   // the same, to nearest
  typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 r = {(bf16_t)a, (bf16_t)b};
  return __builtin_bit_cast(unsigned, r);
}
__device__ __forceinline__ float lower_half(unsigned w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float upper_half(unsigned w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
// The pieces of two numbers, each piece of both in a word.
__device__ __forceinline__ void cut_pair(float a, float b, unsigned (&w)[3]) {
  w[0] = rounded_halves(a, b);
  const float a1 = a - lower_half(w[0]), b1 = b - upper_half(w[0]);
  w[1] = rounded_halves(a1, b1);
  w[2] = upper_halves(a1 - lower_half(w[1]), b1 - upper_half(w[1]));
}
// The same for numbers that bf16 would round to infinity, or that are infinite (their rest is zero, not inf - inf): the first piece cut off.
constexpr float kRoundsUp = 3.396177e38f;   // below the largest bf16 and half of its last place
__device__ __forceinline__ void cut_large(float a, float b, unsigned (&w)[3]) {
  const bool fa = fabsf(a) < INFINITY, fb = fabsf(b) < INFINITY;
  w[0] = rounded_halves(fa ? cut(a) : a, fb ? cut(b) : b);
  const float a1 = fa ? a - cut(a) : 0.0f, b1 = fb ? b - cut(b) : 0.0f;
  w[1] = upper_halves(a1, b1);
  w[2] = upper_halves(a1 - cut(a1), b1 - cut(b1));
}
// max(x, |a|, |b|); what is no number is left out
__device__ __forceinline__ float max_of_sizes(float x, float a, float b) {
  asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(x) : "v"(a), "v"(b));
  return x;
}
// LARGE: with cut_large.  What takes many numbers cuts them the quick way, finds their largest size, and where it is kRoundsUp or more, again the other way: a way
// chosen number by number is a branch that nothing is moved across (the gradients of 4 x 512 x 512, 8 heads of 128, 160 us instead of 146).
template <bool LARGE>
__device__ __forceinline__ void cut_four(const float (&f)[4], unsigned (&a)[3], unsigned (&b)[3]) {
  if constexpr (LARGE) {
    cut_large(f[0], f[1], a);
    cut_large(f[2], f[3], b);
  } else {
    cut_pair(f[0], f[1], a);
    cut_pair(f[2], f[3], b);
  }
}

// The pieces of two weights: above zero, except for the first one of a weight of zero.  (Cut off, they leave up to 1.5 2^-23 out of their products with
// rounded pieces, still of either sign.)
__device__ __forceinline__ void cut_weights(float a, float b, unsigned (&w)[3]) {
  typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
  const ushort2_t least = {0x0080, 0x0080};   // 2^-126
  const float a1 = a - cut(a), b1 = b - cut(b);
  w[0] = upper_halves(a, b);
  w[1] = upper_halves(a1, b1);
  w[2] = upper_halves(a1 - cut(a1), b1 - cut(b1));
#pragma unroll
  for (int k = 1; k < 3; ++k) w[k] = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, w[k]), least));
}

// Tiles of 32 rows in planes, a Rows16 tile for each piece.
template <int DP>
struct Planes {
  static constexpr int VALUES = 32 * DP, BYTES = 2 * VALUES;   // of one plane
};
// four values of row j, from d on, into a tile's planes
template <int DP, int PIECES, bool LARGE>
__device__ __forceinline__ void store_pieces(bf16_t* planes, int j, int d, const float (&f)[4]) {
  unsigned a[3], b[3];
  cut_four<LARGE>(f, a, b);
  bf16_t* to = planes + Rows16<bf16_t, DP>::at(j, d / 8) + d % 8;
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    const unsigned w[2] = {a[k], b[k]};
    __builtin_memcpy(to + k * Planes<DP>::VALUES, w, 8);
  }
}
// A thread's share of a tile (RowsAhead) into the tile's planes.
template <int DP, int PIECES, class Ahead, class Counts>
__device__ __forceinline__ void store_tile(const Ahead& ahead, bf16_t* planes, const typename Ahead::Words& words, Counts counts, int head, int tid) {
  float top = 0.0f;
  ahead.store(
      [&](int j, int d, const float(&f)[4]) {
        top = max_of_sizes(max_of_sizes(top, f[0], f[1]), f[2], f[3]);
        store_pieces<DP, PIECES, false>(planes, j, d, f);
      },
      words, counts, head, tid);
  if (__any(top >= kRoundsUp))
    ahead.store([&](int j, int d, const float(&f)[4]) { store_pieces<DP, PIECES, true>(planes, j, d, f); }, words, counts, head, tid);
}

// The operands of a lane's row (values 16 c + 8 h .. + 7), in pieces.
template <int DP, int PIECES>
struct RowPieces {
  piece8 f[PIECES][DP / 16];
  template <bool LARGE, typename T>
  __device__ __forceinline__ float cut_row(const T* row, int h, int head, bool there) {   // returns the largest size
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const Four lo = load_four(row, 16 * c + 8 * h, head, there), hi = load_four(row, 16 * c + 8 * h + 4, head, there);
      top = max_of_sizes(max_of_sizes(top, lo.v[0], lo.v[1]), lo.v[2], lo.v[3]);
      top = max_of_sizes(max_of_sizes(top, hi.v[0], hi.v[1]), hi.v[2], hi.v[3]);
      unsigned w[4][3];
      cut_four<LARGE>(lo.v, w[0], w[1]);
      cut_four<LARGE>(hi.v, w[2], w[3]);
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const unsigned v[4] = {w[0][k], w[1][k], w[2][k], w[3][k]};
        __builtin_memcpy(&f[k][c], v, 16);
      }
    }
    return top;
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, int h, int head, bool there) {
    if (__any(cut_row<false>(row, h, head, there) >= kRoundsUp)) cut_row<true>(row, h, head, there);
  }
};

// The products of two numbers in pieces: the small ones into `rest`, or first, so that they are added up among themselves (and a number times one is that
// number).  ALL: two pieces of either are the whole numbers, and the smallest product counts, too.
template <int PIECES, bool ALL>
__device__ __forceinline__ void multiply(const piece8 (&x)[PIECES], const piece8 (&f)[PIECES], float16_t& s, float16_t& rest) {
  if constexpr (PIECES == 3) rest = Half8<bf16_t>::mfma(x[2], f[0], rest);
  if constexpr (PIECES == 3) rest = Half8<bf16_t>::mfma(x[0], f[2], rest);
  if constexpr (PIECES == 3 || ALL) rest = Half8<bf16_t>::mfma(x[1], f[1], rest);
  rest = Half8<bf16_t>::mfma(x[1], f[0], rest);
  rest = Half8<bf16_t>::mfma(x[0], f[1], rest);
  s = Half8<bf16_t>::mfma(x[0], f[0], s);
}

// The product over the head of a tile's 32 rows with a row's pieces.  at: LDS address of the planes + rows_place; f(k, c): piece k.  What
// one step multiplies is read while the step before it is multiplied (see OverHead).  INFINITE: results that are infinite stay that.
template <int DP, int PIECES, bool INFINITE, class F>
__device__ __forceinline__ float16_t split_over_head(unsigned at, F f) {
  float16_t s, rest;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = rest[i] = 0.0f;
  piece8 x[2][PIECES], y[2][PIECES];
  auto read = [&](int c) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      x[c & 1][k] = rows_operand<bf16_t, DP>(at + k * Planes<DP>::BYTES, 0, c);
      y[c & 1][k] = f(k, c);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  read(0);
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    if (c + 1 < DP / 16) read(c + 1);
    multiply<PIECES, true>(x[c & 1], y[c & 1], s, rest);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] += !INFINITE || fabsf(s[i]) < INFINITY ? rest[i] : 0.0f;
  return s;
}
// acc[d] += the product over a tile's 32 rows with a product's registers p.  at: LDS address of the planes + columns_place.  WEIGHTS: none of p is below
// zero, and infinite numbers of the tile are to stay infinite.
template <int DP, int PIECES, bool WEIGHTS>
__device__ __forceinline__ void split_over_rows(unsigned at, const float16_t& p, float16_t (&acc)[DP / 32]) {
  constexpr int N = 2 * (DP / 32);
  piece8 x[2][PIECES], f[2][PIECES];
  auto read = [&](int n) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) x[n & 1][k] = columns_operand<bf16_t, DP>(at + k * Planes<DP>::BYTES, 16 * (n / (DP / 32)), n % (DP / 32));
  };
  read(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    unsigned w[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (WEIGHTS) cut_weights(p[8 * c + 2 * i], p[8 * c + 2 * i + 1], w[i]);
      else cut_pair(p[8 * c + 2 * i], p[8 * c + 2 * i + 1], w[i]);
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const unsigned v[4] = {w[0][k], w[1][k], w[2][k], w[3][k]};
      __builtin_memcpy(&f[c][k], v, 16);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (n + 1 < N) read(n + 1);
    __builtin_amdgcn_sched_barrier(0);
    const int c = n / (DP / 32), d = n % (DP / 32);
    multiply<PIECES, false>(x[n & 1], f[c], acc[d], acc[d]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace nnvhip
