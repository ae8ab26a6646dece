// f32 products on the bf16 matrix instructions.  Cut into three pieces of 8 significant bits, an f32 is exactly
//   x = x0 + x1 + x2,   x0 = the upper 16 bits of x, x1 = those of x - x0, x2 = the rest,
// each a bf16.  Of the nine products of two such numbers the six largest are formed, exactly, and added up in f32; the three left out are
// below 2^-24 of the result, where an f32 product rounds as well.  Six products of 32x32x16 take 192 cycles; the f32 instructions
// (32x32x2) take 512 for the same.
#pragma once
#include "points_attend16.h"

namespace nnvhip {

typedef half8<bf16_t> piece8;

// The pieces of four numbers, two to a word.  (An infinity's rest is zero, not inf - inf.)
struct Pieces4 {
  unsigned w[3][2];
};
__device__ __forceinline__ unsigned upper_halves(float a, float b) {   // of a in the lower half of the word, of b in the upper one
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302);
}
__device__ __forceinline__ float cut(float x) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u); }
__device__ __forceinline__ void cut_pair(float a, float b, unsigned (&w)[3]) {
  w[0] = upper_halves(a, b);
  const float a1 = fabsf(a) < INFINITY ? a - cut(a) : 0.0f, b1 = fabsf(b) < INFINITY ? b - cut(b) : 0.0f;
  w[1] = upper_halves(a1, b1);
  w[2] = upper_halves(a1 - cut(a1), b1 - cut(b1));
}

// Tiles of 32 rows in three planes, a Rows16 tile each.
template <int DP>
struct Planes {
  static constexpr int VALUES = 32 * DP, BYTES = 2 * VALUES;   // of one plane
};
// Rows of a token view on their way to a tile's planes: NT threads, four values at a time.
template <typename T, int DP, int NT>
struct SplitStage {
  static constexpr int PER = 32 * DP / 4 / NT;
  Four r[PER];
  template <class Row, class There>
  __device__ __forceinline__ void load(Row row, There there, int head, int tid) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = p * NT + tid, j = at / (DP / 4), d = at % (DP / 4) * 4;
      const bool ok = there(j);
      r[p] = load_four<T>(ok ? row(j) : (const T*)nullptr, d, head, ok);
    }
  }
  __device__ __forceinline__ void store(bf16_t* planes, int tid) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int at = p * NT + tid, j = at / (DP / 4), d = at % (DP / 4) * 4;
      unsigned a[3], b[3];
      cut_pair(r[p].v[0], r[p].v[1], a);
      cut_pair(r[p].v[2], r[p].v[3], b);
      bf16_t* to = planes + Rows16<bf16_t, DP>::at(j, d / 8) + d % 8;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const unsigned w[2] = {a[k], b[k]};
        __builtin_memcpy(to + k * Planes<DP>::VALUES, w, 8);
      }
    }
  }
};

// The operands of a lane's row (values 16 c + 8 h .. + 7), in pieces.
template <int DP>
struct RowPieces {
  piece8 f[3][DP / 16];
  template <typename T>
  __device__ __forceinline__ void load(const T* row, int h, int head, bool there, float by) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const Four lo = load_four(row, 16 * c + 8 * h, head, there), hi = load_four(row, 16 * c + 8 * h + 4, head, there);
      unsigned w[4][3];
      cut_pair(lo.v[0] * by, lo.v[1] * by, w[0]);
      cut_pair(lo.v[2] * by, lo.v[3] * by, w[1]);
      cut_pair(hi.v[0] * by, hi.v[1] * by, w[2]);
      cut_pair(hi.v[2] * by, hi.v[3] * by, w[3]);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const unsigned v[4] = {w[0][k], w[1][k], w[2][k], w[3][k]};
        __builtin_memcpy(&f[k][c], v, 16);
      }
    }
  }
};

// The six products of two numbers in pieces: the small ones into `rest`, so that they are added up among themselves first.
__device__ __forceinline__ void multiply(const piece8 (&x)[3], const piece8& f0, const piece8& f1, const piece8& f2, float16_t& s, float16_t& rest) {
  rest = Half8<bf16_t>::mfma(x[2], f0, rest);
  s = Half8<bf16_t>::mfma(x[0], f0, s);
  rest = Half8<bf16_t>::mfma(x[0], f2, rest);
  rest = Half8<bf16_t>::mfma(x[1], f1, rest);
  rest = Half8<bf16_t>::mfma(x[1], f0, rest);
  rest = Half8<bf16_t>::mfma(x[0], f1, rest);
}

// The product over the head of a tile's 32 rows with a row's pieces.  at: LDS address of the planes + rows_place; f(k, c): piece k.
template <int DP, class F>
__device__ __forceinline__ float16_t split_over_head(unsigned at, F f) {
  float16_t s, rest;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = rest[i] = 0.0f;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    piece8 x[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) x[k] = rows_operand<bf16_t, DP>(at + k * Planes<DP>::BYTES, 0, c);
    multiply(x, f(0, c), f(1, c), f(2, c), s, rest);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] += rest[i];
  return s;
}
// acc[d] += the product over a tile's 32 rows with a product's registers p.  at: LDS address of the planes + columns_place.
template <int DP>
__device__ __forceinline__ void split_over_rows(unsigned at, const float16_t& p, float16_t (&acc)[DP / 32]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    piece8 f[3];
    unsigned w[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) cut_pair(p[8 * c + 2 * i], p[8 * c + 2 * i + 1], w[i]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const unsigned v[4] = {w[0][k], w[1][k], w[2][k], w[3][k]};
      __builtin_memcpy(&f[k], v, 16);
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      piece8 x[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) x[k] = columns_operand<bf16_t, DP>(at + k * Planes<DP>::BYTES, 16 * c, d);
      multiply(x, f[0], f[1], f[2], acc[d], acc[d]);
    }
  }
}

}  // namespace nnvhip
