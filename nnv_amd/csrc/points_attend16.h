// Attention of points in 16 bits: tiles of rows in LDS, as the bf16 / f16 matrix instructions (32x32x16) take them.
#pragma once
#include "lds_dma.h"
#include "points_attend.h"

namespace nnvhip {

template <typename T>
struct Half8;
template <>
struct Half8<bf16_t> {
  typedef bf16_t t __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float16_t mfma(t a, t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Half8<f16_t> {
  typedef f16_t t __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float16_t mfma(t a, t b, float16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <typename T>
using half8 = typename Half8<T>::t;

typedef short short4_t __attribute__((ext_vector_type(4)));

// ROWS rows of DP values in LDS, row after row, filled by 16-byte transfers from global memory (the head size is a multiple of
// 8, so a transfer holds values of one row only; those past the head size are zeroed once and never written again).
//
// Two readers: over_head takes 16 bytes of 32 rows at one column, over_rows (through the transposing read) 64 bytes of 4 rows
// at a time.  Both meet every bank once if the 16-byte pieces of a row are exchanged by
//   piece ^ (row / 4 % 4 + 4 (row % 4 or what of it moves whole groups of four pieces within the row)):
// four consecutive rows then have the same 64-byte group in different quarters of the 256 bytes that the banks span, and rows 4
// apart have the same piece in different places of a group.  (Rows of 32, 96 and 160 values do the first by themselves.)  GROUP: the pieces
// within which they change places.
template <typename T, int DP>
struct Rows16 {
  static constexpr int PIECES = DP / 8, GROUP = DP % 128 == 0 ? 16 : DP % 64 == 0 ? 8 : 4;
  static __device__ __forceinline__ int place(int row) {
    const int low = (row >> 2) & 3;
    if constexpr (GROUP == 16) return (row & 3) << 2 | low;
    if constexpr (GROUP == 8) return (row >> 1 & 1) << 2 | low;
    return low;
  }
  static __device__ __forceinline__ int at(int row, int piece) { return row * DP + ((piece ^ place(row)) << 3); }
};

// A lane's place in a tile for either reader, from which every other read is an exclusive or with a constant and an offset in the
// instruction.  (hide() keeps the compiler from holding all those addresses in registers over the loop.)
__device__ __forceinline__ unsigned hide(unsigned at) {
  asm("" : "+v"(at));
  return at;
}
template <typename T, int DP>
__device__ __forceinline__ unsigned rows_place(int lane) {
  return 2 * Rows16<T, DP>::at(lane & 31, lane >> 5);
}
template <typename T, int DP>
__device__ __forceinline__ unsigned columns_place(int lane) {
  const int h = lane >> 5, j = (lane >> 2) & 3, piece = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  return 2 * (Rows16<T, DP>::at(4 * h + j, piece) + (lane & 1) * 4);
}
// Left operand of a product over the head: rows first .. first + 31, values 16 c .. 16 c + 15 (lane: row first + lane % 32, 8 of
// them).  at: LDS address of the tile + rows_place.
template <typename T, int DP>
__device__ __forceinline__ half8<T> rows_operand(unsigned at, int first, int c) {
  constexpr int G = Rows16<T, DP>::GROUP;
  const unsigned x = (at ^ (c % (G / 2) << 5)) + c / (G / 2) * (G * 16) + first * DP * 2;
  return *(const __attribute__((address_space(3))) half8<T>*)x;
}
// Left operand of a product over rows: values 32 d .. 32 d + 31 (lane: value 32 d + lane % 32) of the 16 rows first + product_row(0..7, h)
// of the lane's half: the order in which a product's registers 0-7 (or 8-15, for the 16 rows behind) hold them.
// ds_read_b64_tr_b16 gives lane i of 16 the i-th value of four rows whose 16 values the lanes 4 j .. 4 j + 3 point to.
// at: LDS address of the tile + columns_place.
template <typename T, int DP>
__device__ __forceinline__ half8<T> columns_operand(unsigned at, int first, int d) {
  constexpr int G = Rows16<T, DP>::GROUP;
  short4_t r[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const unsigned x = (at ^ (half << 5 | d % (G / 4) << 6)) + d / (G / 4) * (G * 16) + (first + 8 * half) * DP * 2;
    r[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)x);
  }
  half8<T> f;
  __builtin_memcpy(&f, r, 16);
  return f;
}

// s[k] = the product over the head of rows first + 32 k .. first + 32 k + 31 of a tile with a row's operands f.  The LDS reads go a batch
// (of up to four) ahead of the products that use them (left to itself the compiler puts every read right in front of its product), and
// the products of a batch alternate between the independent results.  begin() may stand ahead of other work.
template <typename T, int DP, int K, int MOST = 4>
struct OverHead {
  static constexpr int N = K * (DP / 16), BATCH = N % 4 == 0 && MOST == 4 ? 4 : N % 3 == 0 && MOST > 2 ? 3 : 2;
  half8<T> x[2][BATCH];
  __device__ __forceinline__ void read(unsigned tile, int first, int n) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int at = n * BATCH + i;
      x[n & 1][i] = rows_operand<T, DP>(tile, first + 32 * (at % K), at / K);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void begin(unsigned tile, int first) { read(tile, first, 0); }
  __device__ __forceinline__ void finish(unsigned tile, int first, const half8<T> (&f)[DP / 16], float16_t (&s)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[k][i] = 0.0f;
#pragma unroll
    for (int n = 0; n < N / BATCH; ++n) {
      if (n + 1 < N / BATCH) read(tile, first, n + 1);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int at = n * BATCH + i;
        s[at % K] = Half8<T>::mfma(x[n & 1][i], f[at / K], s[at % K]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};
template <typename T, int DP, int K, int MOST = 4>
__device__ __forceinline__ void over_head(unsigned tile, int first, const half8<T> (&f)[DP / 16], float16_t (&s)[K]) {
  OverHead<T, DP, K, MOST> o;
  o.begin(tile, first);
  o.finish(tile, first, f, s);
}

// Eight f32 of a product as the right operand of the next one, each rounded to T.
template <typename T>
__device__ __forceinline__ half8<T> round8(const float16_t& s, int first) {
  half8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (T)s[first + i];
  return r;
}

// The weights of the softmax are multiples of exp(score - the largest score): in f16 of 2^7, so that what is rounded to T keeps weights down to 2^-32 of the
// largest (2^-25 without; a million keys of 2^-26 would be lost), and the largest, which the offset may lag behind by 2^8, stays in f16's range.  (A weight that is rounded to zero gives NaN with an infinite value.)
template <typename T>
constexpr float kLift = std::is_same_v<T, f16_t> ? 7.0f : 0.0f;

// Exponents are score * unit - off in one rounding, off a rounded score * unit: where a rounding is more than a fraction of an exponent, the two do not
// fit together, and a weight may leave the range of its type.  From there on the products are rounded as off is (round_scores), and off is that of the largest,
// not lower by kLift, which might be less than half a place.
constexpr float kFar = 4194304.0f;   // 2^22: places of 1/2
template <typename T>
__device__ __forceinline__ float lowered(float top) {
  return fabsf(top) > kFar ? top : top - kLift<T>;
}
template <int K>
__device__ __forceinline__ void round_scores(float16_t (&s)[K], float unit) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[k][i] = rounded(s[k][i] * unit);
}

// The transfers a wave makes for a pair of tiles (a and b) of ROWS rows each, PER_TILE transfers of 1024 bytes a tile, shared out
// over WAVES waves.  Tiles of evenly spaced rows need no arithmetic on vectors: a scalar address for the tile and an offset that a lane
// keeps (64-bit products of vectors would take as long as a quarter of a tile's exponentials).
template <typename T, int DP, int ROWS, int WAVES>
struct PairLoad {
  static constexpr int PIECES = DP / 8, PER_TILE = ROWS * PIECES / 64, COUNT = 2 * PER_TILE / WAVES;
  static constexpr bool EVEN = PER_TILE % WAVES == 0;        // a wave has the same places in both tiles
  static constexpr int PLACES = EVEN ? COUNT / 2 : COUNT;
  static_assert(2 * PER_TILE % WAVES == 0 && ROWS * PIECES % 64 == 0, "transfers come out even");
  unsigned off_a[PLACES], off_b[EVEN ? PLACES : 1];   // bytes behind the tile's address (not EVEN: of whichever tile the place is in)
  unsigned there;                                     // bit i: place i holds values of the head (not what is behind them)
  __device__ __forceinline__ static int row(int i, int wave, int lane) { return ((i * WAVES + wave) % PER_TILE * 64 + lane) / PIECES; }
  __device__ __forceinline__ static int value(int i, int wave, int lane) {
    const int at = (i * WAVES + wave) % PER_TILE * 64 + lane;
    return (at % PIECES ^ Rows16<T, DP>::place(at / PIECES)) * 8;
  }
  __device__ __forceinline__ void init(int wave, int lane, int head, int64_t stride_a, int64_t stride_b) {
    there = 0;
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int r = row(i, wave, lane), v = value(i, wave, lane);
      const bool in_a = EVEN || i * WAVES + wave < PER_TILE;
      off_a[i] = 2 * (unsigned)(r * (unsigned)(in_a ? stride_a : stride_b) + v);
      if constexpr (EVEN) off_b[i] = 2 * (unsigned)(r * (unsigned)stride_b + v);
      there |= v < head ? 1u << i : 0;
    }
  }
  // tiles whose rows follow one another from pa and pb
  __device__ __forceinline__ void issue(const T* pa, const T* pb, unsigned lds, int wave) const {
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int at = i * WAVES + wave;
      if (there >> i & 1) {
        if constexpr (EVEN) {
          lds_dma16((const double*)pa, off_a[i], __builtin_amdgcn_readfirstlane(lds + at * 1024));
          lds_dma16((const double*)pb, off_b[i], __builtin_amdgcn_readfirstlane(lds + (PER_TILE + at) * 1024));
        } else {
          lds_dma16((const double*)(at < PER_TILE ? pa : pb), off_a[i], __builtin_amdgcn_readfirstlane(lds + at * 1024));
        }
      }
    }
  }
  // tiles whose rows are anywhere: a(row), b(row) are pointers to them
  template <class A, class B>
  __device__ __forceinline__ void issue_any(A a, B b, unsigned lds, int wave, int lane) const {
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int at = i * WAVES + wave, r = row(i, wave, lane), v = value(i, wave, lane);
      if (there >> i & 1) {
        if constexpr (EVEN) {
          lds_dma16_at((const double*)(a(r) + v), __builtin_amdgcn_readfirstlane(lds + at * 1024));
          lds_dma16_at((const double*)(b(r) + v), __builtin_amdgcn_readfirstlane(lds + (PER_TILE + at) * 1024));
        } else {
          lds_dma16_at((const double*)((at < PER_TILE ? a(r) : b(r)) + v), __builtin_amdgcn_readfirstlane(lds + at * 1024));
        }
      }
    }
  }
  // tile ta of a and tile tb of b, of rows that follow one another from pa and pb and end after n: rows past the last one repeat it
  __device__ __forceinline__ void issue_tiles(int ta, int tb, int n, const T* pa, int64_t stride_a, const T* pb, int64_t stride_b, unsigned lds,
                                              int wave, int lane) const {
    const int fa = ta * ROWS, fb = tb * ROWS;
    if (max(fa, fb) + ROWS <= n)
      issue(pa + fa * stride_a, pb + fb * stride_b, lds, wave);
    else
      issue_any([&](int r) { return pa + min(fa + r, n - 1) * stride_a; }, [&](int r) { return pb + min(fb + r, n - 1) * stride_b; }, lds, wave,
                lane);
  }
  // tile t of both
  __device__ __forceinline__ void issue_tile(int t, int n, const T* pa, int64_t stride_a, const T* pb, int64_t stride_b, unsigned lds, int wave,
                                             int lane) const {
    issue_tiles(t, t, n, pa, stride_a, pb, stride_b, lds, wave, lane);
  }
};

// All but the last N transfers of a wave have arrived, and no access to LDS is moved ahead of that.
template <int N>
__device__ __forceinline__ void wave_arrived() {
  __builtin_amdgcn_sched_barrier(0);
  wait_vm<N>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_sched_barrier(0);
}
// A wave's LDS accesses are done, and no instruction is moved across.
__device__ __forceinline__ void phase_wait() {
  __builtin_amdgcn_sched_barrier(0);
  wait_vm_lds<63>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_sched_barrier(0);
}
// A barrier that no instruction is moved across, in front of which a wave's LDS reads are done.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  wait_vm_lds<63>();
  block_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// The rows of a tile that do not take part, made zeros by a wave for itself: a weight of zero must meet a zero.  Every wave that reads the
// tile does so before its own reads, and no wave waits for another.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void zero_rows(T* tile, uint64_t valid, int lane) {
  half8<T> none = {};
#pragma unroll 1
  for (int e = (int)hide(lane); e < ROWS * (DP / 8); e += 64)   // rarely taken: nothing of it is to be kept in registers
    if (!(valid >> (e / (DP / 8)) & 1)) __builtin_memcpy(tile + e * 8, &none, 16);
  wait_vm_lds<63>();
  __builtin_amdgcn_wave_barrier();
}

// the larger of a value and that of lane l ^ 32
__device__ __forceinline__ float max_of_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
// over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_of_quarters(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return max_of_halves(fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])));
}
__device__ __forceinline__ float sum_of_quarters(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return sum_of_halves(__builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]));
}
// max(a, b, c) without the extra instructions that make fmaxf quiet signalling NaNs
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// the largest value of K products' registers: in chains that take turns, for one after the other would wait for each result
template <int K>
__device__ __forceinline__ float largest(const float16_t (&s)[K]) {
  float top[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
  for (int e = 0; e < 16 * K; e += 8)
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = max3(top[j], s[e / 16][e % 16 + 2 * j], s[e / 16][e % 16 + 2 * j + 1]);
  return max3(max3(top[0], top[1], top[2]), top[3], top[3]);
}

// Block `id` of `total` in an order in which each of the 8 XCDs gets consecutive ones (blocks are dealt to the XCDs in turn):
// blocks that read the same keys then find them in one L2.  (The sequences of a batch, whose lengths may differ, follow one another
// within a head, beginning with another one in each: every XCD and every CU gets some of each.)  In the order of the blocks' numbers 8 x 448 x 1500 by length
// takes 44.5 us instead of 41.4, the gradients of 4 x 2048 x 2048, 16 heads of 64, 294 instead of 286; heads of 128 the same.
__device__ __forceinline__ int64_t xcd_order(int64_t id, int64_t total) {
  const int64_t x = id % 8, base = total / 8, more = total % 8;
  return x * base + min(x, more) + id / 8;
}

// A head's row can be moved in 16-byte pieces: head size, strides and start are multiples of 8 values.  And the offsets in a tile of 64 rows
// fit 31 bits.
inline bool by_pieces(const TokenView& t, int64_t head) {
  return t.t >= 0 && t.t < (int64_t(1) << 24) && head % 8 == 0 && t.b % 8 == 0 && t.t % 8 == 0 && t.h % 8 == 0 && (uintptr_t)t.p % 16 == 0;
}

// Whether the 16-bit kernels take a call; else the general ones do.
bool attend16_takes(const AttendArgs& a, int type);
bool grad16_takes(const AttendArgs& a, int type);
int attend16_tile(int64_t head);   // rows of a block, unless few
void launch_attend16(const AttendArgs& a, int type, bool few, hipStream_t st);
void launch_query_grad16(const AttendArgs& a, hipStream_t st);   // tiles of 256 rows
void launch_key_grad16(const AttendArgs& a, hipStream_t st);     // tiles of key_grad16_tile(head) keys
int key_grad16_tile(int64_t head);

}  // namespace nnvhip
