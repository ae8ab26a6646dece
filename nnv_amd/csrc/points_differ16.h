// Differential attention of points in 16 bits: tiles in LDS of the two maps' rows and the wide ones, as the bf16 / f16 matrix instructions take them.
#pragma once
#include "points_attend16.h"
#include "points_differ.h"

namespace nnvhip {

// Eight values in two pieces: p, rounded towards zero, and what that leaves (to 2^-16 of the value in bf16, 2^-22 in f16).  Both have the value's sign, and
// the second one is not zero where the first one is not (2^-23 of the value are added to it): an infinite number times either piece is the same infinity, and their sum no
// NaN.  (In f16 the second piece of a value below 2^-13 may be zero.)  value(i): the i-th one
template <typename T, class Value>
__device__ __forceinline__ void pieces8(Value value, half8<T>& p, half8<T>& rest) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float x[2] = {value(i), value(i + 1)};   // (floats of their own: the bits of a vector's element are taken of its first one)
    if constexpr (std::is_same_v<T, f16_t>) {
      const auto two = __builtin_amdgcn_cvt_pkrtz(x[0], x[1]);
      p[i] = (T)two[0];
      p[i + 1] = (T)two[1];
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) p[i + j] = __builtin_bit_cast(T, (uint16_t)(__builtin_bit_cast(unsigned, x[j]) >> 16));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) rest[i + j] = (T)fmaf(x[j], 1.0f + 0x1p-23f, -(float)p[i + j]);
  }
}

// A tile of ROWS rows: those of the first map (DP values each, the head rounded up to 32), of the second one, and the wide ones (W, twice the head
// rounded up to 16), each as Rows16 has them, one behind the other.  CH: chunks of 16 values of a map's head.
template <int CH>
struct Width16 {
  static constexpr int W = 32 * CH, DP = (16 * CH + 31) / 32 * 32;
};
template <typename T, int CH, int ROWS, int WAVES, bool SAVE = true>   // SAVE: registers, see EVEN
struct TripleLoad {
  static constexpr int DP = Width16<CH>::DP, W = Width16<CH>::W;
  static constexpr int MAP = ROWS * DP, WIDE = ROWS * W, VALUES = 2 * MAP + WIDE;   // values in LDS
  static constexpr int MAP_COUNT = MAP / 512, WIDE_COUNT = WIDE / 512, TOTAL = 2 * MAP_COUNT + WIDE_COUNT;   // transfers of 1024 bytes
  static constexpr int PLACES = (TOTAL + WAVES - 1) / WAVES, LEAST = TOTAL / WAVES;   // of a wave: at most, at least
  // A wave's places of one kind whose rows are a multiple of 16 apart have their pieces in the same order: an offset for each that is not, and the rest goes
  // into the scalar address (32 places of a single wave would take 32 registers).
  static constexpr bool EVEN = SAVE && MAP_COUNT % WAVES == 0 && WIDE_COUNT % WAVES == 0 && WAVES * 512 % DP == 0 && WAVES * 512 % W == 0;
  static constexpr int MAP_STEP = WAVES * 512 / DP, WIDE_STEP = WAVES * 512 / W;   // rows from one place to the next (EVEN)
  static constexpr int MAPS = MAP_COUNT / WAVES, WIDES = WIDE_COUNT / WAVES;       // places of a kind of tile
  static constexpr int least(int x, int y) { return x < y ? x : y; }
  static constexpr int MAP_OFFS = EVEN ? least(MAPS, 16 / least(16, MAP_STEP)) : 1, WIDE_OFFS = EVEN ? least(WIDES, 16 / least(16, WIDE_STEP)) : 1;
  static_assert(!EVEN || ((MAP_STEP & (MAP_STEP - 1)) == 0 && (WIDE_STEP & (WIDE_STEP - 1)) == 0), "steps of rows are powers of two");
  static constexpr int OFFS = EVEN ? MAP_OFFS + WIDE_OFFS : PLACES;
  unsigned off[OFFS];     // bytes behind the address of the place's tile
  __device__ __forceinline__ static constexpr int place_of(int i) { return i < MAP_OFFS ? i : 2 * MAPS + i - MAP_OFFS; }   // which an offset is of (EVEN)
  unsigned there;         // bit i: the place of offset i holds values of the head (some lane's of every transfer are)
  __device__ __forceinline__ static int tile_of(int at) { return at < MAP_COUNT ? 0 : at < 2 * MAP_COUNT ? 1 : 2; }
  __device__ __forceinline__ static int row(int at, int lane) {
    const int e = (at < 2 * MAP_COUNT ? at % MAP_COUNT : at - 2 * MAP_COUNT) * 64 + lane;
    return at < 2 * MAP_COUNT ? e / (DP / 8) : e / (W / 8);
  }
  __device__ __forceinline__ static int value(int at, int lane) {
    const int e = (at < 2 * MAP_COUNT ? at % MAP_COUNT : at - 2 * MAP_COUNT) * 64 + lane;
    return at < 2 * MAP_COUNT ? (e % (DP / 8) ^ Rows16<T, DP>::place(e / (DP / 8))) * 8 : (e % (W / 8) ^ Rows16<T, W>::place(e / (W / 8))) * 8;
  }
  __device__ __forceinline__ void init(int wave, int lane, int head, int64_t map_stride, int64_t wide_stride) {
    there = 0;
#pragma unroll
    for (int i = 0; i < OFFS; ++i) {
      const int at = (EVEN ? place_of(i) : i) * WAVES + wave;
      off[i] = 0;
      if (at >= TOTAL) continue;
      const int v = value(at, lane);
      off[i] = 2 * (unsigned)(row(at, lane) * (unsigned)(at < 2 * MAP_COUNT ? map_stride : wide_stride) + v);
      there |= v < (at < 2 * MAP_COUNT ? head : 2 * head) ? 1u << i : 0;
    }
  }
  // tiles whose rows follow one another from p0, p1 (the maps) and pw
  __device__ __forceinline__ void issue(const T* p0, const T* p1, const T* pw, int64_t map_stride, int64_t wide_stride, unsigned lds, int wave) const {
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int at = i * WAVES + wave, tile = tile_of(at);
      if constexpr (EVEN) {
        const int j = i < MAPS ? i : i < 2 * MAPS ? i - MAPS : i - 2 * MAPS, each = i < 2 * MAPS ? MAP_OFFS : WIDE_OFFS, o = (i < 2 * MAPS ? 0 : MAP_OFFS) + j % each;
        const T* p = (i < MAPS ? p0 : i < 2 * MAPS ? p1 : pw) + j / each * each * (i < 2 * MAPS ? MAP_STEP * map_stride : WIDE_STEP * wide_stride);
        if (there >> o & 1) lds_dma16((const double*)p, off[o], __builtin_amdgcn_readfirstlane(lds + at * 1024));
        continue;
      }
      if ((i + 1) * WAVES > TOTAL && at >= TOTAL) break;
      if (there >> i & 1) lds_dma16((const double*)(tile == 0 ? p0 : tile == 1 ? p1 : pw), off[i % OFFS], __builtin_amdgcn_readfirstlane(lds + at * 1024));
    }
  }
  // The rows from j0 on and in front of j1, of the same; the others' places are left as they are.  (A scalar address for each run of rows instead of a vector's
  // for each row.  The number of transfers varies: for those who wait for all of them.)
  __device__ __forceinline__ void issue_rows(int j0, int j1, const T* p0, const T* p1, const T* pw, unsigned lds, int wave, int lane) const {
    static_assert(!EVEN, "an offset for every place");
    lane = (int)hide(lane);
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int at = i * WAVES + wave, tile = tile_of(at);
      if ((i + 1) * WAVES > TOTAL && at >= TOTAL) break;
      const int j = row(at, lane);
      if ((there >> i & 1) && j >= j0 && j < j1)
        lds_dma16((const double*)(tile == 0 ? p0 : tile == 1 ? p1 : pw), off[i % OFFS], __builtin_amdgcn_readfirstlane(lds + at * 1024));
    }
  }
  // rows anywhere: map(j, m), wide(j) are pointers to them
  template <class Map, class Wide>
  __device__ __forceinline__ void issue_any(Map map, Wide wide, unsigned lds, int wave, int lane) const {
    lane = (int)hide(lane);   // (rarely taken: nothing of it is to be kept in registers)
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int at = i * WAVES + wave, tile = tile_of(at);
      if ((i + 1) * WAVES > TOTAL && at >= TOTAL) break;
      const int o = !EVEN ? i : i < MAPS ? i % MAP_OFFS : i < 2 * MAPS ? (i - MAPS) % MAP_OFFS : MAP_OFFS + (i - 2 * MAPS) % WIDE_OFFS;
      if (there >> o & 1) {
        const int j = row(at, lane);
        lds_dma16_at((const double*)((tile == 2 ? wide(j) : map(j, tile)) + value(at, lane)), __builtin_amdgcn_readfirstlane(lds + at * 1024));
      }
    }
  }
  // Tile ta of the maps and tile tb of the wide rows, of rows that follow one another and end after n: rows past the last one repeat it (and ones in
  // front of the first one that).
  __device__ __forceinline__ void issue_tiles(int ta, int tb, int n, const T* p, int64_t map_stride, int64_t second_map, const T* pw, int64_t wide_stride,
                                              unsigned lds, int wave, int lane) const {
    const int64_t fa = (int64_t)ta * ROWS, fb = (int64_t)tb * ROWS;
    if (fb >= 0 && max(fa, fb) + ROWS <= n) {
      const T* p0 = p + fa * map_stride;
      issue(p0, p0 + second_map, pw + fb * wide_stride, map_stride, wide_stride, lds, wave);
    } else {
      issue_any([&](int j, int m) { return p + min(fa + j, (int64_t)n - 1) * map_stride + m * second_map; },
                [&](int j) { return pw + min(max(fb + j, (int64_t)0), (int64_t)n - 1) * wide_stride; }, lds, wave, lane);
    }
  }
  // tile t of all
  __device__ __forceinline__ void issue_tile(int t, int n, const T* p, int64_t map_stride, int64_t second_map, const T* pw, int64_t wide_stride,
                                             unsigned lds, int wave, int lane) const {
    issue_tiles(t, t, n, p, map_stride, second_map, pw, wide_stride, lds, wave, lane);
  }
};

// s[k] = the product over N chunks of 16 values of rows first + 32 k .. + 31 of a tile of rows of DP values with a row's operands f(c).  As OverHead: the
// reads go a batch ahead of the products.
template <typename T, int DP, int N, int K, int BATCH, class F>
__device__ __forceinline__ void over_chunks(unsigned tile, int first, F f, float16_t (&s)[K]) {
  constexpr int ALL = N * K, STEPS = (ALL + BATCH - 1) / BATCH;
  half8<T> x[2][BATCH], y[2][BATCH];
  auto read = [&](int n) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int at = n * BATCH + i;
      if (at >= ALL) continue;
      x[n & 1][i] = rows_operand<T, DP>(tile, first + 32 * (at % K), at / K);
      y[n & 1][i] = f(at / K);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[k][i] = 0.0f;
  read(0);
#pragma unroll
  for (int n = 0; n < STEPS; ++n) {
    if (n + 1 < STEPS) read(n + 1);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int at = n * BATCH + i;
      if (at < ALL) s[at % K] = Half8<T>::mfma(x[n & 1][i], y[n & 1][i], s[at % K]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// body(c, d, x): the columns 32 d .. of rows first + 16 c .. + 15 of a tile, read one ahead of what uses them
template <typename T, int DP, int C, class Body>
__device__ __forceinline__ void over_columns(unsigned tile, int first, Body body) {
  constexpr int D = DP / 32;
  half8<T> x[2];
  x[0] = columns_operand<T, DP>(tile, first, 0);
#pragma unroll
  for (int n = 0; n < C * D; ++n) {
    if (n + 1 < C * D) x[(n + 1) & 1] = columns_operand<T, DP>(tile, first + (n + 1) / D * 16, (n + 1) % D);
    body(n / D, n % D, x[n & 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// which keys of a tile of 64 (or 32) keys count, in 32 tiles at a time: a wait for one byte of a mask is a wait for all transfers ahead of it
template <int KEYS>
struct KeyWords {
  unsigned words[KEYS / 32];
  // of tile t, the turn-th that is asked for, step tiles apart, below t1
  __device__ __forceinline__ uint64_t operator()(const DifferArgs& a, int b, int n, int t, int t1, int turn, int step, int lane) {
    if (a.mask == nullptr) {
      const int rest = n - t * KEYS;
      return rest >= KEYS ? ~0ull : (1ull << rest) - 1;
    }
    if (turn % 32 == 0)
      for (int i = 0; i < 32; ++i) {
        const uint64_t word = __ballot(t + i * step < t1 && key_counts(a, b, (t + i * step) * KEYS + lane % KEYS, n));
#pragma unroll
        for (int k = 0; k < KEYS / 32; ++k) words[k] = lane == i ? (unsigned)(word >> (32 * k)) : words[k];
      }
    uint64_t valid = (unsigned)__builtin_amdgcn_readlane(words[0], turn % 32);
    return valid | (KEYS == 64 ? (uint64_t)(unsigned)__builtin_amdgcn_readlane(words[KEYS / 32 - 1], turn % 32) << 32 : valid << 32);
  }
};

template <typename T, int VALUES, int THREADS>
__device__ __forceinline__ void zero_lds(T* lds) {
  half8<T> none = {};
  for (int e = threadIdx.x; e < VALUES / 8; e += THREADS) __builtin_memcpy(lds + e * 8, &none, 16);
  __syncthreads();
}

bool differ16_takes(const DifferArgs& a, int type);
constexpr int kDiffer16Rows = 128;   // of a block
constexpr int kDifferFewRows = 16;   // of a block of the form for few rows
void launch_differ16(const DifferArgs& a, int type, bool few, hipStream_t st);
bool differ_grad16_takes(const DifferArgs& a, int type);
int differ_grad16_tile(int64_t head);       // rows of a block
int differ_key_grad16_tile(int64_t head);   // keys
void launch_differ_query_grad16(const DifferArgs& a, int type, hipStream_t st);
void launch_differ_key_grad16(const DifferArgs& a, int type, hipStream_t st);

}  // namespace nnvhip
