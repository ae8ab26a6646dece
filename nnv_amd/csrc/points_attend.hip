// Attention of points, forward: the kernels for every type, head size and alignment.
//
// The products are f32 ones, whatever the type of the tensors (points_attend_split.h): f32 tensors keep f32 results, and tensors of 16 bits, which
// come here where their rows cannot be moved in 16-byte pieces, lose nothing but their final rounding.  That costs them: 2 x 4096 x 4096, 32 heads of 128
// (8 for keys), in bf16 takes 1620 us here and 508 on attend16_wide_kernel; a single token, 2 x 65536 keys of 8 heads of 128, 240 and 95.
#include "points_attend_split.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

// One pass over the keys with the running maximum and sum of every query's softmax: what both kernels do with the scores of a tile.
// s: scores in powers of two; valid: which keys count, from this half's on.  Returns what the sums so far are to be multiplied with.
__device__ __forceinline__ float softmax_step(float16_t& s, uint32_t valid, float& m, float& total) {
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = (valid >> product_row(i, 0)) & 1 ? s[i] : -INFINITY;
    top = fmaxf(top, s[i]);
  }
  top = fmaxf(m, max_of_halves(top));
  const float base = top == -INFINITY ? 0.0f : top;   // no key of this row counts yet
  const float fade = exp2_(m - base);
  m = top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = exp2_(s[i] - base);
    sum += s[i];
  }
  total = total * fade + sum;
  return fade;
}

// Many rows: 32 a wave, 128 a block, whose waves share the tiles of keys; products in pieces.
// Where there are too few blocks for the chip, the keys are split over `splits` blocks, and join_kernel puts their results together.
//
// Bound by the vector units: cutting numbers into pieces and the softmax take as long as the six products.  4 x 1024 x 1024 in f32, 16 heads of 64:
// 120 us, 143 TFLOP/s (a large f32 product of a library: 154), 4 of them for infinities; 8 heads of 128, one wave a SIMD: 132 us, 130 TFLOP/s.
template <typename T, int DP, bool FOUR>
__global__ __launch_bounds__(256, DP <= 96 || sizeof(T) == 2 ? 2 : 1) void attend_kernel(const AttendArgs a) {
  constexpr int R = kWaveRows, PIECES = kPieces<T>;
  __shared__ __attribute__((aligned(1024))) bf16_t ks[PIECES * R * DP], vs[PIECES * R * DP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
  int64_t at = blockIdx.x;
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int bkv = at / a.row_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int tiles = (n + R - 1) / R, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = (int64_t)row_tile * 128 + wave * R + col;
  const bool row_here = r < a.rows, idle = (int64_t)row_tile * 128 + wave * R >= a.rows;
  const unsigned rows_at = rows_place<bf16_t, DP>(lane), columns_at = columns_place<bf16_t, DP>(lane);
  RowPieces<DP, PIECES> qf;
  qf.load((const T*)a.q.p + (row_here ? row_at(a.q, a, b, kv, r) : 0), h, a.head, row_here);
  const float unit = a.scale * kLog2e;
  float16_t acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  float m = -INFINITY, total = 0.0f;
  const T* kp = (const T*)a.k.p + b * a.k.b + kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  RowsAhead<T, DP, 256, FOUR> k_next, v_next;
  typename RowsAhead<T, DP, 256, FOUR>::Words words;
  int counts = 0;
  auto fetch = [&](int t) {
    auto word = [&](int j) { return key_word(a, b, t * R + j, n); };
    words.load(word, threadIdx.x);
    k_next.load([&](int j) { return kp + min(t * R + j, n - 1) * a.k.t; }, a.head, threadIdx.x);
    v_next.load([&](int j) { return vp + min(t * R + j, n - 1) * a.v.t; }, a.head, threadIdx.x);
    counts = key_word(a, b, t * R + col, n);
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    auto counting = [](int word) { return word != 0; };
    store_tile<DP, PIECES>(k_next, ks, words, counting, a.head, threadIdx.x);
    store_tile<DP, PIECES>(v_next, vs, words, counting, a.head, threadIdx.x);
    const uint32_t valid = (uint32_t)__ballot(counts != 0) >> (4 * h);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    if (idle) continue;
    float16_t s = split_over_head<DP, PIECES, true>(hide(lds_addr_of(ks) + rows_at), [&](int k, int c) { return qf.f[k][c]; });
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= unit;
    const float fade = softmax_step(s, valid, m, total);
    if (__any(fade != 1.0f))
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
    split_over_rows<DP, PIECES, true>(hide(lds_addr_of(vs) + columns_at), s, acc);
  }
  total = sum_of_halves(total);
  if (!row_here) return;
  const int64_t flat = (int64_t)bkv * a.rows + r, heads_rows = (int64_t)a.batch * a.kv_heads * a.rows;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (h == 0) (a.splits > 1 ? a.part_lse[split * heads_rows + flat] : a.lse[flat]) = total == 0.0f ? -INFINITY : (m + log2f(total)) * kLn2;
  float* part = a.splits > 1 ? a.part + (split * heads_rows + flat) * a.head : nullptr;
  T* out = (T*)a.out + dense_row_at(a, b, kv, r);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = acc[d][4 * i4 + i] * inv;
      const int at_d = d * 32 + 8 * i4 + 4 * h;
      if (part) store_four(part, at_d, a.head, f);
      else store_four(out, at_d, a.head, f);
    }
}

// What the four waves of a block found for its rows ([wave][row][DP + 4 values], with each row's maximum and sum), joined and written.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void join_waves(const AttendArgs& a, const float* found, const float (&row_max)[4][ROWS], const float (&row_total)[4][ROWS],
                                           int split, int bkv, int row_tile) {
  constexpr int LD = DP + 4;
  for (int e = threadIdx.x; e < ROWS * (DP / 4); e += 256) {
    const int j = e / (DP / 4), d = e % (DP / 4) * 4;
    const int64_t rj = (int64_t)row_tile * ROWS + j;
    if (rj >= a.rows) continue;
    float top = row_max[0][j], all = 0.0f, w[4], f[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 1; k < 4; ++k) top = fmaxf(top, row_max[k][j]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = exp2_(row_max[k][j] - base);
      all += w[k] * row_total[k][j];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] += w[k] * found[(k * ROWS + j) * LD + d + i];
    }
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= inv;
    const int64_t fj = (int64_t)bkv * a.rows + rj;
    const int b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
    const float lse = all == 0.0f ? -INFINITY : (top + log2f(all)) * kLn2;
    const int64_t sj = (int64_t)split * a.batch * a.kv_heads * a.rows + fj;
    if (d == 0) (a.splits > 1 ? a.part_lse[sj] : a.lse[fj]) = lse;
    if (d >= a.head) continue;
    if (a.splits > 1) store_four(a.part + sj * a.head, d, a.head, f);
    else store_four((T*)a.out + dense_row_at(a, b, kv, rj), d, a.head, f);
  }}

// Few rows, many keys for each (single tokens): 32 rows for the block, whose four waves take the tiles of keys in turn, each with LDS of its
// own; what they found is joined at the end.  On the f32 matrix instructions: the keys and values are read once, and cutting each of them into
// pieces would cost more than the instructions.  (64 queries on 8 x 1500 f32 keys, 16 heads of 64: 50 us, in attend_kernel 42; a single token on 16 x 1500:
// 50 here, 61 there.  So this kernel takes up to 32 rows.)
template <typename T, int DP, bool FOUR>
__global__ __launch_bounds__(256) void attend_few_kernel(const AttendArgs a) {
  constexpr int R = kWaveRows, LD = DP + 4;
  __shared__ float lds[4 * 2 * R * LD];
  __shared__ float row_max[4][R], row_total[4][R];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
  int64_t at = blockIdx.x;
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int bkv = at / a.row_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int tiles = (n + R - 1) / R, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per + wave, t1 = min(tiles, split * per + per);
  const int64_t r = (int64_t)row_tile * R + col;
  const bool row_here = r < a.rows;
  float* ks = lds + wave * 2 * R * LD;
  float* vs = ks + R * LD;

  float qf[DP / 8][4];
  {
    const T* q = (const T*)a.q.p + (row_here ? row_at(a.q, a, b, kv, r) : 0);
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      const Four f = load_four<T>(q, 8 * c + 4 * h, a.head, row_here);
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[c][j] = f.v[j] * (a.scale * kLog2e);
    }
  }
  float16_t acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  float m = -INFINITY, total = 0.0f;

  const T* kp = (const T*)a.k.p + b * a.k.b + kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  RowsAhead<T, DP, 64, FOUR> ks_next, vs_next;
  typename RowsAhead<T, DP, 64, FOUR>::Words words;
  int counts = 0;
  auto fetch = [&](int t) {
    auto word = [&](int j) { return key_word(a, b, t * R + j, n); };
    words.load(word, lane);
    ks_next.load([&](int j) { return kp + min(t * R + j, n - 1) * a.k.t; }, a.head, lane);
    vs_next.load([&](int j) { return vp + min(t * R + j, n - 1) * a.v.t; }, a.head, lane);
    counts = key_word(a, b, t * R + col, n);
  };
  auto wave_barrier = [] {   // LDS written by other lanes of the wave
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; t += 4) {
    wave_barrier();
    // rows of DP + 4 floats: a quarter wave's 16-byte reads of one column block then touch every bank once
    auto counting = [](int word) { return word != 0; };
    ks_next.store([&](int j, int d, const float(&f)[4]) { __builtin_memcpy(ks + j * LD + d, f, 16); }, words, counting, a.head, lane);
    vs_next.store([&](int j, int d, const float(&f)[4]) { __builtin_memcpy(vs + j * LD + d, f, 16); }, words, counting, a.head, lane);
    const uint32_t valid = (uint32_t)__ballot(counts != 0) >> (4 * h);
    wave_barrier();
    if (t + 4 < t1) fetch(t + 4);

    float16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      float kf[4];
      __builtin_memcpy(kf, ks + col * LD + 8 * c + 4 * h, 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[c][j], s, 0, 0, 0);
    }
    const float fade = softmax_step(s, valid, m, total);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vs[product_row(i, h) * LD + d * 32 + col], s[i], acc[d], 0, 0, 0);
    }
  }
  total = sum_of_halves(total);

  __syncthreads();
  float* mine = lds + wave * R * LD;   // [row][d] of this wave
  if (h == 0) {
    row_max[wave][col] = m;
    row_total[wave][col] = total;
  }
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) mine[col * LD + d * 32 + product_row(i, h)] = acc[d][i];
  __syncthreads();
  join_waves<T, DP, R>(a, lds, row_max, row_total, split, bkv, row_tile);
}

// 32 rows of f32 on their way from global memory to a wave's own tile in LDS, row after row, with no registers in between: 16 bytes a
// lane and transfer.  The pieces of a row change places by the row, so that 16 rows' pieces of one column, and (heads of 64 and 128) the two
// halves of what 32 lanes read of a row each, meet every bank once.
template <int DP>
struct FewTile {
  static constexpr int PIECES = DP / 4, PER = 32 * PIECES / 64;
  unsigned off[PER], there;   // bytes behind the tile's address; whether place i holds values of the head
  __device__ __forceinline__ static int place(int row) {
    if constexpr (DP % 64 == 0) return (row & 3) | (row >> 3 & 1) << 2 | (row >> 2 & 1) << 3;
    else return row >> 1 & 7;
  }
  __device__ __forceinline__ static int row(int i, int lane) { return (i * 64 + lane) / PIECES; }
  __device__ __forceinline__ static int value(int i, int lane) { return ((i * 64 + lane) % PIECES ^ place(row(i, lane))) * 4; }
  __device__ __forceinline__ void init(int lane, int head, int64_t stride) {
    there = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      off[i] = 4 * (row(i, lane) * (unsigned)stride + value(i, lane));
      there |= value(i, lane) < head ? 1u << i : 0;
    }
  }
  // rows 32 t ... of those from p on; past the last of n, that one again.  Every transfer takes part, if not with every lane: it holds a whole row.
  __device__ __forceinline__ void issue(int t, int n, const float* p, int64_t stride, unsigned lds, int lane) const {
    if (t * 32 + 32 <= n) {
      const float* tile = p + t * 32 * stride;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (there >> i & 1) lds_dma16((const double*)tile, off[i], __builtin_amdgcn_readfirstlane(lds + i * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (there >> i & 1)
          lds_dma16_at((const double*)(p + min(t * 32 + row(i, lane), n - 1) * stride + value(i, lane)), __builtin_amdgcn_readfirstlane(lds + i * 1024));
    }
  }
};

// Up to 16 rows of f32, aligned (single tokens): as attend_few_kernel, on the 16x16x4 instructions.  Lane l holds column l % 16 of a product and
// its rows 4 (l / 16) + i.  A wave's keys and values go to LDS by themselves, one tile of each: the next keys are asked for when the scores
// are formed, the next values when they are multiplied, so that always one tile is on its way, mostly two.
//
// Bound by memory: 2 x 32768 keys of 8 heads of 128 (32 of queries) take 100 us, 5.3 TB/s; in attend_few_kernel, whose rows go through registers, 145.
// 16 x 1500 keys by length, 16 heads of 64: 38 us, 4.0 TB/s (50).
template <int DP>
__global__ __launch_bounds__(256) void attend_few_f32_kernel(const AttendArgs a) {
  constexpr int R = 32, TILE = R * DP, LD = DP + 4, ROWS = 16, PER = FewTile<DP>::PER;
  __shared__ __attribute__((aligned(1024))) float lds[4 * 2 * TILE];
  __shared__ float row_max[4][ROWS], row_total[4][ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q4 = lane >> 4;
  int64_t at = blockIdx.x;
  const int split = at % a.splits;
  const int bkv = at / a.splits, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int tiles = (n + R - 1) / R, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per + wave, t1 = min(tiles, split * per + per);
  const bool row_here = col < a.rows;
  float* ks = lds + wave * 2 * TILE;
  float* vs = ks + TILE;
  const unsigned ks_at = lds_addr_of(ks), vs_at = ks_at + 4 * TILE;
  if (DP != a.head) {   // the columns behind the head size, for good
    for (int e = threadIdx.x; e < 4 * 2 * TILE; e += 256) lds[e] = 0.0f;
    __syncthreads();
  }
  const float* kp = (const float*)a.k.p + b * a.k.b + kv * a.k.h;
  const float* vp = (const float*)a.v.p + b * a.v.b + kv * a.v.h;
  FewTile<DP> k_load, v_load;
  k_load.init(lane, a.head, a.k.t);
  v_load.init(lane, a.head, a.v.t);
  if (t0 < t1) {
    k_load.issue(t0, n, kp, a.k.t, ks_at, lane);
    v_load.issue(t0, n, vp, a.v.t, vs_at, lane);
  }
  Four qf[DP / 16];   // values 16 c + 4 (l / 16) .. + 3 of row l % 16
#pragma unroll
  for (int c = 0; c < DP / 16; ++c)
    qf[c] = load_four((const float*)a.q.p + (row_here ? row_at(a.q, a, b, kv, col) : 0), 16 * c + 4 * q4, a.head, row_here);
  const float unit = a.scale * kLog2e;
  float4_t acc[DP / 32][2];   // values 32 d + 8 (l / 16) + 2 i + j of row l % 16 in acc[d][j][i]
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d][0] = acc[d][1] = float4_t{0, 0, 0, 0};
  float base = -INFINITY, total = 0.0f;
  unsigned words = 0;   // which keys of 32 tiles count, tile i in lane i
  for (int t = t0, turn = 0; t < t1; t += 4, ++turn) {
    uint32_t valid;
    if (a.mask == nullptr) {
      const int rest = n - t * R;
      valid = rest >= R ? ~0u : (1u << rest) - 1;
    } else {
      // (a wait for one of a mask's bytes is a wait for all transfers ahead of it: those of 32 tiles at a time)
      if (turn % 32 == 0)
        for (int i = 0; i < 32; ++i) {
          const unsigned word = (unsigned)__ballot(t + 4 * i < t1 && key_counts(a, b, (t + 4 * i) * R + lane % R, n));
          words = lane == i ? word : words;
        }
      valid = (unsigned)__builtin_amdgcn_readlane(words, turn % 32);
    }
    wave_arrived<PER>();   // the keys; the values may still be on their way
    float4_t s[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) s[k] = float4_t{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float f[4];
        __builtin_memcpy(f, ks + (16 * k + col) * DP + ((4 * c + q4) ^ FewTile<DP>::place(16 * k + col)) * 4, 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[j], qf[c].v[j], s[k], 0, 0, 0);
      }
    phase_wait();
    if (t + 4 < t1) k_load.issue(t + 4, n, kp, a.k.t, ks_at, lane);
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[k][i] = valid >> (16 * k + 4 * q4 + i) & 1 ? s[k][i] * unit : -INFINITY;
        top = fmaxf(top, s[k][i]);
      }
    top = fmaxf(base, max_of_quarters(top));
    const float off = top == -INFINITY ? 0.0f : top, fade = exp2_(base - off);
    base = top;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[k][i] = exp2_(s[k][i] - off);
        sum += s[k][i];
      }
    total = total * fade + sum;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d][0] *= fade, acc[d][1] *= fade;
    if (t + 4 < t1) wave_arrived<PER>();
    else wave_arrived<0>();
    if (valid != ~0u) {   // a weight of zero must meet a zero
#pragma unroll 1
      for (int e = (int)hide(lane); e < R * (DP / 4); e += 64)
        if (!(valid >> (e / (DP / 4)) & 1)) {
          const float none[4] = {0, 0, 0, 0};
          __builtin_memcpy(vs + 4 * e, none, 16);
        }
      phase_wait();
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const int row = 16 * k + 4 * q4 + i;
          float f[2];
          __builtin_memcpy(f, vs + row * DP + ((8 * d + col / 2) ^ FewTile<DP>::place(row)) * 4 + col % 2 * 2, 8);
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[d][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[j], s[k][i], acc[d][j], 0, 0, 0);
        }
    phase_wait();
    if (t + 4 < t1) v_load.issue(t + 4, n, vp, a.v.t, vs_at, lane);
  }
  total = sum_of_quarters(total);

  __syncthreads();
  float* mine = lds + wave * ROWS * LD;   // [row][d] of this wave
  if (q4 == 0) {
    row_max[wave][col] = base;
    row_total[wave][col] = total;
  }
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) mine[col * LD + d * 32 + 8 * q4 + 2 * i + j] = acc[d][j][i];
  __syncthreads();
  join_waves<float, DP, ROWS>(a, lds, row_max, row_total, split, bkv, 0);
}

// o = sum over splits of exp(lse_s - lse) o_s, in the order of the splits within SLICES slices and of the slices: SLICES * 32 threads a
// row, four values and every SLICES-th split each.  Eight slices where there are more than eight splits, else one.  (Single tokens on 2 x 65536 keys, 64
// rows of 32 splits: 94 us with, 98 without; 64 queries on 8 x 1500 keys, 8192 rows of few splits: 30 us with, 22 without.)
template <typename T, int SLICES>
__global__ __launch_bounds__(256) void join_kernel(const AttendArgs a) {
  constexpr int ROWS = 8 / SLICES;
  __shared__ float tops[8], totals[8], found[8][32][4];
  const int64_t all = (int64_t)a.batch * a.kv_heads * a.rows;
  const int slot = threadIdx.x / 32, slice = slot % SLICES, lane = threadIdx.x % 32, d = lane * 4;
  const int64_t flat = (int64_t)blockIdx.x * ROWS + slot / SLICES;
  const bool here = flat < all;
  float top = -INFINITY;
  if (here)
    for (int s = slice * 32 + lane; s < a.splits; s += SLICES * 32) top = fmaxf(top, a.part_lse[s * all + flat]);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
  if constexpr (SLICES > 1) {
    if (lane == 0) tops[slot] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SLICES; ++k) top = fmaxf(top, tops[slot - slice + k]);
  }
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, f[4] = {0, 0, 0, 0};
  if (here)
    for (int s = slice; s < a.splits; s += SLICES * 4) {
      Four p[4];
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int sk = s + k * SLICES;
        const bool one = sk < a.splits;
        p[k] = load_four(a.part + ((one ? sk : 0) * all + flat) * a.head, d, a.head, one);
        w[k] = one ? a.part_lse[sk * all + flat] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = exp2_((w[k] - base) * kLog2e);
        total += e;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] += e * p[k].v[i];
      }
    }
  if constexpr (SLICES > 1) {
    if (lane == 0) totals[slot] = total;
#pragma unroll
    for (int i = 0; i < 4; ++i) found[slot][lane][i] = f[i];
    __syncthreads();
    if (slice) return;
#pragma unroll
    for (int k = 1; k < SLICES; ++k) {
      total += totals[slot + k];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] += found[slot + k][lane][i];
    }
  }
  if (!here) return;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] *= inv;
  const int bkv = (int)(flat / a.rows), b = bkv / a.kv_heads;
  if (d < a.head) store_four((T*)a.out + dense_row_at(a, b, bkv % a.kv_heads, flat % a.rows), d, a.head, f);
  if (lane == 0) a.lse[flat] = total == 0.0f ? -INFINITY : base + log2f(total) * kLn2;
}

// How a forward call is cut: few rows for each head's keys (single tokens) or tiles of many rows (128, or 256 where attend16_wide_kernel
// takes the call), and over how many blocks the keys are split.
//
// Few are up to 64 rows of 16 bits, two tiles: 64 queries on 8 x 1500 keys, 16 heads of 64, take 17.5 us so and 22.3 as many; 96 take 25.5 and 25.0, with heads
// of 128 on 4096 keys 91 and 64.  (f32: see attend_few_kernel.)
//
// Splits (see split_of): without, the single tokens on 2 x 65536 keys take 704 us instead of 94, 4 x 1024 x 1024 in f32 5 more.  Two tiles of keys are
// the least for a split in f32: 96 queries on 477 keys, 8 heads of 80, take 20.7 us, with four 24.6.  The costs of a start and of a join in 16 bits
// are higher, since a tile takes less: with 4 and 5 for 6 and 12, 2 x 538 x 1597, 2 heads of 128, takes 29 us instead of 25, 224 x 512, 16 of 32, 17 instead of 14.
struct Cut {
  bool few;
  int row_tiles, splits;
};
Cut cut_of(int64_t batch, int64_t kv_heads, int64_t rows, int64_t keys, int64_t head, bool by16) {
  Cut c;
  c.few = rows <= (by16 ? 2 : 1) * kWaveRows;
  c.row_tiles = (int)ceil_div(rows, c.few ? kWaveRows : by16 ? attend16_tile(head) : 128);
  // blocks that the chip holds at once; what starting a block, and joining splits, costs in tiles of 32 keys
  const int64_t slots = c.few || head > (by16 ? 64 : 96) ? 256 : 512;
  const int64_t start = c.few ? 16 : by16 ? 6 : 2, join = c.few ? 16 : by16 ? 12 : 3;
  c.splits = split_of(batch * kv_heads * c.row_tiles, ceil_div(keys, kWaveRows), c.few ? 8 : by16 ? 4 : 2, slots, start, join);
  return c;
}

// f32 rows can be moved in 16-byte pieces, and the offsets in a tile of 32 fit 31 bits
inline bool by_fours(const TokenView& t, int64_t head) {
  return t.t >= 0 && t.t < (int64_t(1) << 24) && head % 4 == 0 && t.b % 4 == 0 && t.t % 4 == 0 && t.h % 4 == 0 && (uintptr_t)t.p % 16 == 0;
}

template <typename T, int DP>
void launch_attend(const AttendArgs& a, bool few, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits));
  const bool four = a.head % 4 == 0;
  if constexpr (sizeof(T) == 4)
    if (a.rows <= 16 && by_fours(a.k, a.head) && by_fours(a.v, a.head)) {
      hipLaunchKernelGGL((attend_few_f32_kernel<DP>), grid, dim3(256), 0, st, a);
      return;
    }
  if (few && four) hipLaunchKernelGGL((attend_few_kernel<T, DP, true>), grid, dim3(256), 0, st, a);
  else if (few) hipLaunchKernelGGL((attend_few_kernel<T, DP, false>), grid, dim3(256), 0, st, a);
  else if (four) hipLaunchKernelGGL((attend_kernel<T, DP, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attend_kernel<T, DP, false>), grid, dim3(256), 0, st, a);
}
template <typename T, int>
void launch_join(const AttendArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows;
  if (a.splits > 8) hipLaunchKernelGGL((join_kernel<T, 8>), dim3((unsigned)rows), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((join_kernel<T, 1>), dim3((unsigned)ceil_div(rows, 8)), dim3(256), 0, st, a);
}

// The sizes have to fit the kernels' indexes: a key and a row of a key/value head 31 bits, with room for a tile behind the last one; the rest
// is counted in 64.  And the threads of a grid have to be below 2^32.
int check_sizes(const char* what, const nnvhip_attention* d) {
  if (!known_type(d->type)) NNV_FAIL(NNVHIP_ERR_ARG, "%s: the values are f32, bf16 or f16", what);
  if (d->batch < 0 || d->queries < 0 || d->keys < 0) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: negative size", what);
  if (d->head < 1 || d->head > 128) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: heads of 1 to 128 values are supported", what);
  if (d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads)
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: the number of heads must be a multiple of the number of key/value heads", what);
  const int64_t most = (int64_t(1) << 31) - 256, group = d->heads / d->kv_heads;
  if (d->batch > 65535 || d->heads > 65535 || d->keys > most || d->queries > most / group) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  // (at least so many blocks, first, for the sums by which splits are chosen)
  if (d->batch * d->kv_heads * ceil_div(d->queries * group, 256) > kMostBlocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  for (const bool by16 : {false, true}) {
    const Cut c = cut_of(d->batch, d->kv_heads, d->queries * group, d->keys, d->head, by16);
    if (d->batch * d->kv_heads * c.row_tiles * c.splits > kMostBlocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  }
  return NNVHIP_OK;
}

}  // namespace

int attend_args(const char* what, const nnvhip_attention* d, bool backward, AttendArgs* a) {
  if (!d) NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  NNV_TRY(check_sizes(what, d));
  if (!(std::fabs(d->scale) <= FLT_MAX)) NNV_FAIL(NNVHIP_ERR_ARG, "%s: the scale must be a finite number of f32", what);
  auto view = [](const void* p, const int64_t (&s)[3]) { return TokenView{p, s[0], s[1], s[2]}; };
  *a = AttendArgs{};
  a->q = view(d->q, d->q_stride);
  a->k = view(d->k, d->k_stride);
  a->v = view(d->v, d->v_stride);
  a->go = view(d->go, d->go_stride);
  a->o = TokenView{d->o, d->queries * d->heads * d->head, d->heads * d->head, d->head};
  a->out = d->o;
  a->dq = d->dq;
  a->dk = d->dk;
  a->dv = d->dv;
  a->lse = d->lse;
  a->lengths = d->key_lengths;
  a->mask = d->key_mask;
  a->mask_b = d->mask_stride[0];
  a->mask_k = d->mask_stride[1];
  a->batch = (int)d->batch;
  a->queries = (int)d->queries;
  a->keys = (int)d->keys;
  a->kv_heads = (int)d->kv_heads;
  a->group = (int)(d->heads / d->kv_heads);
  a->head = (int)d->head;
  a->rows = d->queries * a->group;
  a->scale = (float)d->scale;
  const bool no_rows = d->batch == 0 || d->queries == 0, no_keys = d->batch == 0 || d->keys == 0;
  if ((!no_rows && (!d->q || !d->o || !d->lse)) || (!no_rows && !no_keys && (!d->k || !d->v)) ||
      (backward && ((!no_rows && (!d->go || !d->dq)) || (!no_keys && (!d->dk || !d->dv)))))
    NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  return NNVHIP_OK;
}

}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_cross_attention_workspace(const nnvhip_attention* d, int64_t* bytes) {
  if (!d || !bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  NNV_TRY(check_sizes("nnvhip_cross_attention_workspace", d));
  int splits = 1;   // whichever kernels the alignment of the tensors lets take the call
  for (const bool by16 : {false, true})
    splits = std::max(splits, cut_of(d->batch, d->kv_heads, d->queries * (d->heads / d->kv_heads), d->keys, d->head, by16).splits);
  *bytes = splits > 1 ? (int64_t)splits * d->batch * d->heads * d->queries * (d->head + 1) * (int64_t)sizeof(float) : 0;
  return NNVHIP_OK;
}

int nnvhip_cross_attention(nnvhip_ctx* ctx, const nnvhip_attention* d, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  AttendArgs a;
  NNV_TRY(attend_args("nnvhip_cross_attention", d, false, &a));
  int64_t need = 0;
  NNV_TRY(nnvhip_cross_attention_workspace(d, &need));
  if (need > workspace_bytes || (need && !workspace))
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_cross_attention: a workspace of %lld bytes is needed", (long long)need);
  if (a.batch == 0 || a.rows == 0) return NNVHIP_OK;
  const bool by16 = attend16_takes(a, (int)d->type);
  const Cut c = cut_of(a.batch, a.kv_heads, a.rows, a.keys, a.head, by16);
  a.row_tiles = c.row_tiles;
  a.splits = c.splits;
  a.part = static_cast<float*>(workspace);
  a.part_lse = c.splits > 1 ? a.part + (int64_t)c.splits * a.batch * a.kv_heads * a.rows * a.head : nullptr;
  if (by16) launch_attend16(a, (int)d->type, c.few, (hipStream_t)stream);
  else ATTEND_BY_TYPE(d->type, launch_attend, a, c.few, (hipStream_t)stream);
  if (c.splits > 1) ATTEND_BY_TYPE(d->type, launch_join, a, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
