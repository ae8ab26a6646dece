// Attention of points in 16 bits, forward, on v_mfma_f32_32x32x16_{bf16,f16} (2.5 PFLOP/s at best).
#include "points_attend16.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

// FEW = false (heads of up to 64): four waves take 32 rows each and share tiles of 64 keys.  FEW = true (up to 64 rows, single tokens):
// 32 rows for the block, whose 8 waves (4 for heads above 64: LDS) are groups that take tiles of 32 keys in turn; what the groups
// found is joined at the end.  (attend_kernel is the f32 form.)
//
// Tiles are on their way to LDS (no registers in between) STAGES - 1 ahead of the one that is worked on; one barrier a tile.  The running maximum is
// raised only when a row's has grown by more than 2^8: the sums are in f32 and any base serves, so that the accumulators are hardly ever
// multiplied (448 x 1500 by length: 41.4 us, raised with every new maximum 43.0; attend16_wide_kernel's 2 x 4096 x 4096: 516 and 547).
//
// A weight is rounded to T before the product with the values, which adds as much to the error as the result's rounding (bf16: 0.0023 against 64 bits for
// 0.0017), and takes half the products of two pieces.  FEW, which waits for memory, takes two pieces: what rounding leaves is a second weight (single
// tokens as below: 18.0 us for 17.7, 94.5 for 93.7).  The second weights have sums of their own: one may be zero, or below zero, and an infinite value
// times it is not added to what the weight itself makes of that value.
//
// FEW is bound by memory: single tokens on 2 x 65536 keys of 8 heads of 128 (32 of queries) take 94.5 us, 5.0 TB/s; on 16 x 1500 by length, 16 heads of 64, 18 us,
// 4.2 TB/s.  8 groups, where LDS has room for them: 64 such rows on 8 sequences 17.5 us, with 4 groups 23.
// The other form by its two waves a SIMD, which take products and softmax in turn: 8 x 448 x 1500 by length, 16 heads of 64, takes 36 us,
// 475 TFLOP/s.  (Blocks of 64 rows take 52 us, two groups of four waves 36 to 41, three stages instead of four the same, attend16_wide_kernel 38;
// the next tile's scores formed among a tile's exponentials 10 % more.)
constexpr int few_groups(int dp) { return dp > 64 ? 4 : 8; }
template <typename T, int DP, bool FEW>
__global__ __launch_bounds__(FEW ? 64 * few_groups(DP) : 256, FEW ? 1 : 2) void attend16_kernel(const AttendArgs a) {
  constexpr int WAVES = FEW ? 1 : 4, GROUPS = FEW ? few_groups(DP) : 1, STAGES = FEW ? 2 : 4;
  constexpr int KEYS = FEW ? 32 : 64, TILE = KEYS * DP, THREADS = 64 * WAVES * GROUPS;
  typedef PairLoad<T, DP, KEYS, WAVES> Load;
  // STAGES pairs (k, v) of every group; at the end, what the groups found: [group][row][LD values]
  constexpr int ROWS = 32 * WAVES, LD = DP + 4, TILES = GROUPS * STAGES * 2 * TILE, FOUND = GROUPS > 1 ? GROUPS * ROWS * LD * 2 : 0;
  __shared__ __attribute__((aligned(1024))) T lds[TILES > FOUND ? TILES : FOUND];
  __shared__ float row_max[GROUPS][32 * WAVES], row_total[GROUPS][32 * WAVES];
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = any_wave / WAVES, wave = any_wave % WAVES;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int kv = (int)(at / a.row_tiles) / a.batch, b = (int)(at / a.row_tiles + kv) % a.batch, bkv = b * a.kv_heads + kv;
  const int n = keys_that_count(a, b);
  const int tiles = (n + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per + group, t1 = min(tiles, split * per + per);
  const int64_t r = (int64_t)row_tile * (32 * WAVES) + wave * 32 + col;
  const bool row_here = r < a.rows, idle = (int64_t)row_tile * (32 * WAVES) + wave * 32 >= a.rows;
  T* mine = lds + group * STAGES * 2 * TILE;
  const unsigned mine_at = lds_addr_of(mine), rows_at = rows_place<T, DP>(lane), columns_at = columns_place<T, DP>(lane);

  if (DP != a.head) {   // the columns behind the head size, for good
    half8<T> zero = {};
    for (int e = threadIdx.x; e < GROUPS * STAGES * 2 * KEYS * (DP / 8); e += THREADS) __builtin_memcpy(lds + e * 8, &zero, 16);
    __syncthreads();
  }

  // A negative scale is moved into q's sign: the largest score is then the largest product.  (And one of zero is taken as one that
  // leaves every score next to zero, so that the -inf of a key that does not count stays one.)
  const float unit = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
  half8<T> qf[DP / 16];
  {
    const T* q = (const T*)a.q.p + (row_here ? row_at(a.q, a, b, kv, r) : 0);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      qf[c] = half8<T>{};
      if (row_here && 16 * c + 8 * h < a.head) __builtin_memcpy(&qf[c], q + 16 * c + 8 * h, 16);
      if (a.scale < 0) qf[c] = -qf[c];
    }
  }
  float16_t acc[DP / 32], second[FEW ? DP / 32 : 1];   // second: of what the weights' rounding leaves
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = second[FEW ? d : 0][i] = 0.0f;
  float off = -INFINITY, total = 0.0f;   // off: of the exponents, in products times unit
  bool far = false;                      // a row's is beyond kFar

  const T* kp = (const T*)a.k.p + b * a.k.b + kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(wave, lane, a.head, a.k.t, a.v.t);
  auto fetch = [&](int t, int buffer) {
    load.issue_tile(t, n, kp, a.k.t, vp, a.v.t, mine_at + buffer * (4 * TILE), wave, lane);
  };
  // which keys of the next 32 tiles count, tile i in lane i
  unsigned words[KEYS / 32];
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (t0 + s * GROUPS < t1) fetch(t0 + s * GROUPS, s);
  int buffer = 0;
  for (int t = t0, turn = 0; t < t1; t += GROUPS, ++turn) {
    uint64_t valid;
    if (a.mask == nullptr) {
      const int rest = n - t * KEYS;
      valid = rest >= KEYS ? ~0ull : (1ull << rest) - 1;
    } else {
      // A mask's bytes are read for 32 tiles at a time: a wait for one of them is a wait for all transfers ahead of it.
      if (turn % 32 == 0)
        for (int i = 0; i < 32; ++i) {
          const uint64_t word = __ballot(t + i * GROUPS < t1 && key_counts(a, b, (t + i * GROUPS) * KEYS + lane % KEYS, n));
#pragma unroll
          for (int k = 0; k < KEYS / 32; ++k) words[k] = lane == i ? (unsigned)(word >> (32 * k)) : words[k];
        }
      valid = (unsigned)__builtin_amdgcn_readlane(words[0], turn % 32);
      valid |= KEYS == 64 ? (uint64_t)(unsigned)__builtin_amdgcn_readlane(words[KEYS / 32 - 1], turn % 32) << 32 : valid << 32;
    }
    T* vs = mine + (buffer * 2 + 1) * TILE;
    const unsigned ks_at = hide(mine_at + buffer * (4 * TILE) + rows_at), vs_at = hide(mine_at + (buffer * 4 + 2) * TILE + columns_at);
    // the tile after next overwrites the one before this: its readers are done, in this wave or (barrier) in all
    const int ahead = buffer == 0 ? STAGES - 1 : buffer - 1;
    if constexpr (FEW) {
      if (t + (STAGES - 1) * GROUPS < t1) {
        phase_wait();
        fetch(t + (STAGES - 1) * GROUPS, ahead);
        wave_arrived<Load::COUNT * (STAGES - 1)>();
      } else {
        wave_arrived<0>();
      }
    } else {
      if (t + (STAGES - 2) * GROUPS < t1) wait_vm_lds<Load::COUNT * (STAGES - 2)>();
      else wait_vm_lds<0>();
      block_barrier();
      if (t + (STAGES - 1) * GROUPS < t1) fetch(t + (STAGES - 1) * GROUPS, ahead);
    }
    buffer = buffer == STAGES - 1 ? 0 : buffer + 1;
    if (idle) continue;   // the barrier was all that was left to do
    if (valid != ~0ull) zero_rows<T, DP, KEYS>(vs, valid, lane);

    float16_t s[KEYS / 32];
    over_head<T, DP, KEYS / 32>(ks_at, 0, qf, s);
    if (valid != ~0ull) {
#pragma unroll
      for (int k = 0; k < KEYS / 32; ++k) {
        const uint32_t word = (uint32_t)(valid >> (32 * k)) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[k][i] = word >> product_row(i, 0) & 1 ? s[k][i] : -INFINITY;
      }
    }
    float top = largest(s);
    top = max_of_halves(top) * unit;
    if (__any(top > off + (8.0f + kLift<T>))) {   // also: the first keys of a row that count
      const float next = fmaxf(off, lowered<T>(top));
      const float fade = next == -INFINITY ? 1.0f : exp2_(off - next);
      off = next;
      far = __any(fabsf(off) > kFar);
      total *= fade;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[d][i] *= fade;
          if constexpr (FEW) second[d][i] *= fade;
        }
    }
    const float by = off == -INFINITY ? 0.0f : off;
    float times = unit;
    if (far) {
      round_scores(s, unit);
      times = 1.0f;
    }
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[k][i] = exp2_(s[k][i] * times - by);
        sum[i & 1] += s[k][i];
      }
    total += sum[0] + sum[1];
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const half8<T> p = round8<T>(s[k], 8 * c);
        half8<T> rest = {};
        if constexpr (FEW) {
          float16_t left;
#pragma unroll
          for (int i = 0; i < 8; ++i) left[i] = s[k][8 * c + i] - (float)p[i];
          rest = round8<T>(left, 0);
        }
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          const half8<T> v = columns_operand<T, DP>(vs_at, 32 * k + 16 * c, d);
          acc[d] = Half8<T>::mfma(v, p, acc[d]);
          if constexpr (FEW) second[d] = Half8<T>::mfma(v, rest, second[d]);
        }
      }
  }
  total = sum_of_halves(total);

  const int64_t heads_rows = (int64_t)a.batch * a.kv_heads * a.rows;
  if constexpr (!FEW) {
    const int64_t flat = (int64_t)bkv * a.rows + r;
    if (!row_here) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const float lse = total == 0.0f ? -INFINITY : (off + log2f(total)) * kLn2;
    if (h == 0) (a.splits > 1 ? a.part_lse[split * heads_rows + flat] : a.lse[flat]) = lse;
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
  } else {
    __syncthreads();
    float* all_found = (float*)lds;
    float* found = all_found + (group * ROWS + wave * 32 + col) * LD;
    if (h == 0) {
      row_max[group][wave * 32 + col] = off;
      row_total[group][wave * 32 + col] = total;
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float first = acc[d][4 * i4 + i];
          f[i] = fabsf(first) < INFINITY ? first + second[d][4 * i4 + i] : first;
        }
        __builtin_memcpy(found + d * 32 + 8 * i4 + 4 * h, f, 16);
      }
    __syncthreads();
    for (int e = threadIdx.x; e < ROWS * (DP / 4); e += THREADS) {
      const int j = e / (DP / 4), d = e % (DP / 4) * 4;
      const int64_t rj = (int64_t)row_tile * ROWS + j;
      if (rj >= a.rows) continue;
      float top = row_max[0][j], all = 0.0f, f[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 1; k < GROUPS; ++k) top = fmaxf(top, row_max[k][j]);
      const float by = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        const float w = exp2_(row_max[k][j] - by);
        all += w * row_total[k][j];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] += w * all_found[(k * ROWS + j) * LD + d + i];
      }
      const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] *= inv;
      const int64_t fj = (int64_t)bkv * a.rows + rj, sj = split * heads_rows + fj;
      if (d == 0) (a.splits > 1 ? a.part_lse[sj] : a.lse[fj]) = all == 0.0f ? -INFINITY : (top + log2f(all)) * kLn2;
      if (d >= a.head) continue;
      if (a.splits > 1) store_four(a.part + sj * a.head, d, a.head, f);
      else store_four((T*)a.out + dense_row_at(a, b, kv, rj), d, a.head, f);
    }
  }
}

// Many rows: 8 waves of 32 share tiles of 64 keys.  The two waves of a SIMD take turns: while one's products run (the weights of tile t
// times the values, then the scores of tile t + 1), the other works on its softmax, and a barrier ends every such half.  Left to
// themselves the waves of a block, which a barrier a tile keeps together anyway, all form products and then all exponentials:
// the matrix and the vector units of a SIMD, each busy half of the time, took one after the other.
//
//   half     0            1            2            3
//   waves 0-3  products 0   softmax 1    products 1   softmax 2   ...
//   waves 4-7               products 0   softmax 1    products 1  ...
//
// Pair p of tiles in LDS is (keys p + 1, values p): what products p read, in halves 2 p and 2 p + 1.  There are four of them; a wave asks for
// its share of pair p + 3 when it begins the softmax behind products p, with pair p - 1 out of use.
//
// 2 x 4096 x 4096, 32 heads of 128 (8 for keys): 508 us, 1080 TFLOP/s.  Bound by the power that the products may take: on zeros, where the card keeps its
// clock, 405 us.  (Waves that do not take turns: 520 us; blocks of four waves 606.)
template <typename T, int DP>
__global__ __launch_bounds__(512, 2) void attend16_wide_kernel(const AttendArgs a) {
  constexpr int KEYS = 64, TILE = KEYS * DP, WAVES = 8;
  typedef PairLoad<T, DP, KEYS, WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[8 * TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  const bool late = wave >= WAVES / 2;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int kv = (int)(at / a.row_tiles) / a.batch, b = (int)(at / a.row_tiles + kv) % a.batch, bkv = b * a.kv_heads + kv;
  const int n = keys_that_count(a, b);
  const int tiles = (n + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = (int64_t)row_tile * (32 * WAVES) + wave * 32 + col;
  const bool row_here = r < a.rows, idle = (int64_t)row_tile * (32 * WAVES) + wave * 32 >= a.rows;
  const unsigned lds_at = lds_addr_of(lds), rows_at = rows_place<T, DP>(lane), columns_at = columns_place<T, DP>(lane);
  if (DP != a.head) {   // the columns behind the head size, for good
    half8<T> zero = {};
    for (int e = threadIdx.x; e < 8 * KEYS * (DP / 8); e += 64 * WAVES) __builtin_memcpy(lds + e * 8, &zero, 16);
    __syncthreads();
  }
  // (as in attend16_kernel)
  const float unit = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
  half8<T> qf[DP / 16];
  {
    const T* q = (const T*)a.q.p + (row_here ? row_at(a.q, a, b, kv, r) : 0);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      qf[c] = half8<T>{};
      if (row_here && 16 * c + 8 * h < a.head) __builtin_memcpy(&qf[c], q + 16 * c + 8 * h, 16);
      if (a.scale < 0) qf[c] = -qf[c];
    }
  }
  float16_t acc[DP / 32], s[2];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  float off = -INFINITY, total = 0.0f;
  bool far = false;
  half8<T> p[4];
  uint64_t valid = 0;
  unsigned words[2];   // which keys of 32 tiles count, tile i in lane i

  const T* kp = (const T*)a.k.p + b * a.k.b + kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(wave, lane, a.head, a.k.t, a.v.t);
  const int64_t k_step = KEYS * a.k.t, v_step = KEYS * a.v.t;
  const T *k_next = kp + t0 * k_step, *v_next = vp + (t0 - 1) * v_step;   // of the pair that is asked for next
  auto fetch = [&](int pair) {   // what there is not of a pair is replaced by a tile that is not read
    const unsigned to = lds_at + ((pair - t0) & 3) * (4 * TILE);
    if (pair >= t0 && (pair + 2) * KEYS <= n) load.issue(k_next, v_next, to, wave);
    else load.issue_tiles(min(pair + 1, t1 - 1), max(pair, t0), n, kp, a.k.t, vp, a.v.t, to, wave, lane);
    k_next += k_step;
    v_next += v_step;
  };
  auto softmax = [&](int t) {
    if (a.mask == nullptr) {
      const int rest = n - t * KEYS;
      valid = rest >= KEYS ? ~0ull : (1ull << rest) - 1;
    } else {
      if ((t - t0) % 32 == 0)
        for (int i = 0; i < 32; ++i) {
          const uint64_t word = __ballot(t + i < t1 && key_counts(a, b, (t + i) * KEYS + lane, n));
          words[0] = lane == i ? (unsigned)word : words[0];
          words[1] = lane == i ? (unsigned)(word >> 32) : words[1];
        }
      valid = (uint64_t)(unsigned)__builtin_amdgcn_readlane(words[1], (t - t0) % 32) << 32 | (unsigned)__builtin_amdgcn_readlane(words[0], (t - t0) % 32);
    }
    if (valid != ~0ull) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t word = (uint32_t)(valid >> (32 * k)) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[k][i] = word >> product_row(i, 0) & 1 ? s[k][i] : -INFINITY;
      }
    }
    const float top = max_of_halves(largest(s)) * unit;
    if (__any(top > off + (8.0f + kLift<T>))) {   // also: the first keys of a row that count
      const float next = fmaxf(off, lowered<T>(top));
      const float fade = next == -INFINITY ? 1.0f : exp2_(off - next);
      off = next;
      far = __any(fabsf(off) > kFar);
      total *= fade;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
    }
    const float by = off == -INFINITY ? 0.0f : off;
    float times = unit;
    if (far) {
      round_scores(s, unit);
      times = 1.0f;
    }
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 8 * c; i < 8 * c + 8; ++i) {
          s[k][i] = exp2_(s[k][i] * times - by);
          sum[i & 1] += s[k][i];
        }
        p[2 * k + c] = round8<T>(s[k], 8 * c);
      }
    total += sum[0] + sum[1];
  };
  auto keys_at = [&](int t) { return hide(lds_at + ((t - t0 - 1) & 3) * (4 * TILE) + rows_at); };
  auto products = [&](int t) {
    __builtin_amdgcn_s_setprio(1);
    if (valid != ~0ull) zero_rows<T, DP, KEYS>(lds + (((t - t0) & 3) * 2 + 1) * TILE, valid, lane);
    const unsigned vs_at = hide(lds_at + (((t - t0) & 3) * 4 + 2) * TILE + columns_at), ks_at = keys_at(t + 1);
    OverHead<T, DP, 2> next;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) acc[d] = Half8<T>::mfma(columns_operand<T, DP>(vs_at, 16 * c, d), p[c], acc[d]);
      if (c == 2) next.begin(ks_at, 0);   // (behind the last tile: read, and not used)
    }
    next.finish(ks_at, 0, qf, s);
    __builtin_amdgcn_s_setprio(0);
  };

  if (t0 < t1) {
#pragma unroll
    for (int k = -1; k < 3; ++k)
      if (t0 + k < t1) fetch(t0 + k);
    // pair p has arrived when no more than the pairs behind it are on their way
    auto arrived = [&](int pair, int asked) {
      const int behind = min(asked, t1 - 1) - pair;
      if (behind >= 3) wait_vm<3 * Load::COUNT>();
      else if (behind == 2) wait_vm<2 * Load::COUNT>();
      else if (behind == 1) wait_vm<Load::COUNT>();
      else wait_vm<0>();
    };
    arrived(t0 - 1, t0 + 2);
    phase_barrier();
    if (!idle) {
      over_head<T, DP, 2>(keys_at(t0), 0, qf, s);
      softmax(t0);
    }
    arrived(t0, t0 + 2);
    if (late) phase_barrier();
    for (int t = t0; t < t1; ++t) {
      phase_barrier();
      if (!idle) products(t);
      if (late) arrived(t + 1, t + 2);
      if (!late || t + 1 < t1) phase_barrier();
      if (t + 3 < t1) fetch(t + 3);
      if (!idle && t + 1 < t1) softmax(t + 1);
      if (!late) arrived(t + 1, t + 3);
    }
  }
  if (!row_here) return;
  total = sum_of_halves(total);
  const int64_t heads_rows = (int64_t)a.batch * a.kv_heads * a.rows, flat = (int64_t)bkv * a.rows + r;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const float lse = total == 0.0f ? -INFINITY : (off + log2f(total)) * kLn2;
  if (h == 0) (a.splits > 1 ? a.part_lse[split * heads_rows + flat] : a.lse[flat]) = lse;
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

template <typename T, int DP>
void launch(const AttendArgs& a, bool few, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits));
  if (few) {
    hipLaunchKernelGGL((attend16_kernel<T, DP, true>), grid, dim3(64 * few_groups(DP)), 0, st, a);
  } else if constexpr (DP > 64) {
    hipLaunchKernelGGL((attend16_wide_kernel<T, DP>), grid, dim3(512), 0, st, a);
  } else {
    hipLaunchKernelGGL((attend16_kernel<T, DP, false>), grid, dim3(256), 0, st, a);
  }
}

}  // namespace

int attend16_tile(int64_t head) { return head > 64 ? 256 : 128; }
bool attend16_takes(const AttendArgs& a, int type) {
  return type != NNVHIP_TYPE_F32 && by_pieces(a.q, a.head) && by_pieces(a.k, a.head) && by_pieces(a.v, a.head);
}

void launch_attend16(const AttendArgs& a, int type, bool few, hipStream_t st) {
  if (type == NNVHIP_TYPE_BF16) ATTEND_BY_HEAD(launch, bf16_t, a, few, st);
  else ATTEND_BY_HEAD(launch, f16_t, a, few, st);
}

}  // namespace nnvhip
