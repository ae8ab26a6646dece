// Differential attention of points in 16 bits, forward, on v_mfma_f32_32x32x16_{bf16,f16}.  What is said of the softmax's weights, their lift
// in f16 and of scores that are far from zero in points_attend16.h holds here.
#include "points_differ16.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

// A tile's scores (of a lane's row, masked) to weights: raises the running maximum where it has grown by more than 2^8; returns what the sums so far are
// to be multiplied with (1 mostly).
template <typename T, int K>
__device__ __forceinline__ float to_weights(float16_t (&s)[K], float unit, float& off, float& total, bool& far) {
  float fade = 1.0f;
  const float top = max_of_halves(largest(s)) * unit;
  if (__any(top > off + (8.0f + kLift<T>))) {   // also: the first keys that a row sees
    const float next = fmaxf(off, lowered<T>(top));
    fade = next == -INFINITY ? 1.0f : exp2_(off - next);
    off = next;
    far = __any(fabsf(off) > kFar);
    total *= fade;
  }
  const float by = off == -INFINITY ? 0.0f : off;
  float times = unit;
  if (far) {
    round_scores(s, unit);
    times = 1.0f;
  }
  float sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[k][i] = exp2_(s[k][i] * times - by);
      sum[i & 1] += s[k][i];
    }
  total += sum[0] + sum[1];
  return fade;
}
// keys that do not take part: -inf.  word: of 32 keys, from this half's on
__device__ __forceinline__ void mask_scores(float16_t& s, uint32_t word) {
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = word >> product_row(i, 0) & 1 ? s[i] : -INFINITY;
}
// A negative scale is moved into q's sign; one of zero is taken as one that leaves every score next to zero.
__device__ __forceinline__ float unit_of(float scale) { return fmaxf(fabsf(scale) * kLog2e, 1e-30f); }
template <typename T, int CH>
__device__ __forceinline__ void query_operands(half8<T> (&f)[CH], const T* q, int h, int head, bool here, float scale) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    f[c] = half8<T>{};
    if (here && 16 * c + 8 * h < head) __builtin_memcpy(&f[c], q + 16 * c + 8 * h, 16);
    if (scale < 0) f[c] = -f[c];
  }
}

// Many rows: a wave takes 32 rows of one map, eight waves share tiles of 64 keys: four groups of rows, both maps, whose two waves are of one SIMD.  Tiles are
// on their way to LDS STAGES - 1 ahead; one barrier a tile.  (The two waves of a SIMD taking turns at products and softmax, as attend16_wide_kernel's
// do, with rounded weights: 4096 x 4096, heads of 128, 530 us instead of 471, 577 x 1000, heads of 40, 76 instead of 65: with values twice as wide the products take longer than the
// softmax beside them.)  At the end the second map's result meets the first one's in LDS, lane by lane.
// (Four stages where they fit and every wave has as many transfers; with rounded weights, 2 x 2048 x 2048, 16 heads of 64: 126 us, with two 136.  Else two: heads of 40 as above 64 us,
// with four 67, of 96 109 us, with three 112.)
// A map's weights go into the product with v in two pieces of 16 bits each (pieces8), all of them: the difference of the maps is smaller than either, so that
// rounded weights alone leave the result up to 1.6 times as far off as its own rounding (bf16: 0.0026 for 0.0017), and what is off must not go by where a key lies.
// (2 x 4096 x 4096, 16 heads of 128, causal: 567 us, 1210 TFLOP/s, matrix units busy 62 %, with rounded weights alone 450; 8 x 577 x 1000 by length, 12 heads of 40: 61 us, matrix units busy
// 34 %.)
template <int CH>
constexpr int differ_stages = CH == 2 || CH == 4 ? 4 : 2;
template <typename T, int CH>
__global__ __launch_bounds__(512, 2) void differ16_kernel(const DifferArgs a) {
  constexpr int KEYS = 64, STAGES = differ_stages<CH>, DP = Width16<CH>::DP, W = Width16<CH>::W;
  typedef TripleLoad<T, CH, KEYS, 8> Load;
  __shared__ __attribute__((aligned(1024))) T lds[STAGES * Load::VALUES];
  static_assert(STAGES >= 2 && STAGES * Load::VALUES * 2 >= 4 * 32 * W * 4, "the second map's result fits the tiles' place");
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int map = wave >> 2, part_of = wave & 3;
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)a.row_tiles * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = (uint32_t)at.x % (uint32_t)a.splits, row_tile = row_tile_of(a, (uint32_t)at.x / (uint32_t)a.splits);
  const int n = keys_that_count(a, b);
  const int64_t first = (int64_t)row_tile * kDiffer16Rows, last = min(first + kDiffer16Rows, a.rows) - 1;
  const int tiles = (most_seen(a, first, last, n) + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = first + part_of * 32 + col;
  const bool here = r < a.rows, idle = first + part_of * 32 >= a.rows;
  const int seen = here ? seen_by(a, r, n) : 0;
  // keys that all, and that any, of the wave's rows see
  const int seen_by_all = fewest_seen(a, min(first + part_of * 32, last), min(first + part_of * 32 + 31, last), n);
  const int seen_by_any = most_seen(a, min(first + part_of * 32, last), min(first + part_of * 32 + 31, last), n);
  const unsigned lds_at = lds_addr_of(lds), rows_at = rows_place<T, DP>(lane) + map * (2 * Load::MAP), columns_at = columns_place<T, W>(lane) + 4 * Load::MAP;
  if (DP != a.head || W != 2 * a.head) zero_lds<T, STAGES * Load::VALUES, 512>(lds);   // the columns behind the head size, for good

  const float unit = unit_of(a.scale);
  half8<T> qf[CH];
  query_operands<T, CH>(qf, (const T*)a.q.p + (here ? map_row_at(a.q, a, b, kv, r, map) : 0), h, a.head, here, a.scale);
  float16_t acc[CH];
#pragma unroll
  for (int d = 0; d < CH; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  float off = -INFINITY, total = 0.0f;   // off: of the exponents, in products times unit
  bool far = false;                      // a row's is beyond kFar

  const T* kp = (const T*)a.k.p + b * a.k.b + 2 * kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(wave, lane, a.head, a.k.t, a.v.t);
  auto fetch = [&](int t, int buffer) {
    load.issue_tile(t, n, kp, a.k.t, a.k.h, vp, a.v.t, lds_at + buffer * (2 * Load::VALUES), wave, lane);
  };
  KeyWords<KEYS> words;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (t0 + s < t1) fetch(t0 + s, s);
  int buffer = 0;
  for (int t = t0; t < t1; ++t) {
    const uint64_t valid = words(a, b, n, t, t1, t - t0, 1, lane);
    const unsigned stage = lds_at + buffer * (2 * Load::VALUES);
    const unsigned ks_at = hide(stage + rows_at), vs_at = hide(stage + columns_at);
    T* vs = lds + buffer * Load::VALUES + 2 * Load::MAP;
    const int ahead = buffer == 0 ? STAGES - 1 : buffer - 1;
    if (t + STAGES - 2 < t1) wait_vm_lds<Load::LEAST * (STAGES - 2)>();
    else wait_vm_lds<0>();
    block_barrier();
    if (t + STAGES - 1 < t1) fetch(t + STAGES - 1, ahead);
    buffer = buffer == STAGES - 1 ? 0 : buffer + 1;
    if (idle || t * KEYS >= seen_by_any) continue;   // the barrier was all that was left to do
    if (valid != ~0ull) zero_rows<T, W, KEYS>(vs, valid, lane);

    float16_t s[2];
    over_chunks<T, DP, CH, 2, CH == 8 ? 2 : 4>(ks_at, 0, [&](int c) { return qf[c]; }, s);
    if (valid != ~0ull || (t + 1) * KEYS > seen_by_all) {
#pragma unroll
      for (int k = 0; k < 2; ++k) mask_scores(s[k], ((uint32_t)(valid >> (32 * k)) & first_bits(seen - t * KEYS - 32 * k)) >> (4 * h));
    }
    const float fade = to_weights<T, 2>(s, unit, off, total, far);
    if (__any(fade != 1.0f))
#pragma unroll
      for (int d = 0; d < CH; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        half8<T> p, rest;
        pieces8<T>([&](int i) { return s[k][8 * c + i]; }, p, rest);
        constexpr int SOME = CH % 4 == 0 ? 4 : CH % 3 == 0 ? 3 : CH;
#pragma unroll
        for (int d0 = 0; d0 < CH; d0 += SOME) {
          half8<T> x[SOME];
#pragma unroll
          for (int d = 0; d < SOME; ++d) x[d] = columns_operand<T, W>(vs_at, 32 * k + 16 * c, d0 + d);
#pragma unroll
          for (int d = 0; d < SOME; ++d) acc[d0 + d] = Half8<T>::mfma(x[d], p, acc[d0 + d]);
#pragma unroll
          for (int d = 0; d < SOME; ++d) acc[d0 + d] = Half8<T>::mfma(x[d], rest, acc[d0 + d]);
        }
      }
  }
  total = sum_of_halves(total);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total, lse = total == 0.0f ? -INFINITY : (off + log2f(total)) * kLn2;
  const int size = 2 * a.head;
  if (a.splits > 1) {
    if (!here) return;
    const int64_t own = split * own_rows(a) + own_row(a, bkv, r, map);
    if (h == 0) a.part_lse[own] = lse;
#pragma unroll
    for (int d = 0; d < CH; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const float f[4] = {acc[d][4 * i4] * inv, acc[d][4 * i4 + 1] * inv, acc[d][4 * i4 + 2] * inv, acc[d][4 * i4 + 3] * inv};
        put_four(a.part + own * size, d * 32 + 8 * i4 + 4 * h, size, f);
      }
    return;
  }
  if (here && h == 0) a.lse[lse_at(a, b, kv, r, map)] = lse;
  wait_vm_lds<0>();
  __syncthreads();
  float* found = (float*)lds + part_of * 32 * W + 4 * lane;
  const int64_t dense = here ? wide_row_at(a, b, kv, r) : 0;
  if (map) {
#pragma unroll
    for (int d = 0; d < CH; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const float f[4] = {acc[d][4 * i4] * inv, acc[d][4 * i4 + 1] * inv, acc[d][4 * i4 + 2] * inv, acc[d][4 * i4 + 3] * inv};
        __builtin_memcpy(found + 256 * (4 * d + i4), f, 16);
        if (a.second && here) put_four((T*)a.second + dense, d * 32 + 8 * i4 + 4 * h, size, f);
      }
  }
  __syncthreads();
  if (map || !here) return;
  const float w = weight_of<T>(a, head_of_row(a, kv, r));
#pragma unroll
  for (int d = 0; d < CH; ++d)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      float f[4];
      __builtin_memcpy(f, found + 256 * (4 * d + i4), 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = rounded(acc[d][4 * i4 + i] * inv) - w * f[i];
      put_four((T*)a.out + dense, d * 32 + 8 * i4 + 4 * h, size, f);
    }
}

// Few rows (single tokens): 16 rows for the block, and a product's 32 columns are their first maps and their second ones, so that the values are multiplied with
// both at once.  (The scores of each map's keys are formed for all columns, of which half are taken.)  The block's waves take tiles of 32 keys in
// turn, each with LDS of its own, two stages; what they found is joined at the end.  Bound by memory, so that weights go in two pieces: what their rounding leaves is
// a second weight.
template <int CH>
constexpr int differ_groups() {
  constexpr int two_stages = 2 * 32 * (2 * Width16<CH>::DP + Width16<CH>::W) * 2;
  return 147456 / two_stages >= 8 ? 8 : 147456 / two_stages >= 4 ? 4 : 2;
}
template <typename T, int CH>
__global__ __launch_bounds__(64 * differ_groups<CH>(), 1) void differ16_few_kernel(const DifferArgs a) {
  constexpr int KEYS = 32, STAGES = 2, GROUPS = differ_groups<CH>(), DP = Width16<CH>::DP, W = Width16<CH>::W, LD = W + 4;
  typedef TripleLoad<T, CH, KEYS, 1> Load;
  constexpr int TILES = GROUPS * STAGES * Load::VALUES, FOUND = GROUPS * 32 * LD * 2;   // at the end: [group][column][LD floats]
  __shared__ __attribute__((aligned(1024))) T lds[TILES > FOUND ? TILES : FOUND];
  __shared__ float col_max[GROUPS][32], col_total[GROUPS][32];
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5, group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)a.row_tiles * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = at.x % a.splits, row_tile = at.x / a.splits;
  const int n = keys_that_count(a, b);
  const int64_t first = (int64_t)row_tile * kDifferFewRows, last = min(first + kDifferFewRows, a.rows) - 1;
  const int tiles = (most_seen(a, first, last, n) + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per + group, t1 = min(tiles, split * per + per);
  const int map = col >> 4;
  const int64_t r = first + (col & 15);
  const bool here = r < a.rows;
  const int seen = here ? seen_by(a, r, n) : 0, seen_by_all = fewest_seen(a, first, last, n);
  T* mine = lds + group * STAGES * Load::VALUES;
  const unsigned mine_at = lds_addr_of(mine), rows_at = rows_place<T, DP>(lane), columns_at = columns_place<T, W>(lane) + 4 * Load::MAP;
  if (DP != a.head || W != 2 * a.head) zero_lds<T, TILES, 64 * GROUPS>(lds);

  const float unit = unit_of(a.scale);
  half8<T> qf[CH];
  query_operands<T, CH>(qf, (const T*)a.q.p + (here ? map_row_at(a.q, a, b, kv, r, map) : 0), h, a.head, here, a.scale);
  float16_t acc[CH];
#pragma unroll
  for (int d = 0; d < CH; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  float off = -INFINITY, total = 0.0f;
  bool far = false;
  const T* kp = (const T*)a.k.p + b * a.k.b + 2 * kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(0, lane, a.head, a.k.t, a.v.t);
  auto fetch = [&](int t, int buffer) {
    load.issue_tile(t, n, kp, a.k.t, a.k.h, vp, a.v.t, mine_at + buffer * (2 * Load::VALUES), 0, lane);
  };
  KeyWords<KEYS> words;
  if (t0 < t1) fetch(t0, 0);
  int buffer = 0;
  for (int t = t0, turn = 0; t < t1; t += GROUPS, ++turn) {
    const uint32_t valid = (uint32_t)words(a, b, n, t, t1, turn, GROUPS, lane);
    const unsigned stage = mine_at + buffer * (2 * Load::VALUES);
    const unsigned ks_at = hide(stage + rows_at), vs_at = hide(stage + columns_at);
    if (t + GROUPS < t1) {
      phase_wait();
      fetch(t + GROUPS, buffer ^ 1);
      wave_arrived<Load::TOTAL>();
    } else {
      wave_arrived<0>();
    }
    if (valid != ~0u) zero_rows<T, W, KEYS>(mine + buffer * Load::VALUES + 2 * Load::MAP, (uint64_t)valid, lane);
    buffer ^= 1;
    float16_t s[1], other[1];
    over_chunks<T, DP, CH, 1, 2>(ks_at, 0, [&](int c) { return qf[c]; }, s);
    over_chunks<T, DP, CH, 1, 2>(ks_at + 2 * Load::MAP, 0, [&](int c) { return qf[c]; }, other);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = map ? other[0][i] : s[0][i];
    if (valid != ~0u || (t + 1) * KEYS > seen_by_all) mask_scores(s[0], (valid & first_bits(seen - t * KEYS)) >> (4 * h));
    const float fade = to_weights<T, 1>(s, unit, off, total, far);
    if (__any(fade != 1.0f))
#pragma unroll
      for (int d = 0; d < CH; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
    half8<T> p[2], rest[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) pieces8<T>([&](int i) { return s[0][8 * c + i]; }, p[c], rest[c]);
    over_columns<T, W, 2>(vs_at, 0, [&](int c, int d, const half8<T>& v) {
      acc[d] = Half8<T>::mfma(v, p[c], acc[d]);
      acc[d] = Half8<T>::mfma(v, rest[c], acc[d]);
    });
  }
  total = sum_of_halves(total);
  __syncthreads();
  float* all_found = (float*)lds;
  float* found = all_found + (group * 32 + col) * LD;
  if (h == 0) {
    col_max[group][col] = off;
    col_total[group][col] = total;
  }
#pragma unroll
  for (int d = 0; d < CH; ++d)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const float f[4] = {acc[d][4 * i4], acc[d][4 * i4 + 1], acc[d][4 * i4 + 2], acc[d][4 * i4 + 3]};
      __builtin_memcpy(found + d * 32 + 8 * i4 + 4 * h, f, 16);
    }
  __syncthreads();
  const int size = 2 * a.head;
  for (int e = threadIdx.x; e < kDifferFewRows * (W / 4); e += 64 * GROUPS) {
    const int j = e / (W / 4), d = e % (W / 4) * 4;
    const int64_t rj = first + j;
    if (rj >= a.rows) continue;
    float f[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int cj = 16 * m + j;
      float top = col_max[0][cj], all = 0.0f;
#pragma unroll
      for (int k = 1; k < GROUPS; ++k) top = fmaxf(top, col_max[k][cj]);
      const float by = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[m][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        const float w = exp2_(col_max[k][cj] - by);
        all += w * col_total[k][cj];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[m][i] += w * all_found[(k * 32 + cj) * LD + d + i];
      }
      const float inv = all == 0.0f ? 0.0f : 1.0f / all, lse = all == 0.0f ? -INFINITY : (top + log2f(all)) * kLn2;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[m][i] = rounded(f[m][i] * inv);
      const int64_t own = split * own_rows(a) + own_row(a, bkv, rj, m);
      if (d == 0) (a.splits > 1 ? a.part_lse[own] : a.lse[lse_at(a, b, kv, rj, m)]) = lse;
      if (a.splits > 1 && d < size) put_four(a.part + own * size, d, size, f[m]);
    }
    if (a.splits > 1 || d >= size) continue;
    const int64_t dense = wide_row_at(a, b, kv, rj);
    if (a.second) put_four((T*)a.second + dense, d, size, f[1]);
    const float w = weight_of<T>(a, head_of_row(a, kv, rj));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[0][i] -= w * f[1][i];
    put_four((T*)a.out + dense, d, size, f[0]);
  }
}

template <typename T, int CH>
void launch(const DifferArgs& a, bool few, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits));
  if (few) hipLaunchKernelGGL((differ16_few_kernel<T, CH>), grid, dim3(64 * differ_groups<CH>()), 0, st, a);
  else hipLaunchKernelGGL((differ16_kernel<T, CH>), grid, dim3(512), 0, st, a);
}

}  // namespace

bool differ16_takes(const DifferArgs& a, int type) {
  return type != NNVHIP_TYPE_F32 && by_pieces(a.q, a.head) && by_pieces(a.k, a.head) && by_pieces(a.v, a.head);
}
void launch_differ16(const DifferArgs& a, int type, bool few, hipStream_t st) {
  if (type == NNVHIP_TYPE_BF16) DIFFER_BY_HEAD(launch, bf16_t, a, few, st);
  else DIFFER_BY_HEAD(launch, f16_t, a, few, st);
}

}  // namespace nnvhip
