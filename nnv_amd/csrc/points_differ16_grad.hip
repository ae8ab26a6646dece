// Differential attention of points in 16 bits, backward, on v_mfma_f32_32x32x16_{bf16,f16}: the 16-bit forms of differ_query_grad_kernel and
// differ_key_grad_kernel.  The weights' difference and the scores' gradients go into their products in two pieces of 16 bits each.  dq takes D from
// the rounded o and second, but where keys are few (kTwice); on the way it finds D again as the sum of weights times dP, in f32, which the gradients of weights and keys take:
// a row that sees one key has a scores' gradient of zero, and what rounding makes of it would reach dk.
//
// f16 does not hold the scores' gradients as they are: weights far below one times differences of any size.  What a lane rounds is all of one column of the
// product that takes it, and so of one row of the result; a power of two that brings the column's largest value so far to 2^14 (Lift) is taken out of the
// result at the end, and when a larger value comes the sums so far are scaled, as a softmax's are: what is below 2^-38 of the largest is lost, what is above 2^-28
// keeps all bits.
//
// 2 x 4096 x 4096, 16 heads of 64, 4 for keys, causal, in bf16: dq 346 to 373 us, dk and dv 461 to 501.  Matrix units are busy 38 and 44 % of it, LDS 14 and 30: two waves a
// SIMD, whose exponentials, roundings and reads from LDS follow one another between the products.  More waves would not have the registers.  (Those of the keys' kernel that
// do not fit, in scratch: 5 for heads of 49 to 64, 10 above 96; in f16 8, 6 for heads of 65 to 80, 86 to 96, 165 above.)
#include "points_differ16.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

// max(x, |a|, |b|)
__device__ __forceinline__ float max3_of_sizes(float x, float a, float b) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(x), "v"(a), "v"(b));
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void load_operands(half8<T> (&f)[N], const T* row, int h, int size, bool there) {
#pragma unroll
  for (int c = 0; c < N; ++c) {
    f[c] = half8<T>{};
    if (there && 16 * c + 8 * h < size) __builtin_memcpy(&f[c], row + 16 * c + 8 * h, 16);
  }
}
template <int N>
__device__ __forceinline__ void zero(float16_t (&acc)[N]) {
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
}
// The power of two by which a column's values are rounded in f16 (bf16: none).
template <typename T>
struct Lift {
  static constexpr bool USED = std::is_same_v<T, f16_t>;
  float up = USED ? 0x1p40f : 1.0f;
  // values of a column, in this lane and l ^ 32: what has been added up of them so far is scaled where a value is larger than any before
  template <int N>
  __device__ __forceinline__ void raise(float16_t& s, float16_t (&acc)[N]) {
    if constexpr (USED) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) top = max3_of_sizes(top, s[i], s[i + 1]);
      top = max_of_halves(top);
      if (__any(top * up > 32768.0f)) {
        // (an infinite or missing value is not lifted, and does what it would)
        const float next = top * up > 32768.0f && top < INFINITY ? __builtin_amdgcn_ldexpf(1.0f, 14 - __builtin_amdgcn_frexp_expf(top)) : up, fade = next / up;
        up = next;
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] *= up;
    }
  }
  __device__ __forceinline__ float down() const { return USED ? 1.0f / up : 1.0f; }
};

// acc[d] += the product over 32 rows, from `first` on, of a tile of rows of DP values with p in two pieces.  (The scores' gradients
// cancel: of rounded ones alone dq and dk are up to 1.6 times as far off as their own rounding, 0.0026 for 0.0017 in bf16.  The gradients of 2 x 4096 x 4096, 16 / 4 heads of 64,
// causal, take 865 us, with rounded ones alone 710.)
template <typename T, int DP>
__device__ __forceinline__ void over_rows(unsigned tile, int first, const float16_t& p, float16_t (&acc)[DP / 32]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    half8<T> f, left;
    pieces8<T>([&](int i) { return p[8 * c + i]; }, f, left);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      const half8<T> x = columns_operand<T, DP>(tile, first + 16 * c, d);
      acc[d] = Half8<T>::mfma(x, f, acc[d]);
      acc[d] = Half8<T>::mfma(x, left, acc[d]);
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_result(T* row, const float16_t (&acc)[N], float by, int h, int size) {
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const float f[4] = {acc[d][4 * i4] * by, acc[d][4 * i4 + 1] * by, acc[d][4 * i4 + 2] * by, acc[d][4 * i4 + 3] * by};
      put_four(row, d * 32 + 8 * i4 + 4 * h, size, f);
    }
}

// Heads of up to 64: eight waves, two a SIMD; above, four with all of a SIMD's registers.
template <int CH>
constexpr int kWaves = CH <= 4 ? 8 : 4;
template <int CH>
constexpr int kKeyWaves = CH <= 4 ? 8 : 4;

// dq of 32 rows a wave, both maps: do v^T is formed once.
template <typename T, int CH>
__global__ __launch_bounds__(64 * kWaves<CH>, kWaves<CH> / 4) void differ_query_grad16_kernel(const DifferArgs a) {
  constexpr int KEYS = 64, WAVES = kWaves<CH>, ROWS = 32 * WAVES, DP = Width16<CH>::DP, W = Width16<CH>::W;
  typedef TripleLoad<T, CH, KEYS, WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[2 * Load::VALUES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)a.row_tiles * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = (uint32_t)at.x % (uint32_t)a.splits, row_tile = row_tile_of(a, (uint32_t)at.x / (uint32_t)a.splits);
  const int n = keys_that_count(a, b);
  const int64_t first = (int64_t)row_tile * ROWS, last = min(first + ROWS, a.rows) - 1;
  const int tiles = (most_seen(a, first, last, n) + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = first + wave * 32 + col;
  const bool here = r < a.rows, idle = first + wave * 32 >= a.rows;
  const int seen_by_all = fewest_seen(a, min(first + wave * 32, last), min(first + wave * 32 + 31, last), n);
  const int seen_by_any = most_seen(a, min(first + wave * 32, last), min(first + wave * 32 + 31, last), n);
  const unsigned lds_at = lds_addr_of(lds), rows_at = rows_place<T, DP>(lane), wide_at = rows_place<T, W>(lane) + 4 * Load::MAP,
                 columns_at = columns_place<T, DP>(lane);
  if (DP != a.head || W != 2 * a.head) zero_lds<T, 2 * Load::VALUES, 64 * WAVES>(lds);

  float offset[2], delta[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) offset[m] = offset_of(here ? a.lse[lse_at(a, b, kv, r, m)] : -INFINITY);
  const bool takes_part = offset[0] != INFINITY;
#pragma unroll
  for (int m = 0; m < 2; ++m) delta[m] = takes_part ? a.delta[own_row(a, bkv, r, m)] : 0.0f;
  const int seen = takes_part ? seen_by(a, r, n) : 0;
  const float w = here ? weight_of<T>(a, head_of_row(a, kv, r)) : 0.0f, unit = a.scale * kLog2e;
  half8<T> qf[2][CH], gf[2 * CH];
#pragma unroll
  for (int m = 0; m < 2; ++m) load_operands<T, CH>(qf[m], (const T*)a.q.p + (here ? map_row_at(a.q, a, b, kv, r, m) : 0), h, a.head, takes_part);
  load_operands<T, 2 * CH>(gf, (const T*)a.go.p + (here ? row_at(a.go, a, b, kv, r) : 0), h, 2 * a.head, takes_part);
  float16_t dq[2][DP / 32];
  Lift<T> lift[2];
  float dot[2] = {0.0f, 0.0f};   // D again, of the weights and dP, for the weights' and the keys' gradients (o and second are rounded)
#pragma unroll
  for (int m = 0; m < 2; ++m) zero(dq[m]);
  const T* kp = (const T*)a.k.p + b * a.k.b + 2 * kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(wave, lane, a.head, a.k.t, a.v.t);
  int counts = 0;
  auto fetch = [&](int t, int buffer) {
    load.issue_tile(t, n, kp, a.k.t, a.k.h, vp, a.v.t, lds_at + buffer * (2 * Load::VALUES), wave, lane);
    counts = key_word(a, b, t * KEYS + lane, n);
  };
  int buffer = 0;
#pragma unroll 1
  for (int sweep = tiles * KEYS <= kTwice ? 0 : 1; sweep < 2; ++sweep) {   // the first one, if any, for D alone, of all splits' keys
    const int first_tile = sweep ? t0 : 0, end = sweep ? t1 : tiles;
    if (first_tile < end) fetch(first_tile, buffer);   // (where the tile before the last one was)
    for (int t = first_tile; t < end; ++t, buffer ^= 1) {
      const uint64_t valid = __ballot(counts != 0);
      const unsigned stage = lds_at + buffer * (2 * Load::VALUES);
      wait_vm_lds<0>();
      block_barrier();
      if (t + 1 < end) fetch(t + 1, buffer ^ 1);
      if (idle || t * KEYS >= seen_by_any) continue;
      if (valid != ~0ull) {   // the maps' keys, which a gradient of zero meets
        zero_rows<T, DP, KEYS>(lds + buffer * Load::VALUES, valid, lane);
        zero_rows<T, DP, KEYS>(lds + buffer * Load::VALUES + Load::MAP, valid, lane);
      }
      const bool masked = valid != ~0ull || (t + 1) * KEYS > seen_by_all;
#pragma unroll 1
      for (int k = 0; k < KEYS / 32; ++k) {
        const unsigned map_k = stage + k * (64 * DP), ks_at = hide(map_k + rows_at), vs_at = hide(stage + k * (64 * W) + wide_at), kc_at = hide(map_k + columns_at);
        float16_t dp[1], s[2][1];
        over_chunks<T, W, 2 * CH, 1, 4>(vs_at, 0, [&](int c) { return gf[c]; }, dp);
        const uint32_t word = ((uint32_t)(valid >> (32 * k)) & first_bits(seen - t * KEYS - 32 * k)) >> (4 * h);
        if (masked)
#pragma unroll
          for (int i = 0; i < 16; ++i) dp[0][i] = word >> product_row(i, 0) & 1 ? dp[0][i] : 0.0f;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          over_chunks<T, DP, CH, 1, 4>(ks_at + m * (2 * Load::MAP), 0, [&](int c) { return qf[m][c]; }, s[m]);
          const float by = m ? -w : 1.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[m][0][i] = exp2_(s[m][0][i] * unit - offset[m]);
          if (masked)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[m][0][i] = word >> product_row(i, 0) & 1 ? s[m][0][i] : 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            dot[m] += s[m][0][i] * dp[0][i];
            s[m][0][i] *= by * (dp[0][i] - delta[m]);
          }
          if (sweep == 0) continue;
          lift[m].raise(s[m][0], dq[m]);
          over_rows<T, DP>(kc_at + m * (2 * Load::MAP), 0, s[m][0], dq[m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) dot[m] = sum_of_halves(dot[m]);
    if (sweep) break;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      delta[m] = dot[m];
      dot[m] = 0.0f;
    }
  }
  if (!here) return;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (h == 0) {
      a.dots[split * own_rows(a) + own_row(a, bkv, r, m)] = dot[m];
      if (a.splits == 1) *info_at(a, bkv, r, kDelta0 + m) = dot[m];   // else differ_sum_rows_kernel does
    }
    if (a.splits > 1) store_result(a.part + (split * own_rows(a) + own_row(a, bkv, r, m)) * a.head, dq[m], a.scale * lift[m].down(), h, a.head);
    else store_result((T*)a.dq + dense_map_row_at(a, b, kv, r, m), dq[m], a.scale * lift[m].down(), h, a.head);
  }
}

// dk of both maps, and dv, of 32 keys a wave.  Two waves a SIMD have no room for the values' operands beside the gradients: they lie in LDS.
template <typename T, int CH>
__global__ __launch_bounds__(64 * kKeyWaves<CH>, kKeyWaves<CH> / 4) void differ_key_grad16_kernel(const DifferArgs a) {
  constexpr int PARKED = CH == 3 || CH == 4 ? 3 * CH : CH == 8 ? 2 * CH : 0;   // operands in LDS: the values', and the second map's keys'
  constexpr int ROWS = PARKED ? 32 : 64, WAVES = kKeyWaves<CH>, KEYS = 32 * WAVES, DP = Width16<CH>::DP, W = Width16<CH>::W;
  typedef TripleLoad<T, CH, ROWS, WAVES, false> Load;
  __shared__ __attribute__((aligned(1024))) T lds[2 * Load::VALUES + WAVES * 512 * PARKED];
  __shared__ __attribute__((aligned(1024))) float info[2][kInfos * ROWS < 256 ? 256 : 512];   // [buffer][RowInfo * ROWS + row]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  const int blocks = key_blocks_of(a);
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)blocks * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = (uint32_t)at.x % (uint32_t)a.splits, block = (uint32_t)at.x / (uint32_t)a.splits;
  const int n = keys_that_count(a, b);
  const unsigned lds_at = lds_addr_of(lds), rows_at = rows_place<T, DP>(lane), wide_at = rows_place<T, W>(lane) + 4 * Load::MAP;
  const unsigned columns_at = columns_place<T, DP>(lane), wide_columns_at = columns_place<T, W>(lane) + 4 * Load::MAP;
  if (DP != a.head || W != 2 * a.head) zero_lds<T, 2 * Load::VALUES, 64 * WAVES>(lds);
  const float unit = a.scale * kLog2e;
  Load load;
  load.init(wave, lane, a.head, a.q.t, a.go.t);
  const T* qp = (const T*)a.q.p + b * a.q.b + 2 * (kv * (int64_t)a.group) * a.q.h;
  const T* gp = (const T*)a.go.p + b * a.go.b + kv * (int64_t)a.group * a.go.h;
  // the weights' difference is at most 1 + |w|: in f16 of 2^14 (the largest, all bits down to 2^-28).  (Without rows there may be no weights, and there is nothing to lift.)
  float wide_up = 1.0f;
  if constexpr (Lift<T>::USED) {
    float most = 0.0f;
    for (int g = 0; g < a.group && a.rows > 0; ++g) most = fmaxf(most, fabsf(weight_of<T>(a, kv * a.group + g)));
    if (most < INFINITY) wide_up = __builtin_amdgcn_ldexpf(1.0f, 14 - __builtin_amdgcn_frexp_expf(1.0f + most));
  }
#pragma unroll 1
  for (int key_tile = block;; key_tile = a.key_tiles - 1 - block) {
    const int first = key_tile * KEYS, key = first + wave * 32 + col;
    const bool here = key < a.keys, counts = key_counts(a, b, key, n);
    const int i_min = a.causal ? first - (n - a.queries) : 0;   // the first query that sees one of the block's keys
    // where no key of the block counts there is nothing to add up
    const bool any = __syncthreads_or(counts);
    const int t0 = first_row_tile(a, split, ROWS, i_min), t1 = any ? first_row_tile(a, split + 1, ROWS, i_min) : 0;

    half8<T> kf[2][CH], vf[2 * CH];
    T* parked = lds + 2 * Load::VALUES + wave * (512 * PARKED) + lane * 8;   // operand c at parked + 512 c; no other wave's
#pragma unroll
    for (int m = 0; m < 2; ++m)
      load_operands<T, CH>(kf[m], (const T*)a.k.p + (counts ? b * a.k.b + (2 * kv + m) * a.k.h + key * a.k.t : 0), h, a.head, counts);
    load_operands<T, 2 * CH>(vf, (const T*)a.v.p + (counts ? b * a.v.b + kv * a.v.h + key * a.v.t : 0), h, 2 * a.head, counts);
#pragma unroll
    for (int c = 0; c < PARKED; ++c) __builtin_memcpy(parked + 512 * c, c < 2 * CH ? &vf[c < 2 * CH ? c : 0] : &kf[1][c < 2 * CH ? 0 : c - 2 * CH], 16);
    auto operand = [&](int c) {
      half8<T> x;
      __builtin_memcpy(&x, parked + 512 * c, 16);
      return x;
    };
    float16_t dk[2][DP / 32], dv[CH];
    Lift<T> lift[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) zero(dk[m]);
    zero(dv);
    auto fetch = [&](int t, int buffer) {
      const int64_t r0 = (int64_t)t * ROWS;
      int g = (int)((uint32_t)r0 / (uint32_t)a.queries), i = (int)(r0 - (int64_t)g * a.queries);
      const unsigned stage = lds_at + buffer * (2 * Load::VALUES);
      const T *q = qp + (i * a.q.t + 2 * g * a.q.h), *go = gp + (i * a.go.t + g * a.go.h);
      if (i + ROWS <= a.queries) {
        load.issue(q, q + a.q.h, go, a.q.t, a.go.t, stage, wave);
      } else {   // head after head; rows past the last one stay what they are, and are made zeros below
        for (int j = 0; j < ROWS && g < a.group; ++g) {
          const int end = min(ROWS, j + a.queries - i);
          load.issue_rows(j, end, q, q + a.q.h, go, stage, wave, lane);
          // (the next head's row 0 is at row `end` of the tile)
          q = qp + (2 * (g + 1) * a.q.h - end * a.q.t);
          go = gp + ((g + 1) * a.go.h - end * a.go.t);
          j = end;
          i = 0;
        }
      }
      if (wave == 0) {   // kInfos * ROWS floats, four a lane and transfer
        const float* from = a.info + bkv * (int64_t)kInfos * a.info_rows + r0;
#pragma unroll
        for (int k = 0; k < kInfos * ROWS / 256 + (kInfos * ROWS % 256 != 0); ++k) {
          const int array = (k * 64 + lane) / (ROWS / 4);
          if (array < kInfos)
            lds_dma16((const double*)from, 4 * ((unsigned)array * a.info_rows + (k * 64 + lane) % (ROWS / 4) * 4),
                      __builtin_amdgcn_readfirstlane(lds_addr_of(info[buffer]) + k * 1024));
        }
      }
    };
    int buffer = 0, t = next_row_tile(a, t0, ROWS, i_min);
    if (t < t1) fetch(t, 0);
    for (; t < t1; buffer ^= 1) {
      const unsigned stage = lds_at + buffer * (2 * Load::VALUES);
      wait_vm_lds<0>();
      block_barrier();
      const int64_t r0 = (int64_t)t * ROWS;
      t = next_row_tile(a, t + 1, ROWS, i_min);
      if (t < t1) fetch(t, buffer ^ 1);
      // rows past the last one, and those that see no key: nothing of them may reach a sum
      const uint64_t valid = __ballot(info[buffer][kOffset0 * ROWS + lane % ROWS] != INFINITY);
      if (valid != ~0ull) {
        T* tile = lds + buffer * Load::VALUES;
        zero_rows<T, DP, ROWS>(tile, valid, lane);
        zero_rows<T, DP, ROWS>(tile + Load::MAP, valid, lane);
        zero_rows<T, W, ROWS>(tile + 2 * Load::MAP, valid, lane);
      }
      const bool masked = a.causal && fewest_seen(a, r0, min(r0 + ROWS, a.rows) - 1, n) < first + wave * 32 + 32;
#pragma unroll 1
      for (int k = 0; k < ROWS / 32; ++k) {
        const unsigned map_k = stage + k * (64 * DP), wide_k = stage + k * (64 * W);
        const unsigned qs_at = hide(map_k + rows_at), gs_at = hide(wide_k + wide_at), qc_at = hide(map_k + columns_at), gc_at = hide(wide_k + wide_columns_at);
        float16_t s[2][1], dp[1];   // (do v^T first: its operands' registers are then free)
        over_chunks<T, W, 2 * CH, 1, 2>(gs_at, 0, [&](int c) {
          if constexpr (PARKED > 0) return operand(c);
          else return vf[c];
        }, dp);
#pragma unroll
        for (int m = 1; m >= 0; --m) {   // (the one whose keys are read from LDS first)
          over_chunks<T, DP, CH, 1, 2>(qs_at + m * (2 * Load::MAP), 0, [&](int c) {
            if (PARKED > 2 * CH && m) return operand(2 * CH + c);
            else return kf[m][c];
          }, s[m]);
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            float f[4];
            __builtin_memcpy(f, &info[buffer][(kOffset0 + m) * ROWS + 32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][0][4 * i4 + i] = exp2_(s[m][0][4 * i4 + i] * unit - f[i]);
          }
        }
        if (masked)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool is = key < __builtin_bit_cast(int, info[buffer][kSees * ROWS + 32 * k + product_row(i, h)]);
#pragma unroll
            for (int m = 0; m < 2; ++m) s[m][0][i] = is ? s[m][0][i] : 0.0f;
          }
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          float f[4];
          __builtin_memcpy(f, &info[buffer][kWeight * ROWS + 32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[1][0][4 * i4 + i] *= f[i];
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          half8<T> both, left;   // in two pieces, as the scores' gradients
          pieces8<T>([&](int i) { return (s[0][0][8 * c + i] + s[1][0][8 * c + i]) * wide_up; }, both, left);
#pragma unroll
          for (int d = 0; d < CH; ++d) {
            const half8<T> x = columns_operand<T, W>(gc_at, 16 * c, d);
            dv[d] = Half8<T>::mfma(x, both, dv[d]);
            dv[d] = Half8<T>::mfma(x, left, dv[d]);
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            float f[4];
            __builtin_memcpy(f, &info[buffer][(kDelta0 + m) * ROWS + 32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][0][4 * i4 + i] *= dp[0][4 * i4 + i] - f[i];
          }
          lift[m].raise(s[m][0], dk[m]);
          over_rows<T, DP>(qc_at + m * (2 * Load::MAP), 0, s[m][0], dk[m]);
        }
      }
    }
    if (here) {
      if (!counts) {   // what the loop made of a column that does not count reached no other one
#pragma unroll
        for (int m = 0; m < 2; ++m) zero(dk[m]);
        zero(dv);
      }
      const int64_t dense = ((b * (int64_t)a.keys + key) * a.kv_heads + kv) * 2 * a.head;
      if (a.splits > 1) {
        const int64_t all = (int64_t)a.batch * a.keys * a.kv_heads * 2 * a.head;
#pragma unroll
        for (int m = 0; m < 2; ++m) store_result(a.part + split * all + dense + m * a.head, dk[m], a.scale * lift[m].down(), h, a.head);
        store_result(a.part + (a.splits + split) * all + dense, dv, 1.0f / wide_up, h, 2 * a.head);
      } else {
#pragma unroll
        for (int m = 0; m < 2; ++m) store_result((T*)a.dk + dense + m * a.head, dk[m], a.scale * lift[m].down(), h, a.head);
        store_result((T*)a.dv + dense, dv, 1.0f / wide_up, h, 2 * a.head);
      }
    }
    if (key_tile != block || blocks == a.key_tiles || a.key_tiles - 1 - block == block) break;
  }
}

template <typename T, int CH>
void launch_query(const DifferArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((differ_query_grad16_kernel<T, CH>), dim3((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits)), dim3(64 * kWaves<CH>), 0,
                     st, a);
}
template <typename T, int CH>
void launch_key(const DifferArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((differ_key_grad16_kernel<T, CH>), dim3((unsigned)((int64_t)a.batch * a.kv_heads * key_blocks_of(a.key_tiles, a.queries, a.keys, a.causal) * a.splits)), dim3(64 * kKeyWaves<CH>), 0,
                     st, a);
}

}  // namespace

int differ_grad16_tile(int64_t head) { return head <= 64 ? 256 : 128; }
int differ_key_grad16_tile(int64_t head) { return head <= 64 ? 256 : 128; }
bool differ_grad16_takes(const DifferArgs& a, int type) {
  return type != NNVHIP_TYPE_F32 && by_pieces(a.q, a.head) && by_pieces(a.k, a.head) && by_pieces(a.v, a.head) && by_pieces(a.go, a.head) && a.rows < (1 << 27);   // (kInfos * rows floats within 32 bits)
}
void launch_differ_query_grad16(const DifferArgs& a, int type, hipStream_t st) {
  if (type == NNVHIP_TYPE_BF16) DIFFER_BY_HEAD(launch_query, bf16_t, a, st);
  else DIFFER_BY_HEAD(launch_query, f16_t, a, st);
}
void launch_differ_key_grad16(const DifferArgs& a, int type, hipStream_t st) {
  if (type == NNVHIP_TYPE_BF16) DIFFER_BY_HEAD(launch_key, bf16_t, a, st);
  else DIFFER_BY_HEAD(launch_key, f16_t, a, st);
}

}  // namespace nnvhip
