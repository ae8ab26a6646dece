// Differential attention of points, backward: the kernels for every type, head size and alignment, with f32 products.
//
// As in points_attend_grad.hip two kernels form dq (a wave per 16 queries, both maps) and dk, dv (a wave per 16 keys), each sum in the registers of
// one wave, in a fixed order, with no atomics.  do v^T, half of what the scores' gradients take, is one product for both maps.  D of both maps and
// the weights' gradients come first.  Of 16-bit tensors, whose o and second are rounded, the kernel of dq finds D again on its way, as the sum of weights times dP in f32, which the gradients
// of weights and keys take: a row that sees one key has a scores' gradient of zero, and what rounding makes of it would reach dk.
//
// Bound by the f32 matrix instructions (4 x 1024 x 1024, 16 heads of 64: dq 475 us, dk and dv 740; 4 x 333 x 577, 6 heads of 40: 49 and 68, matrix units busy 48
// and 44 %: blocks of six or seven tiles, in whose beginning and end nothing is multiplied).  Two buffers in LDS, and so one barrier a tile instead of two, measured the same.  Heads of 65 to 96,
// and those that are no multiple of 4, have some registers in scratch (dq of heads of 92 in f32 125, of 90 208; dk and dv of 92 50, of 126 189): 4 x 333 x 577, 6 heads of 92 take 352 us, of 90 594.
#include "points_differ16.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

constexpr int kBlockRows = 64;   // rows, or keys, of a block
template <typename T>
constexpr bool kHalves = sizeof(T) == 2;

// D_1 = rowsum(do second), D_0 = rowsum(do o) + w D_1: 16 lanes a row.
template <typename T, int>
__global__ __launch_bounds__(256) void differ_delta_kernel(const DifferArgs a) {
  const uint32_t flat = blockIdx.x * 16 + threadIdx.x / 16, per = a.info ? a.info_rows : (uint32_t)a.rows;   // (fewer than 2^28)
  if (flat >= (int64_t)a.batch * a.kv_heads * per) return;   // (the lanes of a row go together)
  const uint32_t own = flat / per;
  const int64_t bkv = own, r = flat - own * per;
  const int b = own / (uint32_t)a.kv_heads, kv = own - b * a.kv_heads, size = 2 * a.head;
  float* info = a.info ? a.info + bkv * kInfos * per + r : nullptr;
  if (r >= a.rows) {
    if (threadIdx.x % 16 < kInfos) info[threadIdx.x % 16 * per] = threadIdx.x % 16 <= kOffset1 ? INFINITY : 0.0f;
    return;
  }
  const T* o = (const T*)a.out + wide_row_at(a, b, kv, r);
  const T* second = (const T*)a.second + wide_row_at(a, b, kv, r);
  const T* g = (const T*)a.go.p + row_at(a.go, a, b, kv, r);
  float s[2] = {0, 0};
  for (int d = threadIdx.x % 16 * 4; d < size; d += 64) {
    const Four x = load_four(o, d, size, true), z = load_four(second, d, size, true), y = load_four(g, d, size, true);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[0] += x.v[i] * y.v[i];
      s[1] += z.v[i] * y.v[i];
    }
  }
#pragma unroll
  for (int k = 8; k > 0; k >>= 1)
#pragma unroll
    for (int m = 0; m < 2; ++m) s[m] += __shfl_xor(s[m], k, 64);
  if (threadIdx.x % 16) return;
  const float lse[2] = {a.lse[lse_at(a, b, kv, r, 0)], a.lse[lse_at(a, b, kv, r, 1)]};
  const bool takes_part = lse[0] != -INFINITY;   // (both maps see the same keys)
  const float w = weight_of<T>(a, head_of_row(a, kv, r)), d0 = takes_part ? s[0] + w * s[1] : 0.0f, d1 = takes_part ? s[1] : 0.0f;
  a.delta[own_row(a, bkv, r, 0)] = d0;
  a.delta[own_row(a, bkv, r, 1)] = d1;
  if (!info) return;
  const float values[kInfos] = {offset_of(lse[0]), offset_of(lse[1]), d0, d1, -w, __builtin_bit_cast(float, seen_by(a, r, keys_that_count(a, b)))};
#pragma unroll
  for (int k = 0; k < kInfos; ++k) info[k * per] = values[k];
}

// dw of a head: a block adds its rows' D_1 (of all splits, where the kernel of dq found it), in f64.  splits: of that kernel.
constexpr int kRowsOfAWave = 256;
template <typename T>
__device__ __forceinline__ void add_weights(const DifferArgs& a, int splits, int head) {
  __shared__ double lds[16];
  const int kv = head / a.group, g = head % a.group, waves = blockDim.x >> 6;
  double s = 0;
  const uint32_t sets = a.dots ? splits * a.batch : a.batch, each = ((uint32_t)a.queries + kRowsOfAWave - 1) / kRowsOfAWave;
  for (uint32_t unit = threadIdx.x >> 6; unit < sets * each; unit += waves) {   // (fewer than 2^31)
    const uint32_t k = unit / each, split = k / (uint32_t)a.batch;
    const int first = (unit - k * each) * kRowsOfAWave + (threadIdx.x & 63);
    const int64_t bkv = (int64_t)(k - split * a.batch) * a.kv_heads + kv;
    const float* from = (a.dots ? a.dots + split * own_rows(a) : a.delta) + own_row(a, bkv, (int64_t)g * a.queries, 1);
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = first + 64 * j < a.queries ? from[first + 64 * j] : 0.0f;
    s += ((double)x[0] + (double)x[1]) + ((double)x[2] + (double)x[3]);
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  double sum = 0;
  for (int k = 0; k < waves; ++k) sum += lds[k];
  const float all = (float)-sum;
  if (a.wide_weights) ((float*)a.dweights)[head] = all;
  else ((T*)a.dweights)[head] = from_f<T>(all);
}
template <typename T, int>
__global__ __launch_bounds__(1024) void differ_weights_kernel(const DifferArgs a) {
  add_weights<T>(a, a.splits, blockIdx.x);
}

template <typename T, int CH, bool FOUR>
__global__ __launch_bounds__(256, CH <= 6 ? 2 : 1) void differ_query_grad_kernel(const DifferArgs a) {
  constexpr int R = 32, LD = F32Tile<CH>::LD;
  __shared__ __attribute__((aligned(16))) float tile[F32Tile<CH>::FLOATS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, q4 = lane >> 4;
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)a.row_tiles * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = (uint32_t)at.x % (uint32_t)a.splits, row_tile = row_tile_of(a, (uint32_t)at.x / (uint32_t)a.splits);
  const int n = keys_that_count(a, b);
  const int64_t first = (int64_t)row_tile * kBlockRows, last = min(first + kBlockRows, a.rows) - 1;
  const int tiles = (most_seen(a, first, last, n) + R - 1) / R, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = first + wave * 16 + col;
  const bool here = r < a.rows, idle = first + wave * 16 >= a.rows;
  float offset[2], delta[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) offset[m] = offset_of(here ? a.lse[lse_at(a, b, kv, r, m)] : -INFINITY);
  const bool takes_part = offset[0] != INFINITY;
#pragma unroll
  for (int m = 0; m < 2; ++m) delta[m] = takes_part ? a.delta[own_row(a, bkv, r, m)] : 0.0f;
  const int seen = takes_part ? seen_by(a, r, n) : 0;
  const float w = here ? weight_of<T>(a, head_of_row(a, kv, r)) : 0.0f, unit = a.scale * kLog2e;
  float qf[2][CH][4], gf[2 * CH][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) f32_operands<T, CH>((const T*)a.q.p + (here ? map_row_at(a.q, a, b, kv, r, m) : 0), q4, a.head, takes_part, qf[m]);
  f32_operands<T, 2 * CH>((const T*)a.go.p + (here ? row_at(a.go, a, b, kv, r) : 0), q4, 2 * a.head, takes_part, gf);
  float4_t dq[2][CH];
  float dot[2] = {0.0f, 0.0f};   // of 16-bit tensors D again, for the gradients of weights and keys (o and second are rounded)
#pragma unroll
  for (int m = 0; m < 2; ++m) f32_zero(dq[m]);
  const T* kp = (const T*)a.k.p + b * a.k.b + 2 * kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  TripleAhead<T, CH, 256, FOUR> next;
  int counts = 0;
  auto fetch = [&](int t) {
    next.load([&](int j, int which) { return kp + min(t * R + j, n - 1) * a.k.t + which * a.k.h; }, [&](int j) { return vp + min(t * R + j, n - 1) * a.v.t; },
              a.head, threadIdx.x);
    counts = key_word(a, b, t * R + (lane & 31), n);
  };
#pragma unroll 1
  for (int sweep = kHalves<T> && tiles * R <= kTwice ? 0 : 1; sweep < 2; ++sweep) {   // the first one, if any, for D alone, of all splits' keys
    const int first_tile = sweep ? t0 : 0, end = sweep ? t1 : tiles;
    if (first_tile < end) fetch(first_tile);
    for (int t = first_tile; t < end; ++t) {
      __syncthreads();
      const uint32_t valid = (uint32_t)__ballot(counts != 0);
      next.store(tile, valid, a.head, threadIdx.x);
      __syncthreads();
      if (t + 1 < end) fetch(t + 1);
      if (idle) continue;
      const uint32_t mine = valid & first_bits(seen - t * R);
      float4_t dp[2];
      f32_over_head<CH, 2 * CH>(tile + col * LD + 4 * q4 + 32 * CH, gf, dp);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float4_t s[2];
        f32_over_head<CH, CH>(tile + col * LD + 4 * q4 + m * 16 * CH, qf[m], s);
        const float by = m ? -w : 1.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool sees = f32_bit(mine, k, i, q4);
            const float p = exp2_(s[k][i] * unit - offset[m]);
            if constexpr (kHalves<T>) dot[m] += sees ? p * dp[k][i] : 0.0f;
            s[k][i] = sees ? by * p * (dp[k][i] - delta[m]) : 0.0f;
          }
        if (kHalves<T> && sweep == 0) continue;
        f32_over_rows<CH, CH>(tile + 4 * q4 * LD + col + m * 16 * CH, s, dq[m]);
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
      if constexpr (kHalves<T>) dot[m] = quarters_sum(dot[m]);
    if (sweep) break;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      delta[m] = dot[m];
      dot[m] = 0.0f;
    }
  }
  if (!here) return;
  if constexpr (kHalves<T>) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
      if (q4 == 0) {
        a.dots[split * own_rows(a) + own_row(a, bkv, r, m)] = dot[m];
        if (a.splits == 1) a.delta[own_row(a, bkv, r, m)] = dot[m];   // (the row's own, read above.  Else differ_sum_rows_kernel does)
      }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (a.splits > 1) f32_store<FOUR>(a.part + (split * own_rows(a) + own_row(a, bkv, r, m)) * a.head, dq[m], a.scale, q4, a.head);
    else f32_store<FOUR>((T*)a.dq + dense_map_row_at(a, b, kv, r, m), dq[m], a.scale, q4, a.head);
  }
}

template <typename T, int CH, bool FOUR>
__global__ __launch_bounds__(256, CH <= 4 ? 2 : 1) void differ_key_grad_kernel(const DifferArgs a) {
  constexpr int R = 32, LD = F32Tile<CH>::LD;
  __shared__ __attribute__((aligned(16))) float tile[F32Tile<CH>::FLOATS];
  __shared__ __attribute__((aligned(16))) float offsets[2][R], deltas[2][R], weights[R], seen_by_row[R];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, q4 = lane >> 4;
  const int blocks = key_blocks_of(a);
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)blocks * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = (uint32_t)at.x % (uint32_t)a.splits, block = (uint32_t)at.x / (uint32_t)a.splits;
  const int n = keys_that_count(a, b);
  const float unit = a.scale * kLog2e;
#pragma unroll 1
  for (int key_tile = block;; key_tile = a.key_tiles - 1 - block) {
    const int first = key_tile * kBlockRows, key = first + wave * 16 + col;
    const bool here = key < a.keys, counts = key_counts(a, b, key, n), idle = first + wave * 16 >= n;
    const int i_min = a.causal ? first - (n - a.queries) : 0;   // the first query that sees one of the block's keys
    int t0 = 0, t1 = 0;
    if (first < n) {   // else no key of the block counts: its gradients are zero
      t0 = first_row_tile(a, split, R, i_min);
      t1 = first_row_tile(a, split + 1, R, i_min);
    }
    const int64_t row = here && counts ? key : 0;
    float kf[2][CH][4], vf[2 * CH][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
      f32_operands<T, CH>((const T*)a.k.p + (counts ? b * a.k.b + (2 * kv + m) * a.k.h + row * a.k.t : 0), q4, a.head, counts, kf[m]);
    f32_operands<T, 2 * CH>((const T*)a.v.p + (counts ? b * a.v.b + kv * a.v.h + row * a.v.t : 0), q4, 2 * a.head, counts, vf);
    float4_t dk[2][CH], dv[2 * CH];
#pragma unroll
    for (int m = 0; m < 2; ++m) f32_zero(dk[m]);
    f32_zero(dv);
    TripleAhead<T, CH, 256, FOUR> next;
    float next_offset[2] = {INFINITY, INFINITY}, next_delta[2] = {0, 0}, next_weight = 0;
    int next_seen = 0;
    auto fetch = [&](int t) {
      auto row = [&](int j) { return min((int64_t)t * R + j, a.rows - 1); };
      next.load([&](int j, int which) { return (const T*)a.q.p + map_row_at(a.q, a, b, kv, row(j), which); },
                [&](int j) { return (const T*)a.go.p + row_at(a.go, a, b, kv, row(j)); }, a.head, threadIdx.x);
      // (every wave of its own: which rows take part decides what the tile's rows are)
      const int64_t r = (int64_t)t * R + (lane & 31);
      const bool is = r < a.rows;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        next_offset[m] = offset_of(is ? a.lse[lse_at(a, b, kv, r, m)] : -INFINITY);
        next_delta[m] = is ? a.delta[own_row(a, bkv, r, m)] : 0.0f;
      }
      next_weight = is ? weight_of<T>(a, head_of_row(a, kv, r)) : 0.0f;
      next_seen = is ? seen_by(a, r, n) : 0;
    };
    int t = next_row_tile(a, t0, R, i_min);
    if (t < t1) fetch(t);
    while (t < t1) {
      __syncthreads();
      // a row without keys counts for nothing: what it holds must not reach the sums
      next.store(tile, (uint32_t)__ballot(next_offset[0] != INFINITY), a.head, threadIdx.x);
      if (threadIdx.x < R) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          offsets[m][threadIdx.x] = next_offset[m];
          deltas[m][threadIdx.x] = next_delta[m];
        }
        weights[threadIdx.x] = next_weight;
        seen_by_row[threadIdx.x] = __builtin_bit_cast(float, next_seen);
      }
      __syncthreads();
      t = next_row_tile(a, t + 1, R, i_min);
      if (t < t1) fetch(t);
      if (idle) continue;
      float4_t s[2][2], dp[2], both[2];
      bool sees[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) f32_over_head<CH, CH>(tile + col * LD + 4 * q4 + m * 16 * CH, kf[m], s[m]);
      f32_over_head<CH, 2 * CH>(tile + col * LD + 4 * q4 + 32 * CH, vf, dp);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 16 * k + 4 * q4 + i;
          sees[k][i] = key < __builtin_bit_cast(int, seen_by_row[j]);
          const float w = weights[j];
#pragma unroll
          for (int m = 0; m < 2; ++m) s[m][k][i] = sees[k][i] ? exp2_(s[m][k][i] * unit - offsets[m][j]) : 0.0f;
          both[k][i] = s[0][k][i] - w * s[1][k][i];
          s[0][k][i] *= sees[k][i] ? dp[k][i] - deltas[0][j] : 0.0f;
          s[1][k][i] *= sees[k][i] ? -w * (dp[k][i] - deltas[1][j]) : 0.0f;
        }
      f32_over_rows<CH, 2 * CH>(tile + 4 * q4 * LD + col + 32 * CH, both, dv);
#pragma unroll
      for (int m = 0; m < 2; ++m) f32_over_rows<CH, CH>(tile + 4 * q4 * LD + col + m * 16 * CH, s[m], dk[m]);
    }
    if (here) {
      if (!counts) {
#pragma unroll
        for (int m = 0; m < 2; ++m) f32_zero(dk[m]);
        f32_zero(dv);
      }
      const int64_t dense = ((b * (int64_t)a.keys + key) * a.kv_heads + kv) * 2 * a.head;   // of dv; of dk's first map as well
      if (a.splits > 1) {
        const int64_t all = (int64_t)a.batch * a.keys * a.kv_heads * 2 * a.head;
#pragma unroll
        for (int m = 0; m < 2; ++m) f32_store<FOUR>(a.part + split * all + dense + m * a.head, dk[m], a.scale, q4, a.head);
        f32_store<FOUR>(a.part + (a.splits + split) * all + dense, dv, 1.0f, q4, 2 * a.head);
      } else {
#pragma unroll
        for (int m = 0; m < 2; ++m) f32_store<FOUR>((T*)a.dk + dense + m * a.head, dk[m], a.scale, q4, a.head);
        f32_store<FOUR>((T*)a.dv + dense, dv, 1.0f, q4, 2 * a.head);
      }
    }
    if (key_tile != block || blocks == a.key_tiles || a.key_tiles - 1 - block == block) break;
  }
}

// dk[e] = sum over splits of part[s][e], in order, and dv[e] of those behind (the second half of the blocks).  The first `heads` blocks add the weights' gradients.
template <typename T, int>
__global__ __launch_bounds__(256) void differ_sum_kernel(const DifferArgs a, int heads, int query_splits, int64_t n) {
  if ((int)blockIdx.x < heads) {
    add_weights<T>(a, query_splits, blockIdx.x);
    return;
  }
  const uint32_t half = (gridDim.x - heads) / 2, which = blockIdx.x - heads >= half;
  const int64_t e = (int64_t)(blockIdx.x - heads - which * half) * 256 + threadIdx.x;
  if (e >= n) return;
  const int splits = a.splits;
  const float* __restrict__ part = a.part + which * splits * n + e;
  float s = 0.0f;
  for (int k = 0; k < splits; k += 4) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < splits ? part[(k + i) * n] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += v[i];
  }
  ((T*)(which ? a.dv : a.dk))[e] = from_f<T>(s);
}
// dq's maps' rows from the splits', written in the order of the tensor, and D of 16-bit tensors: a wave a row
template <typename T, int>
__global__ __launch_bounds__(256) void differ_sum_rows_kernel(const DifferArgs a) {
  const int64_t all = own_rows(a), own = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (own >= all) return;
  const uint32_t rows = (uint32_t)a.rows, set = (uint32_t)own / rows, b = set / 2 / (uint32_t)a.kv_heads;   // (a call that is split has fewer than 2^23 rows)
  const int64_t bkv = set / 2, r = own - (int64_t)set * rows;
  const int m = set % 2;
  T* row = (T*)a.dq + dense_map_row_at(a, b, (int)bkv - b * a.kv_heads, r, m);
  if (a.dots && (threadIdx.x & 63) == 0) {
    float s = 0.0f;
    for (int k = 0; k < a.splits; ++k) s += a.dots[k * all + own];
    (a.info ? *info_at(a, bkv, r, kDelta0 + m) : a.delta[own]) = s;
  }
  for (int d = threadIdx.x & 63; d < a.head; d += 64) {
    float s = 0.0f;
    for (int k = 0; k < a.splits; ++k) s += a.part[(k * all + own) * a.head + d];
    row[d] = from_f<T>(s);
  }
}

struct GradCut {
  int row_tiles, key_tiles, key_blocks, query_splits, key_splits;
  int64_t delta, info, dots, part;   // floats of the workspace
};
GradCut grad_cut(int64_t batch, int64_t kv_heads, int64_t queries, int64_t rows, int64_t keys, int64_t head, bool causal, bool halves, bool by16) {
  GradCut c;
  c.row_tiles = (int)ceil_div(rows, by16 ? differ_grad16_tile(head) : kBlockRows);
  c.key_tiles = (int)ceil_div(keys, by16 ? differ_key_grad16_tile(head) : kBlockRows);
  c.key_blocks = key_blocks_of(c.key_tiles, queries, keys, causal);
  // blocks that the chip holds at once; what starting a block, and adding splits up, costs in tiles of 32 rows.  A tile takes the 16-bit kernels a microsecond or more: a launch is
  // three, and so are 12 MB of parts.  (With half of the second pieces, 2 x 200 x 300, 4 heads of 40 in f16: 59 us, with twelve for every sum 95; 8 x 577 x 1000, 12 heads of 64: 275, with four 314.)
  const int64_t start = by16 ? 6 : 2, heads = batch * kv_heads;
  auto join = [&](int64_t values) { return by16 ? 3 + 16 * values / 4000000 : 3; };   // of f32, of two splits, written and read
  c.query_splits = split_of(heads * c.row_tiles, ceil_div(keys, 32), 2, by16 || head > 96 ? 256 : 512, start, join(heads * 2 * rows * head));
  const int64_t useful = causal ? std::min(queries, keys) * (rows / std::max<int64_t>(queries, 1)) : rows;   // rows that see a key
  c.key_splits = split_of(heads * c.key_blocks, ceil_div(useful, 32), 2, by16 || head > 64 ? 256 : 512, start, join(heads * 4 * keys * head));
  c.delta = round_up(batch * kv_heads * 2 * rows, 64);
  c.info = by16 ? batch * kv_heads * kInfos * round_up(rows, kInfoRows) : 0;
  c.dots = halves ? round_up(c.query_splits * batch * kv_heads * 2 * rows, 64) : 0;
  const int64_t q = c.query_splits > 1 ? c.query_splits * batch * kv_heads * 2 * rows * head : 0;
  const int64_t k = c.key_splits > 1 ? 2 * c.key_splits * batch * kv_heads * keys * 2 * head : 0;
  c.part = std::max(q, k);
  return c;
}

template <typename T>
constexpr int kType = std::is_same_v<T, float> ? NNVHIP_TYPE_F32 : std::is_same_v<T, bf16_t> ? NNVHIP_TYPE_BF16 : NNVHIP_TYPE_F16;
template <typename T, int CH>
void launch_grad(DifferArgs a, const GradCut& c, bool by16, hipStream_t st) {
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  const bool four = a.head % 4 == 0;
  if (a.rows > 0 && heads > 0) {
    hipLaunchKernelGGL((differ_delta_kernel<T, 0>), dim3((unsigned)ceil_div(heads * (a.info ? a.info_rows : a.rows), 16)), dim3(256), 0, st, a);
    a.row_tiles = c.row_tiles;
    a.splits = c.query_splits;
    const dim3 grid((unsigned)(heads * c.row_tiles * a.splits));
    if (by16) launch_differ_query_grad16(a, kType<T>, st);
    else if (four) hipLaunchKernelGGL((differ_query_grad_kernel<T, CH, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((differ_query_grad_kernel<T, CH, false>), grid, dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL((differ_sum_rows_kernel<T, 0>), dim3((unsigned)ceil_div(heads * 2 * a.rows, 4)), dim3(256), 0, st, a);
  } else {
    a.batch = 0;   // (for the sums over no rows)
  }
  // the weights' gradients beside the sums of dk and dv, where there are such and a wave there takes sixteen turns at most
  const int64_t turns = ceil_div((a.dots ? a.splits : 1) * (int64_t)a.batch * ceil_div(a.queries, kRowsOfAWave), 4);
  const int beside = a.batch > 0 && a.keys > 0 && c.key_splits > 1 && turns <= 16 ? a.kv_heads * a.group : 0, query_splits = a.splits;
  if (!beside) hipLaunchKernelGGL((differ_weights_kernel<T, 0>), dim3((unsigned)(a.kv_heads * a.group)), dim3(1024), 0, st, a);
  if (a.keys > 0 && heads > 0) {
    a.batch = (int)(heads / a.kv_heads);
    a.key_tiles = c.key_tiles;
    a.splits = c.key_splits;
    const dim3 grid((unsigned)(heads * c.key_blocks * a.splits));
    if (by16) launch_differ_key_grad16(a, kType<T>, st);
    else if (four) hipLaunchKernelGGL((differ_key_grad_kernel<T, CH, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((differ_key_grad_kernel<T, CH, false>), grid, dim3(256), 0, st, a);
    if (a.splits > 1) {
      const int64_t n = heads * a.keys * 2 * a.head;
      hipLaunchKernelGGL((differ_sum_kernel<T, 0>), dim3((unsigned)(beside + 2 * ceil_div(n, 256))), dim3(256), 0, st, a, beside, query_splits, n);
    }
  }
}

}  // namespace
}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_differential_attention_backward_workspace(const nnvhip_differ_args* d, int64_t* bytes) {
  int64_t forward = 0;
  NNV_TRY(nnvhip_differential_attention_workspace(d, &forward));   // checks the sizes
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  const int64_t heads = d->batch * d->kv_heads, blocks = kMostBlocks;
  if (ceil_div(heads * round_up(d->queries * (d->heads / d->kv_heads), kInfoRows), 16) > 2 * blocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_differential_attention_backward: too many rows");
  if (heads * ceil_div(d->keys, kBlockRows) > blocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_differential_attention_backward: too many keys");
  *bytes = 0;   // whichever kernels the alignment of the tensors lets take the call
  for (const bool by16 : {false, true}) {
    const GradCut c = grad_cut(d->batch, d->kv_heads, d->queries, d->queries * (d->heads / d->kv_heads), d->keys, d->head, d->causal != 0, d->type != NNVHIP_TYPE_F32, by16);
    if (heads * c.row_tiles * c.query_splits > blocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_differential_attention_backward: too many rows");
    if (heads * c.key_blocks * c.key_splits > blocks || (c.key_splits > 1 && ceil_div(heads * d->keys * 2 * d->head, 256) > blocks))
      NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_differential_attention_backward: too many keys");
    *bytes = std::max(*bytes, (c.delta + c.info + c.dots + c.part) * (int64_t)sizeof(float));
  }
  return NNVHIP_OK;
}

int nnvhip_differential_attention_backward(nnvhip_ctx* ctx, const nnvhip_differ_args* d, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  DifferArgs a;
  NNV_TRY(differ_args("nnvhip_differential_attention_backward", d, true, &a));
  int64_t need = 0;
  NNV_TRY(nnvhip_differential_attention_backward_workspace(d, &need));
  if (need > workspace_bytes || (need && !workspace))
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_differential_attention_backward: a workspace of %lld bytes is needed", (long long)need);
  const bool by16 = differ_grad16_takes(a, (int)d->type);
  const GradCut c = grad_cut(a.batch, a.kv_heads, a.queries, a.rows, a.keys, a.head, a.causal, d->type != NNVHIP_TYPE_F32, by16);
  a.delta = static_cast<float*>(workspace);
  a.info = c.info ? a.delta + c.delta : nullptr;
  a.info_rows = (int)round_up(a.rows, kInfoRows);
  a.dots = c.dots ? a.delta + c.delta + c.info : nullptr;
  a.part = a.delta + c.delta + c.info + c.dots;
  DIFFER_BY_TYPE(d->type, launch_grad, a, c, by16, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
