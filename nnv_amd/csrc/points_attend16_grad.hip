// Attention of points in bf16, backward, on v_mfma_f32_32x32x16_bf16: the 16-bit forms of query_grad_kernel and key_grad_kernel.
//
// The weights P, and the gradients dS of the scores, are rounded to bf16 before the products that use them, whatever the number of rows; D comes from the o
// that the forward pass rounded.  The error against 64 bits is 0.0024 of the largest gradient, 0.0017 of it the results' own rounding.  (Not f16: a
// gradient of a score is a weight, often far below one, times a difference, and leaves f16's range on either side; f16
// tensors take the products in pieces.)
//
// Bound by the power that the seven products may take: 2 x 4096 x 4096, 32 heads of 128 (8 for keys), 1770 us: 28 for D, 726 for dq, 1040 for dk and dv;
// 780 TFLOP/s of the five products that one kernel would need, 1090 of all.  4 x 2048 x 2048, 16 heads of 64: 285 us, 600 TFLOP/s.
#include "points_attend16.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

template <typename T, int DP>
__device__ __forceinline__ void load_operands(half8<T> (&f)[DP / 16], const T* row, int h, int head, bool there) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    f[c] = half8<T>{};
    if (there && 16 * c + 8 * h < head) __builtin_memcpy(&f[c], row + 16 * c + 8 * h, 16);
  }
}
template <int DP>
__device__ __forceinline__ void zero(float16_t (&acc)[DP / 32]) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
}
// over_head with the operands of the row in LDS as well (16 bytes a lane, 1024 bytes apart), read along with the tile's.
template <typename T, int DP>
__device__ __forceinline__ void over_head_parked(unsigned tile, int first, const T* parked, float16_t& s) {
  constexpr int N = DP / 16, BATCH = 2;
  half8<T> x[2][BATCH], f[2][BATCH];
  auto read = [&](int n) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      x[n & 1][i] = rows_operand<T, DP>(tile, first, n * BATCH + i);
      __builtin_memcpy(&f[n & 1][i], parked + 512 * (n * BATCH + i), 16);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
  read(0);
#pragma unroll
  for (int n = 0; n < N / BATCH; ++n) {
    if (n + 1 < N / BATCH) read(n + 1);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) s = Half8<T>::mfma(x[n & 1][i], f[n & 1][i], s);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <typename T, int DP>
__device__ __forceinline__ void over_rows(unsigned tile, int first, const float16_t& p, float16_t (&acc)[DP / 32]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const half8<T> f = round8<T>(p, 8 * c);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = Half8<T>::mfma(columns_operand<T, DP>(tile, first + 16 * c, d), f, acc[d]);
  }
}
template <typename T, int DP>
__device__ __forceinline__ void store_result(T* row, const float16_t (&acc)[DP / 32], float by, int h, int head) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = acc[d][4 * i4 + i] * by;
      store_four(row, d * 32 + 8 * i4 + 4 * h, head, f);
    }
}
template <typename T, int PACKS, int THREADS>
__device__ __forceinline__ void zero_all(T* lds) {
  half8<T> none = {};
  for (int e = threadIdx.x; e < PACKS; e += THREADS) __builtin_memcpy(lds + e * 8, &none, 16);
  __syncthreads();
}

// Eight waves share a tile of keys (heads of 128 in blocks of four: 812 us for dq above instead of 740).
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void query_grad16_kernel(const AttendArgs a) {
  constexpr int KEYS = 64, TILE = KEYS * DP;
  typedef PairLoad<T, DP, KEYS, WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[4 * TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int b = (int)(at / a.row_tiles) % a.batch, kv = (int)(at / a.row_tiles) / a.batch, bkv = b * a.kv_heads + kv;
  const int n = keys_that_count(a, b);
  const int tiles = (n + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = (int64_t)row_tile * (32 * WAVES) + wave * 32 + col, flat = (int64_t)bkv * a.rows + r;
  const bool here = r < a.rows;
  const unsigned lds_at = lds_addr_of(lds), rows_at = rows_place<T, DP>(lane), columns_at = columns_place<T, DP>(lane);
  if (DP != a.head) zero_all<T, 4 * TILE / 8, 64 * WAVES>(lds);

  const float lse = here ? a.lse[flat] : -INFINITY;
  const bool takes_part = lse != -INFINITY;
  const float offset = takes_part ? lse * kLog2e : INFINITY, delta = takes_part ? a.delta[flat] : 0.0f, unit = a.scale * kLog2e;
  half8<T> qf[DP / 16], gf[DP / 16];
  load_operands<T, DP>(qf, (const T*)a.q.p + (here ? row_at(a.q, a, b, kv, r) : 0), h, a.head, takes_part);
  load_operands<T, DP>(gf, (const T*)a.go.p + (here ? row_at(a.go, a, b, kv, r) : 0), h, a.head, takes_part);
  float16_t dq[DP / 32];
  zero<DP>(dq);
  const T* kp = (const T*)a.k.p + b * a.k.b + kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(wave, lane, a.head, a.k.t, a.v.t);
  int counts = 0;
  auto fetch = [&](int t, int buffer) {
    load.issue_tile(t, n, kp, a.k.t, vp, a.v.t, lds_at + buffer * (4 * TILE), wave, lane);
    counts = key_word(a, b, t * KEYS + lane, n);
  };
  int buffer = 0;
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t, buffer ^= 1) {
    const uint64_t valid = __ballot(counts != 0);
    const unsigned pair = lds_at + buffer * (4 * TILE);
    const unsigned ks_at = hide(pair + rows_at), vs_at = ks_at + 2 * TILE, kc_at = hide(pair + columns_at);
    wait_vm_lds<0>();
    block_barrier();
    if (t + 1 < t1) fetch(t + 1, buffer ^ 1);
    if (valid != ~0ull) {
      zero_rows<T, DP, KEYS>(lds + buffer * 2 * TILE, valid, lane);
    }
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k) {
      float16_t ps[1], dps[1];
      over_head<T, DP, 1>(ks_at, 32 * k, qf, ps);
      over_head<T, DP, 1>(vs_at, 32 * k, gf, dps);
      float16_t& s = ps[0];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = exp2_(s[i] * unit - offset) * (dps[0][i] - delta);
      if (valid != ~0ull) {
        const uint32_t word = (uint32_t)(valid >> (32 * k)) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = word >> product_row(i, 0) & 1 ? s[i] : 0.0f;
      }
      over_rows<T, DP>(kc_at, 32 * k, s, dq);
    }
  }
  if (!here) return;
  if (a.splits > 1)
    store_result<float, DP>(a.part + ((int64_t)split * a.batch * a.kv_heads * a.rows + flat) * a.head, dq, a.scale, h, a.head);
  else
    store_result<T, DP>((T*)a.dq + dense_row_at(a, b, kv, r), dq, a.scale, h, a.head);
}

// Two waves a SIMD, so that one's exponentials run beside the other's products: 256 registers a wave.  The accumulators take 2 DP of them
// and the operands of the wave's keys DP / 2, as many again those of its values, which lie in LDS where they would not fit (heads of 96: 4 x 2048 x 2048, 16
// heads, 396 us with them in registers, 403 without).  Three registers of heads of 128 are spilled all the same.  Eight waves a block for heads above 64 (four: 1930 us for the gradients above), else four (eight:
// 8 x 448 x 1500 by length, 16 heads of 64, 125 us instead of 119).
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void key_grad16_kernel(const AttendArgs a) {
  constexpr int ROWS = 64, TILE = ROWS * DP;
  constexpr bool PARKED = DP > 96;   // the values' operands, in LDS
  typedef PairLoad<T, DP, ROWS, WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[4 * TILE + (PARKED ? WAVES * 32 * DP : 0)];
  __shared__ __attribute__((aligned(16))) float offsets[2][ROWS], deltas[2][ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int key_tile = at % a.key_tiles;
  const int b = (int)(at / a.key_tiles) % a.batch, kv = (int)(at / a.key_tiles) / a.batch, bkv = b * a.kv_heads + kv;
  const int n = keys_that_count(a, b);
  const int key = key_tile * (32 * WAVES) + wave * 32 + col;
  const bool here = key < a.keys, counts = key_counts(a, b, key, n);
  const unsigned lds_at = lds_addr_of(lds), rows_at = rows_place<T, DP>(lane), columns_at = columns_place<T, DP>(lane);
  if (DP != a.head) zero_all<T, 4 * TILE / 8, 64 * WAVES>(lds);
  // where no key of the block counts there is nothing to add up (and rows without any key take part in no block)
  const bool any = __syncthreads_or(counts);
  const int tiles = any ? (int)((a.rows + ROWS - 1) / ROWS) : 0, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);

  half8<T> kf[DP / 16], vf[DP / 16];
  T* parked = lds + 4 * TILE + wave * (32 * DP) + lane * 8;   // operand c at parked + 512 c; no other wave's
  load_operands<T, DP>(kf, (const T*)a.k.p + (counts ? b * a.k.b + kv * a.k.h + key * a.k.t : 0), h, a.head, counts);
  load_operands<T, DP>(vf, (const T*)a.v.p + (counts ? b * a.v.b + kv * a.v.h + key * a.v.t : 0), h, a.head, counts);
  if constexpr (PARKED)
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) __builtin_memcpy(parked + 512 * c, &vf[c], 16);
  const float unit = a.scale * kLog2e;
  float16_t dk[DP / 32], dv[DP / 32];
  zero<DP>(dk);
  zero<DP>(dv);
  const float* lse = a.lse + (int64_t)bkv * a.rows;
  const float* del = a.delta + (int64_t)bkv * a.rows;
  Load load;
  load.init(wave, lane, a.head, a.q.t, a.go.t);
  const T* qp = (const T*)a.q.p + b * a.q.b + kv * (int64_t)a.group * a.q.h;
  const T* gp = (const T*)a.go.p + b * a.go.b + kv * (int64_t)a.group * a.go.h;
  const float per_query = 1.0f / a.queries;
  struct Place {
    int head, query;
  };
  float next_lse = 0.0f, next_delta = 0.0f;
  auto fetch = [&](int t, int buffer) {
    // Head of the group and query of the tile's first row, then of every row: a tile reaches into the next head at most where heads have
    // ROWS queries, and the quotient is small where they have fewer.  Rows past the last one repeat it, and are made zeros below.
    const int g0 = (uint32_t)t * ROWS / (uint32_t)a.queries, i0 = t * ROWS - g0 * a.queries, last = (int)a.rows - 1 - g0 * a.queries;
    const unsigned pair = lds_at + buffer * (4 * TILE);
    if (i0 + ROWS <= a.queries) {
      load.issue(qp + (i0 * a.q.t + g0 * a.q.h), gp + (i0 * a.go.t + g0 * a.go.h), pair, wave);
    } else {
      auto where = [&](int j) {
        const int i = min(i0 + j, last);
        const int more = a.queries >= ROWS ? (int)(i >= a.queries) : (int)((i + 0.5f) * per_query);
        return Place{g0 + more, i - more * a.queries};
      };
      auto at_row = [&](const T* p, const TokenView& v, Place w) { return p + (w.query * v.t + w.head * v.h); };
      load.issue_any([&](int j) { return at_row(qp, a.q, where(j)); }, [&](int j) { return at_row(gp, a.go, where(j)); }, pair, wave, lane);
    }
    if (threadIdx.x < ROWS) {
      const int64_t r = (int64_t)t * ROWS + threadIdx.x;
      next_lse = r < a.rows ? lse[r] : -INFINITY;
      next_delta = r < a.rows ? del[r] : 0.0f;
    }
  };
  int buffer = 0;
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t, buffer ^= 1) {
    const unsigned pair = lds_at + buffer * (4 * TILE);
    if (threadIdx.x < ROWS) {
      offsets[buffer][threadIdx.x] = next_lse == -INFINITY ? INFINITY : next_lse * kLog2e;
      deltas[buffer][threadIdx.x] = next_delta;
    }
    wait_vm_lds<0>();
    block_barrier();
    if (t + 1 < t1) fetch(t + 1, buffer ^ 1);
    if ((int64_t)(t + 1) * ROWS > a.rows) {
      const uint64_t valid = (1ull << (int)(a.rows - (int64_t)t * ROWS)) - 1;
      zero_rows<T, DP, ROWS>(lds + buffer * 2 * TILE, valid, lane);
      zero_rows<T, DP, ROWS>(lds + (buffer * 2 + 1) * TILE, valid, lane);
    }
#pragma unroll 1
    for (int k = 0; k < ROWS / 32; ++k) {   // (both at once would need more registers than there are)
      const unsigned rows_k = rows_at + pair + k * (64 * DP), columns_k = columns_at + pair + k * (64 * DP);
      const unsigned qs_at = hide(rows_k), gs_at = qs_at + 2 * TILE, qc_at = hide(columns_k), gc_at = qc_at + 2 * TILE;
      float16_t ps[1], dps[1];
      over_head<T, DP, 1, DP == 128 ? 2 : 4>(qs_at, 0, kf, ps);
      float16_t& s = ps[0];
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
        __builtin_memcpy(f, &offsets[buffer][32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * i4 + i] = exp2_(s[4 * i4 + i] * unit - f[i]);
      }
      if constexpr (PARKED) over_head_parked<T, DP>(gs_at, 0, parked, dps[0]);
      else over_head<T, DP, 1>(gs_at, 0, vf, dps);
      over_rows<T, DP>(gc_at, 0, s, dv);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
        __builtin_memcpy(f, &deltas[buffer][32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * i4 + i] *= dps[0][4 * i4 + i] - f[i];
      }
      over_rows<T, DP>(qc_at, 0, s, dk);
    }
  }
  if (!here) return;
  if (!counts) {   // what the loop made of a column that does not count reached no other one
    zero<DP>(dk);
    zero<DP>(dv);
  }
  const int64_t dense = ((b * (int64_t)a.keys + key) * a.kv_heads + kv) * a.head;
  if (a.splits > 1) {
    const int64_t all = (int64_t)a.batch * a.keys * a.kv_heads * a.head;
    store_result<float, DP>(a.part + split * all + dense, dk, a.scale, h, a.head);
    store_result<float, DP>(a.part + (a.splits + split) * all + dense, dv, 1.0f, h, a.head);
  } else {
    store_result<T, DP>((T*)a.dk + dense, dk, a.scale, h, a.head);
    store_result<T, DP>((T*)a.dv + dense, dv, 1.0f, h, a.head);
  }
}

template <typename T, int DP>
void launch_query(const AttendArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((query_grad16_kernel<T, DP, 8>), dim3((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits)), dim3(512), 0,
                     st, a);
}
template <typename T, int DP>
void launch_key(const AttendArgs& a, hipStream_t st) {
  constexpr int WAVES = DP > 64 ? 8 : 4;
  hipLaunchKernelGGL((key_grad16_kernel<T, DP, WAVES>), dim3((unsigned)((int64_t)a.batch * a.kv_heads * a.key_tiles * a.splits)),
                     dim3(64 * WAVES), 0, st, a);
}

}  // namespace

int key_grad16_tile(int64_t head) { return head > 64 ? 256 : 128; }
bool grad16_takes(const AttendArgs& a, int type) {
  return type == NNVHIP_TYPE_BF16 && by_pieces(a.q, a.head) && by_pieces(a.k, a.head) && by_pieces(a.v, a.head) && by_pieces(a.go, a.head);
}
void launch_query_grad16(const AttendArgs& a, hipStream_t st) { ATTEND_BY_HEAD(launch_query, bf16_t, a, st); }
void launch_key_grad16(const AttendArgs& a, hipStream_t st) { ATTEND_BY_HEAD(launch_key, bf16_t, a, st); }

}  // namespace nnvhip
