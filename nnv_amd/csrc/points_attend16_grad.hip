// Attention of points in bf16, backward, on v_mfma_f32_32x32x16_bf16: the 16-bit forms of query_grad_kernel and key_grad_kernel.
//
// The weights P, and the gradients dS of the scores, are rounded to bf16 before the products that use them.  (Not f16: a
// gradient of a score is a weight, often far below one, times a difference, and leaves f16's range on either side; f16
// tensors take the f32 products.)
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
template <typename T, int DP>
__device__ __forceinline__ float16_t over_head(const T* tile, int first, const half8<T> (&f)[DP / 16], int col, int h) {
  float16_t s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) s = Half8<T>::mfma(rows_operand<T, DP>(tile, first, c, col, h), f[c], s);
  return s;
}
template <typename T, int DP>
__device__ __forceinline__ void over_rows(const T* tile, int first, const float16_t& p, float16_t (&acc)[DP / 32], int lane) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const half8<T> f = round8<T>(p, 8 * c);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = Half8<T>::mfma(columns_operand<T, DP>(tile, first + 16 * c, d, lane), f, acc[d]);
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
// rows of a tile that do not take part, as zeros
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void zero_rows(T* tile, uint64_t valid) {
  half8<T> none = {};
  for (int e = threadIdx.x; e < ROWS * (DP / 8); e += THREADS)
    if (!(valid >> (e / (DP / 8)) & 1)) __builtin_memcpy(tile + e * 8, &none, 16);
}
template <typename T, int PACKS, int THREADS>
__device__ __forceinline__ void zero_all(T* lds) {
  half8<T> none = {};
  for (int e = threadIdx.x; e < PACKS; e += THREADS) __builtin_memcpy(lds + e * 8, &none, 16);
  __syncthreads();
}

template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void query_grad16_kernel(const AttendArgs a) {
  constexpr int KEYS = 64, TILE = KEYS * DP;
  typedef PairLoad<T, DP, KEYS, WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[4 * TILE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int bkv = at / a.row_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int tiles = (n + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = (int64_t)row_tile * (32 * WAVES) + wave * 32 + col, flat = (int64_t)bkv * a.rows + r;
  const bool here = r < a.rows;
  const unsigned lds_at = lds_addr_of(lds);
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
  load.init(wave, lane, a.head);
  bool counts = false;
  auto fetch = [&](int t, int buffer) {
    load.issue([&](int j) { return kp + (int64_t)min(t * KEYS + j, n - 1) * a.k.t; },
               [&](int j) { return vp + (int64_t)min(t * KEYS + j, n - 1) * a.v.t; }, lds_at + buffer * (4 * TILE), wave);
    counts = key_counts(a, b, t * KEYS + lane, n);
  };
  int buffer = 0;
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t, buffer ^= 1) {
    const uint64_t valid = __ballot(counts);
    T* ks = lds + buffer * 2 * TILE;
    T* vs = ks + TILE;
    wait_vm_lds<0>();
    block_barrier();
    if (t + 1 < t1) fetch(t + 1, buffer ^ 1);
    if (valid != ~0ull) {
      zero_rows<T, DP, KEYS, 64 * WAVES>(ks, valid);
      wait_vm_lds<63>();
      block_barrier();
    }
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k) {
      float16_t s = over_head<T, DP>(ks, 32 * k, qf, col, h);
      const float16_t dp = over_head<T, DP>(vs, 32 * k, gf, col, h);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = exp2_(s[i] * unit - offset) * (dp[i] - delta);
      if (valid != ~0ull) {
        const uint32_t word = (uint32_t)(valid >> (32 * k)) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = word >> product_row(i, 0) & 1 ? s[i] : 0.0f;
      }
      over_rows<T, DP>(ks, 32 * k, s, dq, lane);
    }
  }
  if (!here) return;
  if (a.splits > 1)
    store_result<float, DP>(a.part + ((int64_t)split * a.batch * a.kv_heads * a.rows + flat) * a.head, dq, a.scale, h, a.head);
  else
    store_result<T, DP>((T*)a.dq + dense_row_at(a, b, kv, r), dq, a.scale, h, a.head);
}

template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void key_grad16_kernel(const AttendArgs a) {
  constexpr int ROWS = 64, TILE = ROWS * DP;
  typedef PairLoad<T, DP, ROWS, WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[4 * TILE];
  __shared__ __attribute__((aligned(16))) float offsets[2][ROWS], deltas[2][ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int key_tile = at % a.key_tiles;
  const int bkv = at / a.key_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int key = key_tile * (32 * WAVES) + wave * 32 + col;
  const bool here = key < a.keys, counts = key_counts(a, b, key, n);
  const unsigned lds_at = lds_addr_of(lds);
  if (DP != a.head) zero_all<T, 4 * TILE / 8, 64 * WAVES>(lds);
  // where no key of the block counts there is nothing to add up (and rows without any key take part in no block)
  const bool any = __syncthreads_or(counts);
  const int tiles = any ? (int)((a.rows + ROWS - 1) / ROWS) : 0, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);

  half8<T> kf[DP / 16], vf[DP / 16];
  load_operands<T, DP>(kf, (const T*)a.k.p + (counts ? b * a.k.b + kv * a.k.h + key * a.k.t : 0), h, a.head, counts);
  load_operands<T, DP>(vf, (const T*)a.v.p + (counts ? b * a.v.b + kv * a.v.h + key * a.v.t : 0), h, a.head, counts);
  const float unit = a.scale * kLog2e;
  float16_t dk[DP / 32], dv[DP / 32];
  zero<DP>(dk);
  zero<DP>(dv);
  const float* lse = a.lse + (int64_t)bkv * a.rows;
  const float* del = a.delta + (int64_t)bkv * a.rows;
  Load load;
  load.init(wave, lane, a.head);
  float next_offset = 0.0f, next_delta = 0.0f;
  auto fetch = [&](int t, int buffer) {
    // rows past the last one repeat it, and are made zeros below
    auto row = [&](int j) { return min((int64_t)t * ROWS + j, a.rows - 1); };
    load.issue([&](int j) { return (const T*)a.q.p + row_at(a.q, a, b, kv, row(j)); },
               [&](int j) { return (const T*)a.go.p + row_at(a.go, a, b, kv, row(j)); }, lds_at + buffer * (4 * TILE), wave);
    if (threadIdx.x < ROWS) {
      const int64_t r = (int64_t)t * ROWS + threadIdx.x;
      const float x = lse[row(threadIdx.x)];
      next_offset = r < a.rows && x != -INFINITY ? x * kLog2e : INFINITY;
      next_delta = r < a.rows ? del[row(threadIdx.x)] : 0.0f;
    }
  };
  int buffer = 0;
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t, buffer ^= 1) {
    T* qs = lds + buffer * 2 * TILE;
    T* gs = qs + TILE;
    if (threadIdx.x < ROWS) {
      offsets[buffer][threadIdx.x] = next_offset;
      deltas[buffer][threadIdx.x] = next_delta;
    }
    wait_vm_lds<0>();
    block_barrier();
    if (t + 1 < t1) fetch(t + 1, buffer ^ 1);
    if ((int64_t)(t + 1) * ROWS > a.rows) {
      const uint64_t valid = (1ull << (int)(a.rows - (int64_t)t * ROWS)) - 1;
      zero_rows<T, DP, ROWS, 64 * WAVES>(qs, valid);
      zero_rows<T, DP, ROWS, 64 * WAVES>(gs, valid);
      wait_vm_lds<63>();
      block_barrier();
    }
#pragma unroll
    for (int k = 0; k < ROWS / 32; ++k) {
      float16_t s = over_head<T, DP>(qs, 32 * k, kf, col, h);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
        __builtin_memcpy(f, &offsets[buffer][32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * i4 + i] = counts ? exp2_(s[4 * i4 + i] * unit - f[i]) : 0.0f;
      }
      const float16_t dp = over_head<T, DP>(gs, 32 * k, vf, col, h);
      over_rows<T, DP>(gs, 32 * k, s, dv, lane);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
        __builtin_memcpy(f, &deltas[buffer][32 * k + 8 * i4 + 4 * h], 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * i4 + i] *= dp[4 * i4 + i] - f[i];
      }
      over_rows<T, DP>(qs, 32 * k, s, dk, lane);
    }
  }
  if (!here) return;
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
  hipLaunchKernelGGL((key_grad16_kernel<T, DP, 4>), dim3((unsigned)((int64_t)a.batch * a.kv_heads * a.key_tiles * a.splits)), dim3(256), 0,
                     st, a);
}

}  // namespace

bool grad16_takes(const AttendArgs& a, int type) {
  return type == NNVHIP_TYPE_BF16 && by_pieces(a.q, a.head) && by_pieces(a.k, a.head) && by_pieces(a.v, a.head) && by_pieces(a.go, a.head);
}
void launch_query_grad16(const AttendArgs& a, hipStream_t st) { ATTEND_BY_HEAD(launch_query, bf16_t, a, st); }
void launch_key_grad16(const AttendArgs& a, hipStream_t st) { ATTEND_BY_HEAD(launch_key, bf16_t, a, st); }

}  // namespace nnvhip
