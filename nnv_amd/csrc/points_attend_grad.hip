// Attention of points, backward: the kernels for every type, head size and alignment, with f32 products (points_attend_split.h).
//
// Two kernels form dq (a wave per 32 queries, over the keys) and dk, dv (a wave per 32 keys, over the queries of every head that
// shares them).  Both form S and dP again: seven products instead of the five that one kernel would need, but every
// gradient is a sum in the registers of one wave, in a fixed order, with no atomics.  What both need of a row besides, D = rowsum(do o),
// is formed first.  Where one axis gives too few blocks for the chip, the other is split, and sum_kernel adds the parts in order.
//
// Bound by the vector units, which cut what the products take into pieces, and by blocks that are too few: 4 x 333 x 577, 12 heads of 80, in f32 take 157 us
// (5 for D, 92 for dq in 144 blocks, 72 for dk and dv in 240), 47 TFLOP/s of
// the five products that one kernel would need.  4 x 512 x 512, 8 heads of 128: 156 us.
// In 16 bits, where points_attend16_grad.hip does not take the call (f16, or rows that cannot be moved in 16-byte pieces): 2 x 1024 x 1024, 16 heads of 64, 141 us;
// 4 x 2048 x 2048 in bf16 732 us here, 286 there.
#include "points_attend_split.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

// D = rowsum(do o): 16 lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void delta_kernel(const AttendArgs a) {
  const int64_t flat = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const bool here = flat < (int64_t)a.batch * a.kv_heads * a.rows;
  const int64_t f = here ? flat : 0;
  const int bkv = (int)(f / a.rows), b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const T* o = (const T*)a.o.p + row_at(a.o, a, b, kv, f % a.rows);
  const T* g = (const T*)a.go.p + row_at(a.go, a, b, kv, f % a.rows);
  float s = 0.0f;
  for (int d = threadIdx.x % 16 * 4; d < a.head; d += 64) {
    const Four x = load_four(o, d, a.head, true), y = load_four(g, d, a.head, true);
#pragma unroll
    for (int i = 0; i < 4; ++i) s += x.v[i] * y.v[i];
  }
#pragma unroll
  for (int k = 8; k > 0; k >>= 1) s += __shfl_xor(s, k, 64);
  if (here && threadIdx.x % 16 == 0) a.delta[flat] = s;
}

template <int DP>
__device__ __forceinline__ void zero(float16_t (&acc)[DP / 32]) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
}

template <typename T, int DP>
__device__ __forceinline__ void store_fragments(T* row, const float16_t (&acc)[DP / 32], float by, int h, int head) {
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

// lse of a row as the exponent's offset in powers of two; a row without keys takes no part (exp2(s - inf) = 0)
__device__ __forceinline__ float offset_of(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// Above heads of 64 the pieces of a wave's gradients of o lie in LDS: in registers they would be one set too many, and what is asked for
// ahead would be moved to the accumulation registers, and waited for, as soon as it is asked for (4 x 512 x 512, 8 heads of 128: 156 us, else 171; heads of
// 80 the same).  In 16 bits heads of up to 96 alone: two waves a SIMD would spill 28 registers (3 x 2304 x 302, 48 heads of 80, 12 for keys, f16: 687 us, else 721).
template <typename T, int DP, bool FOUR>
__global__ __launch_bounds__(256, DP <= (sizeof(T) == 4 ? 64 : 96) ? 2 : 1) void query_grad_kernel(const AttendArgs a) {
  constexpr int R = kWaveRows, PIECES = kPieces<T>;
  constexpr bool PARKED = DP > 64 && (PIECES == 3 || DP == 96);
  __shared__ __attribute__((aligned(1024))) bf16_t ks[PIECES * R * DP], vs[PIECES * R * DP];
  __shared__ piece8 parked[PARKED ? 4 : 1][PARKED ? PIECES * (DP / 16) : 1][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
  int64_t at = blockIdx.x;
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int bkv = at / a.row_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int tiles = (n + R - 1) / R, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = (int64_t)row_tile * 128 + wave * R + col, flat = (int64_t)bkv * a.rows + r;
  const bool here = r < a.rows, idle = (int64_t)row_tile * 128 + wave * R >= a.rows;
  const float lse = here ? a.lse[flat] : -INFINITY;
  const bool takes_part = here && lse != -INFINITY;
  const float offset = offset_of(lse), delta = takes_part ? a.delta[flat] : 0.0f, unit = a.scale * kLog2e;
  const unsigned rows_at = rows_place<bf16_t, DP>(lane), columns_at = columns_place<bf16_t, DP>(lane);
  RowPieces<DP, PIECES> qf, gf;
  qf.load((const T*)a.q.p + (here ? row_at(a.q, a, b, kv, r) : 0), h, a.head, takes_part);
  gf.load((const T*)a.go.p + (here ? row_at(a.go, a, b, kv, r) : 0), h, a.head, takes_part);
  if constexpr (PARKED)
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) parked[wave][k * (DP / 16) + c][lane] = gf.f[k][c];
  float16_t dq[DP / 32];
  zero<DP>(dq);
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
    float16_t s = split_over_head<DP, PIECES, false>(hide(lds_addr_of(ks) + rows_at), [&](int k, int c) { return qf.f[k][c]; });
    const float16_t dp = split_over_head<DP, PIECES, false>(hide(lds_addr_of(vs) + rows_at), [&](int k, int c) {
      if constexpr (PARKED) return parked[wave][k * (DP / 16) + c][lane];
      else return gf.f[k][c];
    });
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = exp2_(s[i] * unit - offset);
      s[i] = (valid >> product_row(i, 0)) & 1 ? p * (dp[i] - delta) : 0.0f;
    }
    split_over_rows<DP, PIECES, false>(hide(lds_addr_of(ks) + columns_at), s, dq);
  }
  if (!here) return;
  if (a.splits > 1)
    store_fragments<float, DP>(a.part + ((int64_t)split * a.batch * a.kv_heads * a.rows + flat) * a.head, dq, a.scale, h, a.head);
  else
    store_fragments<T, DP>((T*)a.dq + dense_row_at(a, b, kv, r), dq, a.scale, h, a.head);
}

// (as above, with the wave's keys in registers and its values in LDS; in f32 five registers of heads of 128 are spilled)
template <typename T, int DP, bool FOUR>
__global__ __launch_bounds__(256, DP <= (sizeof(T) == 4 ? 32 : 64) ? 2 : 1) void key_grad_kernel(const AttendArgs a) {
  constexpr int R = kWaveRows, PIECES = kPieces<T>;
  constexpr bool PARKED = DP > 64 && PIECES == 3;
  __shared__ __attribute__((aligned(1024))) bf16_t qs[PIECES * R * DP], gs[PIECES * R * DP];
  __shared__ float offsets[R], deltas[R];
  __shared__ piece8 parked[PARKED ? 4 : 1][PARKED ? PIECES * (DP / 16) : 1][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h = lane >> 5;
  int64_t at = blockIdx.x;
  const int split = at % a.splits;
  at /= a.splits;
  const int key_tile = at % a.key_tiles;
  const int bkv = at / a.key_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int key = key_tile * 128 + wave * R + col;
  const bool here = key < a.keys, counts = key_counts(a, b, key, n), idle = key_tile * 128 + wave * R >= n;
  int t0 = 0, t1 = 0;
  if (key_tile * 128 < n) {   // else no key of the block counts: its gradients are zero
    const int tiles = (int)((a.rows + R - 1) / R), per = (tiles + a.splits - 1) / a.splits;
    t0 = split * per;
    t1 = min(tiles, t0 + per);
  }
  const unsigned rows_at = rows_place<bf16_t, DP>(lane), columns_at = columns_place<bf16_t, DP>(lane);
  RowPieces<DP, PIECES> kf, vf;
  kf.load((const T*)a.k.p + (counts ? b * a.k.b + kv * a.k.h + key * a.k.t : 0), h, a.head, counts);
  vf.load((const T*)a.v.p + (counts ? b * a.v.b + kv * a.v.h + key * a.v.t : 0), h, a.head, counts);
  if constexpr (PARKED)
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) parked[wave][k * (DP / 16) + c][lane] = vf.f[k][c];
  const float unit = a.scale * kLog2e;
  float16_t dk[DP / 32], dv[DP / 32];
  zero<DP>(dk);
  zero<DP>(dv);
  RowsAhead<T, DP, 256, FOUR> q_next, g_next;
  typename RowsAhead<T, DP, 256, FOUR>::Words words;
  constexpr int kNone = (int)0xff800000;   // the bits of -inf
  float next_lse = -INFINITY, next_delta = 0.0f;
  const float* lse = a.lse + (int64_t)bkv * a.rows;
  auto fetch = [&](int t) {
    // a row without keys (lse = -inf) counts for nothing: what it holds must not reach the sums
    auto row = [&](int j) { return min((int64_t)t * R + j, a.rows - 1); };
    auto word = [&](int j) { return (int64_t)t * R + j < a.rows ? __builtin_bit_cast(int, lse[(int64_t)t * R + j]) : kNone; };
    words.load(word, threadIdx.x);
    q_next.load([&](int j) { return (const T*)a.q.p + row_at(a.q, a, b, kv, row(j)); }, a.head, threadIdx.x);
    g_next.load([&](int j) { return (const T*)a.go.p + row_at(a.go, a, b, kv, row(j)); }, a.head, threadIdx.x);
    if (threadIdx.x < R) {
      const int64_t r = (int64_t)t * R + threadIdx.x;
      next_lse = r < a.rows ? lse[r] : -INFINITY;
      next_delta = r < a.rows ? a.delta[(int64_t)bkv * a.rows + r] : 0.0f;
    }
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    auto counting = [](int word) { return word != kNone; };
    store_tile<DP, PIECES>(q_next, qs, words, counting, a.head, threadIdx.x);
    store_tile<DP, PIECES>(g_next, gs, words, counting, a.head, threadIdx.x);
    if (threadIdx.x < R) {
      offsets[threadIdx.x] = offset_of(next_lse);
      deltas[threadIdx.x] = next_lse == -INFINITY ? 0.0f : next_delta;
    }
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    if (idle) continue;
    float16_t s = split_over_head<DP, PIECES, false>(hide(lds_addr_of(qs) + rows_at), [&](int k, int c) { return kf.f[k][c]; });
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = exp2_(s[i] * unit - offsets[product_row(i, h)]);   // (of a key that does not count: dropped below)
    split_over_rows<DP, PIECES, false>(hide(lds_addr_of(gs) + columns_at), s, dv);
    const float16_t dp = split_over_head<DP, PIECES, false>(hide(lds_addr_of(gs) + rows_at), [&](int k, int c) {
      if constexpr (PARKED) return parked[wave][k * (DP / 16) + c][lane];
      else return vf.f[k][c];
    });
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= dp[i] - deltas[product_row(i, h)];
    split_over_rows<DP, PIECES, false>(hide(lds_addr_of(qs) + columns_at), s, dk);
  }
  if (!here) return;
  if (!counts) {
    zero<DP>(dk);
    zero<DP>(dv);
  }
  const int64_t dense = ((b * (int64_t)a.keys + key) * a.kv_heads + kv) * a.head;
  if (a.splits > 1) {
    const int64_t all = (int64_t)a.batch * a.keys * a.kv_heads * a.head;
    store_fragments<float, DP>(a.part + split * all + dense, dk, a.scale, h, a.head);
    store_fragments<float, DP>(a.part + (a.splits + split) * all + dense, dv, 1.0f, h, a.head);
  } else {
    store_fragments<T, DP>((T*)a.dk + dense, dk, a.scale, h, a.head);
    store_fragments<T, DP>((T*)a.dv + dense, dv, 1.0f, h, a.head);
  }
}

// dk[e] = sum over splits of part[s][e], in order, and dv[e] of those behind (blockIdx.y)
template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(const float* __restrict__ part, int splits, int64_t n, T* __restrict__ dk, T* __restrict__ dv) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  part += blockIdx.y * splits * n + e;
  float s = 0.0f;
  for (int k = 0; k < splits; k += 4) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < splits ? part[(k + i) * n] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += v[i];
  }
  (blockIdx.y ? dv : dk)[e] = from_f<T>(s);
}
// the same for rows in the order of lse, written in the order of the tensor
template <typename T>
__global__ __launch_bounds__(256) void sum_rows_kernel(const AttendArgs a, T* __restrict__ out) {
  const int64_t all = (int64_t)a.batch * a.kv_heads * a.rows, flat = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (flat >= all) return;
  const int bkv = (int)(flat / a.rows), b = bkv / a.kv_heads;
  T* row = out + dense_row_at(a, b, bkv % a.kv_heads, flat % a.rows);
  for (int d = threadIdx.x & 63; d < a.head; d += 64) {
    float s = 0.0f;
    for (int k = 0; k < a.splits; ++k) s += a.part[(k * all + flat) * a.head + d];
    row[d] = from_f<T>(s);
  }
}

struct GradCut {
  int row_tiles, key_tiles, query_splits, key_splits;
  int64_t delta, part;   // floats of the workspace
};
GradCut grad_cut(int64_t batch, int64_t kv_heads, int64_t rows, int64_t keys, int64_t head, bool by16) {
  GradCut c;
  c.row_tiles = (int)ceil_div(rows, by16 ? 256 : 128);
  c.key_tiles = (int)ceil_div(keys, by16 ? key_grad16_tile(head) : 128);
  // blocks that the chip holds at once; what starting a block, and adding splits up, costs in tiles of 32 rows.  Two tiles are the least for a
  // split: 640 x 40, a head of 80, in f32 take 40 us, with four 49; 55 x 260 in bf16, 16 heads of 128 for 2, 51 and 72.
  const int64_t start = by16 ? 6 : 2, join = by16 ? 12 : 3;
  c.query_splits = split_of(batch * kv_heads * c.row_tiles, ceil_div(keys, kWaveRows), 2, by16 || head > 64 ? 256 : 512, start, join);
  c.key_splits = split_of(batch * kv_heads * c.key_tiles, ceil_div(rows, kWaveRows), 2, head > (by16 ? 64 : 32) ? 256 : 512, start, join);
  c.delta = round_up(batch * kv_heads * rows, 64);
  const int64_t q = c.query_splits > 1 ? c.query_splits * batch * kv_heads * rows * head : 0;
  const int64_t k = c.key_splits > 1 ? 2 * c.key_splits * batch * kv_heads * keys * head : 0;
  c.part = std::max(q, k);
  return c;
}

template <typename T, int DP>
void launch_grad(AttendArgs a, const GradCut& c, bool by16, hipStream_t st) {
  const int64_t heads = (int64_t)a.batch * a.kv_heads;
  const bool four = a.head % 4 == 0;
  if (a.rows > 0) {
    hipLaunchKernelGGL((delta_kernel<T>), dim3((unsigned)ceil_div(heads * a.rows, 16)), dim3(256), 0, st, a);
    a.row_tiles = c.row_tiles;
    a.splits = c.query_splits;
    if (by16) launch_query_grad16(a, st);
    else if (four) hipLaunchKernelGGL((query_grad_kernel<T, DP, true>), dim3((unsigned)(heads * c.row_tiles * a.splits)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((query_grad_kernel<T, DP, false>), dim3((unsigned)(heads * c.row_tiles * a.splits)), dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL((sum_rows_kernel<T>), dim3((unsigned)ceil_div(heads * a.rows, 4)), dim3(256), 0, st, a, (T*)a.dq);
  }
  if (a.keys > 0) {
    a.key_tiles = c.key_tiles;
    a.splits = c.key_splits;
    if (by16) launch_key_grad16(a, st);
    else if (four) hipLaunchKernelGGL((key_grad_kernel<T, DP, true>), dim3((unsigned)(heads * c.key_tiles * a.splits)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((key_grad_kernel<T, DP, false>), dim3((unsigned)(heads * c.key_tiles * a.splits)), dim3(256), 0, st, a);
    if (a.splits > 1) {
      const int64_t n = heads * a.keys * a.head;
      hipLaunchKernelGGL((sum_kernel<T>), dim3((unsigned)ceil_div(n, 256), 2), dim3(256), 0, st, a.part, a.splits, n, (T*)a.dk, (T*)a.dv);
    }
  }
}

}  // namespace
}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_cross_attention_backward_workspace(const nnvhip_attention* d, int64_t* bytes) {
  int64_t forward = 0;
  NNV_TRY(nnvhip_cross_attention_workspace(d, &forward));   // checks the sizes
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  const int64_t heads = d->batch * d->kv_heads;
  if (ceil_div(d->batch * d->heads * d->queries, 16) > 2 * kMostBlocks)   // delta_kernel's blocks, of 256 threads
    NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_cross_attention_backward: too many rows");
  if (heads * ceil_div(d->keys, 256) > kMostBlocks)   // (at least so many blocks, as in the forward pass)
    NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_cross_attention_backward: too many keys");
  *bytes = 0;   // whichever kernels the alignment of the tensors lets take the call
  for (const bool by16 : {false, true}) {
    const GradCut c = grad_cut(d->batch, d->kv_heads, d->queries * (d->heads / d->kv_heads), d->keys, d->head, by16);
    if (heads * c.row_tiles * c.query_splits > kMostBlocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_cross_attention_backward: too many rows");
    if (heads * c.key_tiles * c.key_splits > kMostBlocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_cross_attention_backward: too many keys");
    *bytes = std::max(*bytes, (c.delta + c.part) * (int64_t)sizeof(float));
  }
  return NNVHIP_OK;
}

int nnvhip_cross_attention_backward(nnvhip_ctx* ctx, const nnvhip_attention* d, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  AttendArgs a;
  NNV_TRY(attend_args("nnvhip_cross_attention_backward", d, true, &a));
  int64_t need = 0;
  NNV_TRY(nnvhip_cross_attention_backward_workspace(d, &need));
  if (need > workspace_bytes || (need && !workspace))
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_cross_attention_backward: a workspace of %lld bytes is needed", (long long)need);
  if (a.batch == 0) return NNVHIP_OK;
  const bool by16 = grad16_takes(a, (int)d->type);
  const GradCut c = grad_cut(a.batch, a.kv_heads, a.rows, a.keys, a.head, by16);
  a.delta = static_cast<float*>(workspace);
  a.part = a.delta + c.delta;
  ATTEND_BY_TYPE(d->type, launch_grad, a, c, by16, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
