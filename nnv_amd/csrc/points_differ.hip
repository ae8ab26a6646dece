// Differential attention of points, forward: the kernel for every type, head size and alignment, with f32 products, and the joining of splits.
//
// S_m = scale q_m k_m^T, o = softmax(S_0) v - w softmax(S_1) v: one pass over keys and values with the running maximum and sum of each map's softmax.  Bound by the f32
// matrix instructions (4 x 1024 x 1024, 16 heads of 64: 469 us, 110 TFLOP/s of 154, matrix units busy 74 %).
#include "points_differ16.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

constexpr int kRows = 64;   // of a block

// A wave takes 16 rows of one map; eight waves share the tiles of keys and values: four groups of rows, two maps each.  The second map's result meets the
// first one's in LDS at the end.  Where there are too few blocks for the chip, the keys are split over `splits` blocks, and join_kernel
// puts their results together.
template <typename T, int CH, bool FOUR>
__global__ __launch_bounds__(512, 2) void differ_kernel(const DifferArgs a) {
  constexpr int R = 32, W = 32 * CH, LD = F32Tile<CH>::LD;
  // the tile; at the end, the second map's result: [group of rows][16 values][lane] x 4
  __shared__ __attribute__((aligned(16))) float tile[F32Tile<CH>::FLOATS > 4 * 16 * W ? F32Tile<CH>::FLOATS : 4 * 16 * W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, q4 = lane >> 4;
  const int map = wave & 1, part_of = wave >> 1;
  const BlockPlace at = block_place(a, blockIdx.x, (uint32_t)a.row_tiles * a.splits);
  const int b = at.b, kv = at.kv, bkv = b * a.kv_heads + kv, split = (uint32_t)at.x % (uint32_t)a.splits, row_tile = row_tile_of(a, (uint32_t)at.x / (uint32_t)a.splits);
  const int n = keys_that_count(a, b);
  const int64_t first = (int64_t)row_tile * kRows, last = min(first + kRows, a.rows) - 1;
  const int tiles = (most_seen(a, first, last, n) + R - 1) / R, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int64_t r = first + part_of * 16 + col;
  const bool here = r < a.rows, idle = first + part_of * 16 >= a.rows;
  const int seen = here ? seen_by(a, r, n) : 0;

  float qf[CH][4];
  f32_operands<T, CH>((const T*)a.q.p + (here ? map_row_at(a.q, a, b, kv, r, map) : 0), q4, a.head, here, qf);
  const float unit = a.scale * kLog2e;
  float4_t acc[2 * CH];
  f32_zero(acc);
  float m = -INFINITY, total = 0.0f;
  const T* kp = (const T*)a.k.p + b * a.k.b + 2 * kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  TripleAhead<T, CH, 512, FOUR> next;
  int counts = 0;
  auto fetch = [&](int t) {
    next.load([&](int j, int which) { return kp + min(t * R + j, n - 1) * a.k.t + which * a.k.h; }, [&](int j) { return vp + min(t * R + j, n - 1) * a.v.t; },
              a.head, threadIdx.x);
    counts = key_word(a, b, t * R + (lane & 31), n);
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    const uint32_t valid = (uint32_t)__ballot(counts != 0);
    next.store(tile, valid, a.head, threadIdx.x);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    if (idle) continue;
    const uint32_t mine = valid & first_bits(seen - t * R);
    float4_t s[2];
    f32_over_head<CH, CH>(tile + col * LD + 4 * q4 + map * 16 * CH, qf, s);
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[k][i] = f32_bit(mine, k, i, q4) ? s[k][i] * unit : -INFINITY;
        top = fmaxf(top, s[k][i]);
      }
    top = fmaxf(m, quarters_max(top));
    const float base = top == -INFINITY ? 0.0f : top;   // no key of this row yet
    const float fade = exp2_(m - base);
    m = top;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[k][i] = exp2_(s[k][i] - base);
        sum += s[k][i];
      }
    total = total * fade + sum;
    if (__any(fade != 1.0f))
#pragma unroll
      for (int d = 0; d < 2 * CH; ++d) acc[d] *= fade;
    f32_over_rows<CH, 2 * CH>(tile + 4 * q4 * LD + col + 32 * CH, s, acc);
  }
  total = quarters_sum(total);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total, lse = total == 0.0f ? -INFINITY : (m + log2f(total)) * kLn2;
  if (a.splits > 1) {
    if (!here) return;
    const int64_t own = split * own_rows(a) + own_row(a, bkv, r, map);
    if (q4 == 0) a.part_lse[own] = lse;
    f32_store<FOUR>(a.part + own * 2 * a.head, acc, inv, q4, 2 * a.head);
    return;
  }
  if (here && q4 == 0) a.lse[lse_at(a, b, kv, r, map)] = lse;
  __syncthreads();
  float* found = tile + part_of * 16 * W + 4 * lane;
  if (map) {
#pragma unroll
    for (int d = 0; d < 2 * CH; ++d) {
      const float f[4] = {acc[d][0] * inv, acc[d][1] * inv, acc[d][2] * inv, acc[d][3] * inv};
      __builtin_memcpy(found + 256 * d, f, 16);
    }
    if (a.second && here) f32_store<FOUR>((T*)a.second + wide_row_at(a, b, kv, r), acc, inv, q4, 2 * a.head);
  }
  __syncthreads();
  if (map || !here) return;
  const float w = weight_of<T>(a, head_of_row(a, kv, r));
#pragma unroll
  for (int d = 0; d < 2 * CH; ++d) {
    float f[4];
    __builtin_memcpy(f, found + 256 * d, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[d][i] = rounded(acc[d][i] * inv) - w * f[i];   // (of equal maps and a weight of one nothing is left)
  }
  f32_store<FOUR>((T*)a.out + wide_row_at(a, b, kv, r), acc, 1.0f, q4, 2 * a.head);
}

// The parts of a row's two maps, joined: 64 lanes (four values each, of up to 256) a row, SLICES of which take the splits in turn.
template <typename T, int SLICES>
__global__ __launch_bounds__(256) void differ_join_kernel(const DifferArgs a) {
  __shared__ float4_t found[4][64][2];
  const int slot = threadIdx.x >> 6, lane = threadIdx.x & 63, slice = SLICES > 1 ? slot : 0;
  const int64_t all = (int64_t)a.batch * a.kv_heads * a.rows, flat = SLICES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + slot;
  const bool here = flat < all;
  const uint32_t set = here ? (uint32_t)flat / (uint32_t)a.rows : 0;   // (a call that is split has fewer than 2^23 rows)
  const int64_t bkv = set, r = here ? flat - (int64_t)set * a.rows : 0;
  const int b = set / (uint32_t)a.kv_heads, kv = set - b * a.kv_heads, d = 4 * lane;
  const int64_t rows = own_rows(a);
  float4_t f[2];
  float lse[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int64_t own = own_row(a, bkv, r, m);
    f[m] = float4_t{0, 0, 0, 0};
    // every lane the parts' weights of some splits, then all of them
    float top = -INFINITY;
    for (int k = lane; k < a.splits; k += 64) top = fmaxf(top, a.part_lse[k * rows + own]);
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int k = lane; k < a.splits; k += 64) sum += exp2_((a.part_lse[k * rows + own] - base) * kLog2e);
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k, 64);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    lse[m] = sum == 0.0f ? -INFINITY : base + log2f(sum) * kLn2;
    if (d < 2 * a.head)
      for (int k = slice; k < a.splits; k += SLICES) {
        const float w = exp2_((a.part_lse[k * rows + own] - base) * kLog2e) * inv;
        const Four x = load_four(a.part + (k * rows + own) * 2 * a.head, d, 2 * a.head, true);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[m][i] += w == 0.0f ? 0.0f : w * x.v[i];   // (a part without keys holds zeros; one too small to count may be infinite)
      }
  }
  if constexpr (SLICES > 1) {
#pragma unroll
    for (int m = 0; m < 2; ++m) found[slot][lane][m] = f[m];
    __syncthreads();
    if (slot) return;
#pragma unroll
    for (int k = 1; k < SLICES; ++k)
#pragma unroll
      for (int m = 0; m < 2; ++m) f[m] += found[k][lane][m];
  }
  if (!here) return;
  if (lane < 2) a.lse[lse_at(a, b, kv, r, lane)] = lane ? lse[1] : lse[0];
  if (d >= 2 * a.head) return;
  const float w = weight_of<T>(a, head_of_row(a, kv, r));
  float o[4], second[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    second[i] = f[1][i];
    o[i] = rounded(f[0][i]) - w * f[1][i];
  }
  store_four((T*)a.out + wide_row_at(a, b, kv, r), d, 2 * a.head, o);
  if (a.second) store_four((T*)a.second + wide_row_at(a, b, kv, r), d, 2 * a.head, second);
}

// How a forward call is cut: few rows for each head's keys (single tokens, 16 bits) or tiles of many, and over how many blocks the keys are split (see
// split_of).
struct Cut {
  bool few;
  int row_tiles, splits;
};
Cut cut_of(int64_t batch, int64_t kv_heads, int64_t rows, int64_t keys, int64_t head, bool by16) {
  Cut c;
  c.few = by16 && rows <= kDifferFewRows;
  c.row_tiles = (int)ceil_div(rows, c.few ? kDifferFewRows : by16 ? kDiffer16Rows : kRows);
  const int64_t start = c.few ? 16 : by16 ? 6 : 2, join = c.few ? 16 : by16 ? 12 : 3;
  c.splits = split_of(batch * kv_heads * c.row_tiles, ceil_div(keys, 32), c.few ? 8 : by16 ? 4 : 2, by16 ? 256 : 512, start, join);
  return c;
}

template <typename T, int CH>
void launch_differ(const DifferArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits));
  if (a.head % 4 == 0) hipLaunchKernelGGL((differ_kernel<T, CH, true>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((differ_kernel<T, CH, false>), grid, dim3(512), 0, st, a);
}
template <typename T, int>
void launch_join(const DifferArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows;
  if (a.splits > 8 || (a.splits > 2 && rows <= 4096)) hipLaunchKernelGGL((differ_join_kernel<T, 4>), dim3((unsigned)rows), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((differ_join_kernel<T, 1>), dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, st, a);
}

// The sizes have to fit the kernels' indexes (see check_sizes in points_attend.hip), and a launch has fewer than 2^32 threads.
int check_sizes(const char* what, const nnvhip_differ_args* d) {
  if (!d) NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  if (d->type < 0 || d->type > 2 || !known_type((int)d->type) || !(d->weight_type == d->type || d->weight_type == NNVHIP_TYPE_F32))
    NNV_FAIL(NNVHIP_ERR_ARG, "%s: the values are f32, bf16 or f16, the weights of the same type or f32", what);
  if (d->batch < 0 || d->queries < 0 || d->keys < 0) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: negative size", what);
  if (d->head < 1 || d->head > 128) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: heads of 1 to 128 values are supported", what);
  if (d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads)
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: the number of heads must be a multiple of the number of key/value heads", what);
  const int64_t most = (int64_t(1) << 31) - 256, group = d->heads / d->kv_heads, blocks = kMostBlocks / 2;   // of up to 1024 threads, in two maps
  if (d->batch > 65535 || d->heads > 32767 || d->keys > most || d->queries > most / group) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  if (d->batch * d->kv_heads * ceil_div(d->queries * group, kRows) > blocks) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  for (const bool by16 : {false, true}) {
    const Cut c = cut_of(d->batch, d->kv_heads, d->queries * group, d->keys, d->head, by16);
    if (d->batch * d->kv_heads * c.row_tiles * c.splits > blocks || (c.splits > 1 && d->batch * d->heads * d->queries >= (int64_t(1) << 23)))
      NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  }
  return NNVHIP_OK;
}

}  // namespace

int differ_args(const char* what, const nnvhip_differ_args* d, bool backward, DifferArgs* a) {
  NNV_TRY(check_sizes(what, d));
  if (!(std::fabs(d->scale) <= FLT_MAX)) NNV_FAIL(NNVHIP_ERR_ARG, "%s: the scale must be a finite number of f32", what);
  auto view = [](const void* p, const int64_t (&s)[3]) { return TokenView{p, s[0], s[1], s[2]}; };
  *a = DifferArgs{};
  a->q = view(d->q, d->q_stride);
  a->k = view(d->k, d->k_stride);
  a->v = view(d->v, d->v_stride);
  a->go = view(d->go, d->go_stride);
  a->out = d->o;
  a->second = d->second;
  a->dq = d->dq;
  a->dk = d->dk;
  a->dv = d->dv;
  a->weights = d->weights;
  a->wide_weights = d->weight_type == NNVHIP_TYPE_F32;
  a->dweights = d->dweights;
  a->causal = d->causal != 0;
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
  if ((!no_rows && (!d->q || !d->o || !d->lse || !d->weights)) || (!no_rows && !no_keys && (!d->k || !d->v)) ||
      (backward && ((!no_rows && (!d->go || !d->dq || !d->second)) || (!no_keys && (!d->dk || !d->dv)) || !d->dweights)))
    NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  return NNVHIP_OK;
}

}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_differential_attention_workspace(const nnvhip_differ_args* d, int64_t* bytes) {
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  NNV_TRY(check_sizes("nnvhip_differential_attention_workspace", d));
  int splits = 1;   // whichever kernels the alignment of the tensors lets take the call
  for (const bool by16 : {false, true})
    splits = std::max(splits, cut_of(d->batch, d->kv_heads, d->queries * (d->heads / d->kv_heads), d->keys, d->head, by16).splits);
  *bytes = splits > 1 ? (int64_t)splits * d->batch * d->heads * 2 * d->queries * (2 * d->head + 1) * (int64_t)sizeof(float) : 0;
  return NNVHIP_OK;
}

int nnvhip_differential_attention(nnvhip_ctx* ctx, const nnvhip_differ_args* d, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  DifferArgs a;
  NNV_TRY(differ_args("nnvhip_differential_attention", d, false, &a));
  int64_t need = 0;
  NNV_TRY(nnvhip_differential_attention_workspace(d, &need));
  if (need > workspace_bytes || (need && !workspace))
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_differential_attention: a workspace of %lld bytes is needed", (long long)need);
  if (a.batch == 0 || a.rows == 0) return NNVHIP_OK;
  const bool by16 = differ16_takes(a, (int)d->type);
  const Cut c = cut_of(a.batch, a.kv_heads, a.rows, a.keys, a.head, by16);
  a.row_tiles = c.row_tiles;
  a.splits = c.splits;
  a.part = static_cast<float*>(workspace);
  a.part_lse = c.splits > 1 ? a.part + (int64_t)c.splits * a.batch * a.kv_heads * a.rows * 2 * 2 * a.head : nullptr;
  if (by16) launch_differ16(a, (int)d->type, c.few, (hipStream_t)stream);
  else DIFFER_BY_TYPE(d->type, launch_differ, a, (hipStream_t)stream);
  if (c.splits > 1) DIFFER_BY_TYPE(d->type, launch_join, a, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
