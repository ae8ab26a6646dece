// Rotary positions with several axes (rows and columns of an image, time as well in a video).
//
//   pair i of a head's values (u, w) is turned by t = position[axis(i)] * frequency(i):
//   u' = u cos t - w sin t,  w' = u sin t + w cos t;  the other way round (the gradient): by -t
//
// Bound by memory: each value is read and written once.  A block takes the heads of a few tokens and forms the tokens' cosines and
// sines once, in LDS.  Angles are counted in turns and in f64: position * (frequency / 2 pi), of which the whole turns are dropped, so
// that far positions lose nothing; what is left goes through sincospif, rounded to f32, and what that rounding leaves turns the result by as much.  (2 x 19200 tokens of 32 heads of 128 in bf16: 122 us, 5.15 TB/s; 16 tokens: 4.3 us,
// of which the launch is most; 3 x 1577 tokens of 24 heads of 80 in f32: 17 us among other calls, 4.2 TB/s.)
#include "points.h"

#include <algorithm>

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

constexpr int kThreads = 256;
constexpr int kPairs = NNVHIP_ROTATE_PAIRS;
constexpr int kTensors = NNVHIP_ROTATE_TENSORS;
constexpr int kEntries = 1024;   // cosines of a block, at most

struct RotateArgs {
  double turns[kPairs];        // of a position's unit
  uint8_t axis[kPairs];
  const void* in[kTensors];
  void* out[kTensors];         // dense
  int64_t b[kTensors], t[kTensors], h[kTensors];   // strides of in
  int heads[kTensors], first[kTensors + 1];        // first: packs of a token ahead of this tensor's
  const void* positions;
  int64_t pos_b, pos_t, pos_a;
  int64_t tokens, all;         // of a sequence; of all sequences
  int tensors, pairs, head, packs;   // packs: of a head
  int per_block, slices;       // tokens of a block; blocks that share a token's packs
  int pos_type, interleaved;
  float sign;
};

__device__ __forceinline__ double position(const RotateArgs& a, int64_t token, int axis) {
  const int64_t n = token / a.tokens, at = n * a.pos_b + (token - n * a.tokens) * a.pos_t + axis * a.pos_a;
  if (a.pos_type == NNVHIP_POSITION_I32) return (double)((const int32_t*)a.positions)[at];
  if (a.pos_type == NNVHIP_POSITION_I64) return (double)((const int64_t*)a.positions)[at];
  return (double)((const float*)a.positions)[at];
}

// A head's packs: of the halves form, ceil(pairs / V) of pairs (two packs of memory each) and then those of what is not turned; of the
// interleaved form, ceil(head / V) as they lie.
template <typename T>
__global__ __launch_bounds__(kThreads) void rotate_kernel(const RotateArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float cosines[kEntries], sines[kEntries];
  const int64_t token0 = blockIdx.x / a.slices * (int64_t)a.per_block;
  const int here = (int)min((int64_t)a.per_block, a.all - token0), slice = blockIdx.x % a.slices;
  for (int e = threadIdx.x; e < here * a.pairs; e += kThreads) {
    const int k = e / a.pairs, i = e - k * a.pairs;
    const double turns = position(a, token0 + k, a.axis[i]) * a.turns[i], left = 2.0 * (turns - rint(turns));
    const float half = (float)left, rest = (float)(left - (double)half) * 3.14159265f;
    float s, c;
    sincospif(half, &s, &c);
    cosines[e] = c - s * rest;
    sines[e] = (s + c * rest) * a.sign;
  }
  __syncthreads();
  const int total = a.first[a.tensors], work = here * total;
  for (int e = slice * kThreads + threadIdx.x; e < work; e += a.slices * kThreads) {
    const int k = e / total;
    int at = e - k * total, which = 0;
#pragma unroll 1
    while (at >= a.first[which + 1]) ++which;
    at -= a.first[which];
    const int head = at / a.packs, pack = at - head * a.packs;
    const int64_t token = token0 + k, n = token / a.tokens;
    const T* x = (const T*)a.in[which] + n * a.b[which] + (token - n * a.tokens) * a.t[which] + head * a.h[which];
    T* y = (T*)a.out[which] + (token * a.heads[which] + head) * a.head;
    const float *cs = cosines + k * a.pairs, *sn = sines + k * a.pairs;
    if (a.interleaved) {
      const int d = pack * V;
      Pack<T> p = load_pack(x + d, a.head - d), r;
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const int pair = d / 2 + i / 2;
        const bool turned = pair < a.pairs;
        const float c = turned ? cs[pair] : 1.0f, s = turned ? sn[pair] : 0.0f, u = to_f(p[i]), w = to_f(p[i + 1]);
        r.set(i, turned ? from_f<T>(u * c - w * s) : p[i]);
        r.set(i + 1, turned ? from_f<T>(u * s + w * c) : p[i + 1]);
      }
      store_pack(y + d, r, a.head - d);
    } else {
      const int turned = (a.pairs + V - 1) / V;
      if (pack < turned) {
        const int d = pack * V, left = a.pairs - d;
        const Pack<T> p = load_pack(x + d, left), q = load_pack(x + a.pairs + d, left);
        Pack<T> r, z;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float c = cs[min(d + i, a.pairs - 1)], s = sn[min(d + i, a.pairs - 1)], u = to_f(p[i]), w = to_f(q[i]);
          r.set(i, from_f<T>(u * c - w * s));
          z.set(i, from_f<T>(u * s + w * c));
        }
        store_pack(y + d, r, left);
        store_pack(y + a.pairs + d, z, left);
      } else {
        const int d = 2 * a.pairs + (pack - turned) * V;
        store_pack(y + d, load_pack(x + d, a.head - d), a.head - d);
      }
    }
  }
}

}  // namespace
}  // namespace nnvhip

using namespace nnvhip;

extern "C" int nnvhip_rotate_positions(nnvhip_ctx* ctx, const nnvhip_rotate_args* d, void* stream) {
  ENTER_POINT_CALL(ctx);
  const char* const what = "nnvhip_rotate_positions";
  if (!d) NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  if (d->type < 0 || d->type > 2 || !known_type((int)d->type)) NNV_FAIL(NNVHIP_ERR_ARG, "%s: the values are f32, bf16 or f16", what);
  if (d->position_type < NNVHIP_POSITION_I32 || d->position_type > NNVHIP_POSITION_F32)
    NNV_FAIL(NNVHIP_ERR_ARG, "%s: positions are i32, i64 or f32", what);
  if (d->tensors < 0 || d->tensors > kTensors) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: at most %d tensors", what, kTensors);
  if (d->pairs < 1 || d->pairs > kPairs || d->axes < 1 || d->axes > 255 || d->head < 2 * d->pairs || d->head >= (1 << 20))
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: 1 to %d pairs are expected, and heads that hold them", what, kPairs);
  if (d->batch < 0 || d->tokens < 0 || d->batch >= (int64_t(1) << 31) || d->tokens >= (int64_t(1) << 31))
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many tokens", what);
  RotateArgs a{};
  const int64_t v = 16 / type_size((int)d->type);
  a.packs = (int)(d->interleaved ? ceil_div(d->head, v) : ceil_div(d->pairs, v) + ceil_div(d->head - 2 * d->pairs, v));
  for (int64_t k = 0; k < d->tensors; ++k) {
    if (d->heads[k] < 0 || d->heads[k] > 65535 || a.first[k] + d->heads[k] * a.packs >= (int64_t(1) << 24)) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many heads", what);
    a.heads[k] = (int)d->heads[k];
    a.first[k + 1] = a.first[k] + (int)(d->heads[k] * a.packs);
    a.in[k] = d->in[k];
    a.out[k] = d->out[k];
    a.b[k] = d->in_stride[k][0];
    a.t[k] = d->in_stride[k][1];
    a.h[k] = d->in_stride[k][2];
  }
  a.all = d->batch * d->tokens;
  const int64_t total = a.first[d->tensors];
  if (a.all == 0 || total == 0) return NNVHIP_OK;
  if (!d->positions || !d->frequency || !d->axis) NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  for (int64_t k = 0; k < d->tensors; ++k)
    if (a.heads[k] > 0 && (!a.in[k] || !a.out[k])) NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  for (int64_t i = 0; i < d->pairs; ++i) {
    if (d->axis[i] >= d->axes) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: pair %lld: there is no axis %d", what, (long long)i, (int)d->axis[i]);
    a.turns[i] = d->frequency[i] * 0.15915494309189535;   // 1 / (2 pi)
    a.axis[i] = d->axis[i];
  }
  a.positions = d->positions;
  a.pos_b = d->position_stride[0];
  a.pos_t = d->position_stride[1];
  a.pos_a = d->position_stride[2];
  a.tokens = d->tokens;
  a.tensors = (int)d->tensors;
  a.pairs = (int)d->pairs;
  a.head = (int)d->head;
  a.pos_type = (int)d->position_type;
  a.interleaved = d->interleaved != 0;
  a.sign = d->inverse ? -1.0f : 1.0f;
  // Four packs a thread; tokens that need fewer share a block as long as there are blocks for every CU, those that need more share out their packs.
  a.per_block = (int)std::max<int64_t>(1, std::min({4 * kThreads / std::max<int64_t>(1, total), kEntries / d->pairs, ceil_div(a.all, 1024)}));
  a.slices = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(total * a.per_block, 4 * kThreads), 256));
  if (a.all < 1024) a.slices = (int)std::max<int64_t>(a.slices, std::min(ceil_div(total * a.per_block, kThreads), ceil_div(1024, a.all)));
  const int64_t blocks = ceil_div(a.all, a.per_block) * a.slices;
  if (blocks >= (int64_t(1) << 23)) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many tokens", what);
  const hipStream_t st = (hipStream_t)stream;
  if (d->type == NNVHIP_TYPE_F32) hipLaunchKernelGGL((rotate_kernel<float>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
  else if (d->type == NNVHIP_TYPE_BF16) hipLaunchKernelGGL((rotate_kernel<bf16_t>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((rotate_kernel<f16_t>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}
