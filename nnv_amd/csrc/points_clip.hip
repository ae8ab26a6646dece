// The global norm of a list of gradients, and the list scaled to a norm of at most `threshold`:
//
//   n = sqrt(sum over all tensors and elements of g^2),   out = g * (n > threshold ? threshold / n : 1)
//
// Bound by memory: every gradient is read once for the norm and once more for the scaling (the factor is known only when all
// are summed), and written once.  Squares are formed and summed in f64: the bandwidth of f32 gradients asks for some
// 1.3e12 squares a second, a thirtieth of what the f64 pipes give, and neither a large gradient's square nor a sum of a
// billion terms then needs a second thought.  Each block leaves one partial sum, the scaling pass adds them in order: no
// atomics, the same inputs give the same bits.
//
// 60 tensors of up to 2^24 values in bf16 (0.53 GB): 303 us, of which the sums take 115, the scaling 178; 16 of up to 262144 in f32: 23 us, of which the
// kernels take 10 and the host the rest.
//
// The table of tensors travels in the kernels' arguments, kTensors at a time: it needs no memory that would have to outlive
// the call on the caller's stream.
#include "points.h"

#include <algorithm>
#include <memory>
#include <new>

namespace nnvhip {
namespace {

constexpr int kTensors = 96;
constexpr int kThreads = 256;
constexpr int kPacks = 4;                 // 16-byte packs a thread takes of a tile (the 60 tensors: 304 us; two 325, eight 310)
constexpr int64_t kBlocks = 1024;         // blocks of a launch, at most: 16 waves a CU (304 us; 512 blocks 316, 2048 312)

struct ClipTable {
  int64_t tile_end[kTensors];             // tiles of the tensors up to and including this one
  int64_t n[kTensors];
  const void* in[kTensors];
  void* out[kTensors];
  uint8_t type[kTensors];
  int32_t count;
};

inline int64_t tile_values(int type) { return (int64_t)kThreads * kPacks * 16 / type_size(type); }

// the tensor of a tile: the first whose tiles end behind it
__device__ __forceinline__ int tensor_of(const ClipTable& t, int64_t tile) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (t.tile_end[mid] > tile) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double tile_squares(const T* p, int64_t n) {
  constexpr int V = kVec<T>;
  Pack<T> in[kPacks];
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const int64_t c = (int64_t)(j * kThreads + threadIdx.x) * V;
    in[j] = load_pack(p + c, n - c);
  }
  double s = 0;
#pragma unroll
  for (int j = 0; j < kPacks; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double d = (double)to_f(in[j][i]);
      s = fma(d, d, s);
    }
  return s;
}

__device__ __forceinline__ double block_sum(double s) {
  __shared__ double lds[kThreads / 64];
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) s += lds[w];
  return s;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(const ClipTable t, int64_t tiles, double* __restrict__ part) {
  double s = 0;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int k = tensor_of(t, tile);
    const int type = t.type[k];
    const int64_t per = (int64_t)kThreads * kPacks * (type == NNVHIP_TYPE_F32 ? 4 : 8);
    const int64_t at = (tile - (k ? t.tile_end[k - 1] : 0)) * per;
    if (type == NNVHIP_TYPE_F32) s += tile_squares((const float*)t.in[k] + at, t.n[k] - at);
    else if (type == NNVHIP_TYPE_BF16) s += tile_squares((const bf16_t*)t.in[k] + at, t.n[k] - at);
    else s += tile_squares((const f16_t*)t.in[k] + at, t.n[k] - at);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// F: float, or double for a factor that f32 does not hold, or not in full.
template <typename T, typename F>
__device__ __forceinline__ void tile_scale(const T* p, T* out, int64_t n, F f) {
  constexpr int V = kVec<T>;
  Pack<T> in[kPacks];
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const int64_t c = (int64_t)(j * kThreads + threadIdx.x) * V;
    in[j] = load_pack(p + c, n - c);
  }
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const int64_t c = (int64_t)(j * kThreads + threadIdx.x) * V;
    Pack<T> scaled;
#pragma unroll
    for (int i = 0; i < V; ++i) scaled.set(i, from_f<T>((float)(to_f(in[j][i]) * f)));
    store_pack(out + c, scaled, n - c);
  }
}

template <typename F>
__device__ __forceinline__ void scale_tiles(const ClipTable& t, int64_t tiles, F f) {
  for (int64_t back = blockIdx.x; back < tiles; back += gridDim.x) {
    const int64_t tile = tiles - 1 - back;
    const int k = tensor_of(t, tile);
    const int type = t.type[k];
    const int64_t per = (int64_t)kThreads * kPacks * (type == NNVHIP_TYPE_F32 ? 4 : 8);
    const int64_t at = (tile - (k ? t.tile_end[k - 1] : 0)) * per;
    if (f == 1 && t.in[k] == t.out[k]) continue;   // nothing changes in place
    if (type == NNVHIP_TYPE_F32) tile_scale((const float*)t.in[k] + at, (float*)t.out[k] + at, t.n[k] - at, f);
    else if (type == NNVHIP_TYPE_BF16) tile_scale((const bf16_t*)t.in[k] + at, (bf16_t*)t.out[k] + at, t.n[k] - at, f);
    else tile_scale((const f16_t*)t.in[k] + at, (f16_t*)t.out[k] + at, t.n[k] - at, f);
  }
}

// Tiles are taken from the last to the first: what the sums read last is still in the caches.  The norm of finite f32 gradients may be beyond f32: from some
// way below that on the factor and its products are f64.
__global__ __launch_bounds__(kThreads) void clip_kernel(const ClipTable t, int64_t tiles, const double* __restrict__ part, int parts,
                                                        double threshold, float* __restrict__ norm, int scale) {
  double s = 0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
  s = block_sum(s);
  const double whole = sqrt(s);
  const float n = (float)whole, limit = (float)threshold;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  if (!scale) return;
  const float f = n > limit ? limit / n : 1.0f;
  if (whole > 1e30 || f < 1e-30f) scale_tiles(t, tiles, whole > threshold ? threshold / whole : 1.0);
  else scale_tiles(t, tiles, f);
}

// Whether a tensor that is written to overlaps another one, or the gradient of another one, or its own other than exactly: blocks would read what others
// wrote.  1: it does, 0: none does, -1: no memory to find out.
int outputs_overlap(int64_t count, const int32_t* type, const int64_t* n, const void* const* in, void* const* out) {
  struct Span {
    uintptr_t begin, end;
    int64_t k;
  };
  const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[count]);
  if (!spans) return -1;
  int64_t used = 0;
  for (int64_t k = 0; k < count; ++k)
    if (n[k] > 0) spans[used++] = {(uintptr_t)out[k], (uintptr_t)out[k] + (uintptr_t)n[k] * type_size(type[k]), k};
  Span* const end = spans.get() + used;
  std::sort(spans.get(), end, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (int64_t i = 1; i < used; ++i)
    if (spans[i].begin < spans[i - 1].end) return 1;
  for (int64_t k = 0; k < count; ++k) {
    if (n[k] == 0) continue;
    const uintptr_t from = (uintptr_t)in[k], to = from + (uintptr_t)n[k] * type_size(type[k]);
    // (the spans are apart, so that their ends are in order, too)
    for (const Span* s = std::upper_bound(spans.get(), end, from, [](uintptr_t x, const Span& b) { return x < b.end; }); s != end && s->begin < to; ++s)
      if (s->k != k || s->begin != from) return 1;
  }
  return 0;
}

}  // namespace
}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_clip_gradients_workspace(int64_t count, int64_t* bytes) {
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  if (count < 0) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_clip_gradients: a negative number of tensors");
  *bytes = std::max<int64_t>(1, ceil_div(count, kTensors)) * kBlocks * (int64_t)sizeof(double);
  return NNVHIP_OK;
}

int nnvhip_clip_gradients(nnvhip_ctx* ctx, int64_t count, const int32_t* type, const int64_t* n, const void* const* in,
                          void* const* out, double threshold, float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  int64_t need = 0;
  NNV_TRY(nnvhip_clip_gradients_workspace(count, &need));
  if (!workspace || workspace_bytes < need)
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_clip_gradients: a workspace of %lld bytes is needed", (long long)need);
  if (count > 0 && (!type || !n || !in)) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_clip_gradients: null pointer");
  if (!(threshold > 0)) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_clip_gradients: the threshold must be positive");
  for (int64_t k = 0; k < count; ++k) {
    if (!known_type(type[k])) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_clip_gradients: tensor %lld: the values are f32, bf16 or f16", (long long)k);
    if (n[k] < 0) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_clip_gradients: tensor %lld: a negative size", (long long)k);
    if (n[k] > 0 && (!in[k] || (out && !out[k]))) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_clip_gradients: tensor %lld: null pointer", (long long)k);
  }
  const int overlap = out && count > 0 ? outputs_overlap(count, type, n, in, out) : 0;
  if (overlap > 0) NNV_FAIL(NNVHIP_ERR_SHAPE, "nnvhip_clip_gradients: a tensor to write to overlaps another one, or another gradient");
  if (overlap < 0) NNV_FAIL(NNVHIP_ERR_OOM, "nnvhip_clip_gradients: no host memory for %lld tensors", (long long)count);
  hipStream_t st = (hipStream_t)stream;
  double* part = static_cast<double*>(workspace);
  int64_t parts = 0;
  // Both passes walk the same tables; the second from the last table to the first.
  auto fill = [&](int64_t first, ClipTable& t) {
    t.count = (int32_t)std::min<int64_t>(kTensors, count - first);
    int64_t tiles = 0;
    for (int k = 0; k < t.count; ++k) {
      t.type[k] = (uint8_t)type[first + k];
      t.n[k] = n[first + k];
      t.in[k] = in[first + k];
      t.out[k] = out ? out[first + k] : nullptr;
      tiles += ceil_div(t.n[k], tile_values(t.type[k]));
      t.tile_end[k] = tiles;
    }
    return tiles;
  };
  ClipTable t{};
  for (int64_t first = 0; first < count; first += kTensors) {
    const int64_t tiles = fill(first, t), blocks = std::min(tiles, kBlocks);
    if (blocks == 0) continue;
    hipLaunchKernelGGL(squares_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, t, tiles, part + parts);
    parts += blocks;
  }
  bool told = false;
  for (int64_t first = count > 0 ? (count - 1) / kTensors * kTensors : -1; first >= 0 && out; first -= kTensors) {
    const int64_t tiles = fill(first, t), blocks = std::min(tiles, kBlocks);
    if (blocks == 0) continue;
    hipLaunchKernelGGL(clip_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, t, tiles, part, (int)parts, threshold,
                       told ? nullptr : norm, 1);
    told = true;
  }
  if (!told && norm)   // nothing to scale: the norm alone
    hipLaunchKernelGGL(clip_kernel, dim3(1), dim3(kThreads), 0, st, t, (int64_t)0, part, (int)parts, threshold, norm, 0);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
