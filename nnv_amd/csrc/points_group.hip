// Group normalization of points that are images or videos, channels last, with an activation; forward and backward.
//
//   per sequence n and group g of E channels, over all places p:  mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps)
//   xh = (x - mu) r, z = xh w + b, y = act(z);  act: z, max(z, 0) or z / (1 + exp(-z))
//   h = dy act'(z);  dx = r (h w - mean(h w) - xh mean(h w xh));  dw = sum over n, p of h xh;  db = sum over n, p of h
//
// Both directions are bound by memory: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx.  Where all places of a
// sequence's group (or of a few, next to one another) fit a block's registers, a block takes them, and everything is read once (the resident
// kernels below).  Else each direction is two launches: one leaves sums of parts of the places, the other adds them (in order: no
// atomics, the same inputs give the same bits) and reads again what the caches may still hold.
//
// There a block takes a part of the places of a chunk of channels: whole groups, or a part of a wide one.  Its threads are (pack of
// 16 bytes of channels) x (places): rows are read as they lie in memory, whatever the groups are.  The sums are f64, which the memory's
// rate asks some 1e13 operations a second of, a third of what the f64 pipes give, and they are of x - c and (x - c)^2, c the group's first value: a mean far from zero costs the variance
// nothing, for the variance is no less than a share of (c - mean)^2, and that of equal values is zero.
//
// 16 x 64 x 64 x 320 in bf16: 26 us forward (3.2 TB/s: a block of two groups of 10 channels reads all it has before it writes, and one fits a CU), 54 backward (24 + 27 us a kernel: x and dy are read
// twice, the second time partly from the caches); 5 x 53 x 79 x 96 in f32 backward 17; 4 x 8 x 8 x 256 forward 5.8 us, a launch and one latency of memory.
#include "points.h"

#include <algorithm>

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

constexpr int kThreads = 512;
constexpr int kWide = 1024;   // channels of a chunk, at most
constexpr int kAhead = 4;     // places that a thread has on the way

enum Activation { kNone = 0, kRelu = 1, kSilu = 2 };

struct GroupArgs {
  const void *x, *dy;          // places of `channels` dense values
  int64_t x_b, x_p, dy_b, dy_p;
  void* out;                   // y or dx, dense
  const void *scale, *offset;  // or null
  void *dscale, *doffset;      // or null
  float *mean, *rstd;          // batch x groups
  double* part;                // [batch][parts][groups][2]
  float* columns;              // [batch][splits][channels][2]
  int64_t places, per;         // per: places of a split
  int batch, channels, groups, each;
  int width, chunks, per_group;   // channels of a chunk; chunks of all channels; of a group, where it is wider than a chunk
  int splits, wide_params;        // wide_params: scale and offset are f32
  int resident, threads;          // packs of a thread of the resident form (0: the other one), and its threads
  double eps;
};

struct Chunk {
  int n, split, sub;       // sequence, split of the places, part of a wide group
  int first, size;         // channels
  int group, groups;       // the groups it holds, or is of
};
__device__ __forceinline__ Chunk chunk_of(const GroupArgs& a, int64_t id) {
  Chunk c;
  const int k = (int)(id % a.chunks);
  id /= a.chunks;
  c.split = (int)(id % a.splits);
  c.n = (int)(id / a.splits);
  if (a.per_group > 1) {
    c.group = k / a.per_group;
    c.sub = k % a.per_group;
    c.groups = 1;
    c.first = c.group * a.each + c.sub * a.width;
    c.size = min(a.width, a.each - c.sub * a.width);
  } else {
    c.sub = 0;
    c.first = k * a.width;
    c.size = min(a.width, a.channels - c.first);
    c.group = c.first / a.each;
    c.groups = c.size / a.each;
  }
  return c;
}

template <typename T>
__device__ __forceinline__ float param(const GroupArgs& a, const void* p, int c, float none) {
  if (p == nullptr) return none;
  return a.wide_params ? ((const float*)p)[c] : to_f(((const T*)p)[c]);
}
template <typename T>
__device__ __forceinline__ void set_param(const GroupArgs& a, void* p, int c, float x) {
  if (a.wide_params) ((float*)p)[c] = x;
  else ((T*)p)[c] = from_f<T>(x);
}

// Sums of two values an element over the members of each of `count` groups of a block: value(j, e, v) gives member e < members of group j;
// whoever holds the sums calls found(j, v).  Lanes that share a group: as many as there are for each.
template <class Value, class Found>
__device__ __forceinline__ void sum_groups(int count, int members, Value value, Found found) {
  int lanes = 64;
  while (lanes > 1 && lanes * count > kThreads) lanes >>= 1;
  const int at = threadIdx.x % lanes;
  for (int base = 0; base < count; base += kThreads / lanes) {
    const int j = base + threadIdx.x / lanes;
    double v[2] = {0, 0};
    if (j < count)
      for (int e = at; e < members; e += lanes) {
        double one[2];
        value(j, e, one);
        v[0] += one[0];
        v[1] += one[1];
      }
    for (int k = lanes >> 1; k > 0; k >>= 1) {
      v[0] += __shfl_xor(v[0], k, 64);
      v[1] += __shfl_xor(v[1], k, 64);
    }
    if (j < count && at == 0) found(j, v);
  }
}

// body(place, packs): the packs of up to kAhead places at a time that a thread takes of a split, N tensors at once.  What is behind the
// chunk is zero.
template <typename T, int N, class Body>
__device__ __forceinline__ void over_places(const T* const (&at)[N], const int64_t (&stride)[N], int64_t p0, int64_t p1, int ty, int rows, int left,
                                            Body body) {
  int64_t p = p0 + ty;
  for (; p + (kAhead - 1) * rows < p1; p += kAhead * rows) {
    Pack<T> in[kAhead][N];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) in[k][i] = load_pack(at[i] + (p + k * rows) * stride[i], left);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) body(p + k * rows, in[k]);
  }
  for (; p < p1; p += rows) {
    Pack<T> in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) in[i] = load_pack(at[i] + p * stride[i], left);
    body(p, in);
  }
}

// what a group's values are counted from: its first one, or zero where that is not finite
template <typename T>
__device__ __forceinline__ float origin_of(const GroupArgs& a, int n, int group) {
  const float x = to_f(((const T*)a.x)[n * a.x_b + (int64_t)group * a.each]);
  return fabsf(x) < INFINITY ? x : 0.0f;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void group_sums_kernel(const GroupArgs a) {
  constexpr int V = kVec<T>;
  __shared__ double lds[2][kThreads * V];
  const Chunk c = chunk_of(a, blockIdx.x);
  const int packs = (c.size + V - 1) / V, rows = kThreads / packs, tx = threadIdx.x % packs, ty = threadIdx.x / packs;
  double s[V] = {}, q[V] = {}, from[V];
  if (ty < rows) {
#pragma unroll
    for (int i = 0; i < V; ++i) from[i] = (double)origin_of<T>(a, c.n, (c.first + min(tx * V + i, c.size - 1)) / a.each);
    const T* const at[1] = {(const T*)a.x + c.n * a.x_b + c.first + tx * V};
    const int64_t stride[1] = {a.x_p};
    const int64_t p0 = c.split * a.per, p1 = min(a.places, p0 + a.per);
    over_places<T, 1>(at, stride, p0, p1, ty, rows, c.size - tx * V, [&](int64_t, const Pack<T>(&p)[1]) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double x = (double)to_f(p[0][i]) - from[i];
        s[i] += x;
        q[i] = fma(x, x, q[i]);
      }
    });
#pragma unroll
    for (int i = 0; i < V; ++i) {
      lds[0][ty * packs * V + tx * V + i] = s[i];
      lds[1][ty * packs * V + tx * V + i] = q[i];
    }
  }
  __syncthreads();
  const int each = a.per_group > 1 ? c.size : a.each, parts = a.splits * a.per_group;
  sum_groups(c.groups, rows * each, [&](int j, int e, double(&v)[2]) {
    const int row = e / each, col = j * each + e % each;
    v[0] = lds[0][row * packs * V + col];
    v[1] = lds[1][row * packs * V + col];
  }, [&](int j, const double(&v)[2]) {
    double* to = a.part + (((int64_t)c.n * parts + c.split * a.per_group + c.sub) * a.groups + c.group + j) * 2;
    to[0] = v[0];
    to[1] = v[1];
  });
}

// exp(-z) where a product's rounding in the exponent does not show (f32), or shows less than the result's (16 bits)
template <typename T>
__device__ __forceinline__ float exp_minus(float z) {
  constexpr float kLog2e = 1.44269502162933349609375f, kRest = 1.925963033500011e-08f;   // their sum is log2(e)
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(-z * kLog2e);
  const float hi = -z * kLog2e, lo = fmaf(-z, kLog2e, -hi) - z * kRest;
  const float e = __builtin_amdgcn_exp2f(hi);
  return fabsf(hi) < 126.0f ? fmaf(e, lo * 0.693147180559945f, e) : e;
}
template <typename T>
__device__ __forceinline__ float over(float x, float y) {
  if constexpr (sizeof(T) == 2) return x * __builtin_amdgcn_rcpf(y);
  return x / y;
}
template <typename T, int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == kRelu) return z < 0.0f ? 0.0f : z;    // (NaN stays)
  if constexpr (ACT == kSilu) return over<T>(z, 1.0f + exp_minus<T>(z));
  return z;
}

// Where a group's sums over the parts end up: mean and rstd of the chunk's groups.
template <typename T>
__device__ __forceinline__ void statistics(const GroupArgs& a, const Chunk& c, float* mean, float* rstd) {
  const int parts = a.splits * a.per_group;
  const double inv = 1.0 / ((double)a.places * a.each);
  const double* from = a.part + ((int64_t)c.n * parts * a.groups + c.group) * 2;
  sum_groups(c.groups, parts, [&](int j, int e, double(&v)[2]) {
    v[0] = from[((int64_t)e * a.groups + j) * 2];
    v[1] = from[((int64_t)e * a.groups + j) * 2 + 1];
  }, [&](int j, const double(&v)[2]) {
    const double m = v[0] * inv, var = v[1] * inv - m * m;
    mean[j] = (float)((double)origin_of<T>(a, c.n, c.group + j) + m);
    rstd[j] = (float)(1.0 / sqrt((var < 0 ? 0.0 : var) + a.eps));   // (NaN stays)
    if (c.split == 0 && c.sub == 0) {
      a.mean[(int64_t)c.n * a.groups + c.group + j] = mean[j];
      a.rstd[(int64_t)c.n * a.groups + c.group + j] = rstd[j];
    }
  });
  __syncthreads();
}

template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void group_apply_kernel(const GroupArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float mean[kWide], rstd[kWide];
  const Chunk c = chunk_of(a, gridDim.x - 1 - blockIdx.x);   // what was read last is in the caches
  statistics<T>(a, c, mean, rstd);
  const int packs = (c.size + V - 1) / V, rows = kThreads / packs, tx = threadIdx.x % packs, ty = threadIdx.x / packs, left = c.size - tx * V;
  if (ty >= rows) return;
  float mu[V], times[V], plus[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int col = min(tx * V + i, c.size - 1), j = a.per_group > 1 ? 0 : col / a.each;
    mu[i] = mean[j];
    times[i] = rstd[j] * param<T>(a, a.scale, c.first + col, 1.0f);
    plus[i] = param<T>(a, a.offset, c.first + col, 0.0f);
  }
  const T* const at[1] = {(const T*)a.x + c.n * a.x_b + c.first + tx * V};
  const int64_t stride[1] = {a.x_p};
  T* out = (T*)a.out + c.n * a.places * a.channels + c.first + tx * V;
  const int64_t p0 = c.split * a.per, p1 = min(a.places, p0 + a.per);
  over_places<T, 1>(at, stride, p0, p1, ty, rows, left, [&](int64_t place, const Pack<T>(&p)[1]) {
    Pack<T> y;
#pragma unroll
    for (int i = 0; i < V; ++i) y.set(i, from_f<T>(activate<T, ACT>((to_f(p[0][i]) - mu[i]) * times[i] + plus[i])));
    store_pack(out + place * a.channels, y, left);
  });
}

__device__ __forceinline__ float apart(float x) {
  asm volatile("" : "+v"(x));
  return x;
}
// h = dy act'(z).  Which side of zero z is on decides a whole gradient: next to zero it is formed in 64 bits.
template <typename T, int ACT>
__device__ __forceinline__ float through(float dy, float x, float xh, float mu, float r, float w, float b) {
  if constexpr (ACT == kRelu) {
    const float z = xh * w + b;
    bool on = z > 0.0f;
    if (fabsf(z) <= 4e-7f * (fabsf(xh * w) + fabsf(b)))   // (formed where it is needed: kept, the parameters in 64 bits would take 64 registers)
      on = ((double)apart(x) - (double)apart(mu)) * (double)apart(r) * (double)apart(w) + (double)apart(b) > 0.0;
    return on ? dy : z == z ? 0.0f : z;
  }
  if constexpr (ACT == kSilu) {
    const float z = xh * w + b, sig = over<T>(1.0f, 1.0f + exp_minus<T>(z));
    return dy * (sig * (1.0f + z * (1.0f - sig)));
  }
  return dy;
}

template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void group_grad_sums_kernel(const GroupArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float lds[2][kThreads * V];
  const Chunk c = chunk_of(a, blockIdx.x);
  const int packs = (c.size + V - 1) / V, rows = kThreads / packs, tx = threadIdx.x % packs, ty = threadIdx.x / packs;
  if (ty < rows) {
    float s[V] = {}, q[V] = {}, mu[V], r[V], w[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = min(c.first + tx * V + i, c.first + c.size - 1);
      const int64_t g = (int64_t)c.n * a.groups + col / a.each;
      mu[i] = a.mean[g];
      r[i] = a.rstd[g];
      w[i] = param<T>(a, a.scale, col, 1.0f);
      b[i] = param<T>(a, a.offset, col, 0.0f);
    }
    const T* const at[2] = {(const T*)a.x + c.n * a.x_b + c.first + tx * V, (const T*)a.dy + c.n * a.dy_b + c.first + tx * V};
    const int64_t stride[2] = {a.x_p, a.dy_p};
    const int64_t p0 = c.split * a.per, p1 = min(a.places, p0 + a.per);
    over_places<T, 2>(at, stride, p0, p1, ty, rows, c.size - tx * V, [&](int64_t, const Pack<T>(&p)[2]) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = to_f(p[0][i]), xh = (x - mu[i]) * r[i];
        const float h = through<T, ACT>(to_f(p[1][i]), x, xh, mu[i], r[i], w[i], b[i]);
        s[i] += h;
        q[i] += h * xh;
      }
    });
#pragma unroll
    for (int i = 0; i < V; ++i) {
      lds[0][ty * packs * V + tx * V + i] = s[i];
      lds[1][ty * packs * V + tx * V + i] = q[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < c.size * 8; e += kThreads) {   // 8 threads a channel, of one wave
    const int col = e >> 3;
    float s = 0, q = 0;
    for (int k = e & 7; k < rows; k += 8) {
      s += lds[0][k * packs * V + col];
      q += lds[1][k * packs * V + col];
    }
#pragma unroll
    for (int k = 4; k > 0; k >>= 1) {
      s += __shfl_xor(s, k, 64);
      q += __shfl_xor(q, k, 64);
    }
    if (e & 7) continue;
    float* to = a.columns + (((int64_t)c.n * a.splits + c.split) * a.channels + c.first + col) * 2;
    to[0] = s;
    to[1] = q;
    const float w = param<T>(a, a.scale, c.first + col, 1.0f);
    lds[0][col] = s * w;   // (row 0 of this channel, whose readers are these threads)
    lds[1][col] = q * w;
  }
  __syncthreads();
  const int each = a.per_group > 1 ? c.size : a.each, parts = a.splits * a.per_group;
  sum_groups(c.groups, each, [&](int j, int e, double(&v)[2]) {
    v[0] = (double)lds[0][j * each + e];
    v[1] = (double)lds[1][j * each + e];
  }, [&](int j, const double(&v)[2]) {
    double* to = a.part + (((int64_t)c.n * parts + c.split * a.per_group + c.sub) * a.groups + c.group + j) * 2;
    to[0] = v[0];
    to[1] = v[1];
  });
}

constexpr int kColumns = 16;   // columns of dscale and doffset that a block adds

// dscale and doffset of kColumns channels: 16 threads a channel take the parts in turn.
template <typename T>
__device__ __forceinline__ void add_columns(const GroupArgs& a, int block) {
  __shared__ double lds[2][kThreads / kColumns][kColumns];
  const int cx = threadIdx.x % kColumns, ty = threadIdx.x / kColumns, c = block * kColumns + cx;
  const int64_t parts = (int64_t)a.batch * a.splits;
  double s = 0, q = 0;
  if (c < a.channels)
    for (int64_t p = ty; p < parts; p += kThreads / kColumns) {
      s += (double)a.columns[(p * a.channels + c) * 2];
      q += (double)a.columns[(p * a.channels + c) * 2 + 1];
    }
  lds[0][ty][cx] = s;
  lds[1][ty][cx] = q;
  __syncthreads();
  if (ty == 0 && c < a.channels) {
    for (int k = 1; k < kThreads / kColumns; ++k) {
      s += lds[0][k][cx];
      q += lds[1][k][cx];
    }
    if (a.doffset) set_param<T>(a, a.doffset, c, (float)s);
    if (a.dscale) set_param<T>(a, a.dscale, c, (float)q);
  }
}

// The first blocks add dscale and doffset, the others form dx.
template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void group_grad_apply_kernel(const GroupArgs a, int adders) {
  constexpr int V = kVec<T>;
  if ((int)blockIdx.x < adders) {
    add_columns<T>(a, blockIdx.x);
    return;
  }
  __shared__ float mean_h[kWide], mean_hx[kWide];
  const Chunk c = chunk_of(a, gridDim.x - 1 - blockIdx.x);
  const int parts = a.splits * a.per_group;
  const double inv = 1.0 / ((double)a.places * a.each);
  const double* from = a.part + ((int64_t)c.n * parts * a.groups + c.group) * 2;
  sum_groups(c.groups, parts, [&](int j, int e, double(&v)[2]) {
    v[0] = from[((int64_t)e * a.groups + j) * 2];
    v[1] = from[((int64_t)e * a.groups + j) * 2 + 1];
  }, [&](int j, const double(&v)[2]) {
    mean_h[j] = (float)(v[0] * inv);
    mean_hx[j] = (float)(v[1] * inv);
  });
  __syncthreads();
  const int packs = (c.size + V - 1) / V, rows = kThreads / packs, tx = threadIdx.x % packs, ty = threadIdx.x / packs, left = c.size - tx * V;
  if (ty >= rows) return;
  float mu[V], r[V], w[V], b[V], rw[V], m0[V], m1[V];   // the means times r
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int col = min(tx * V + i, c.size - 1), j = a.per_group > 1 ? 0 : col / a.each;
    const int64_t g = (int64_t)c.n * a.groups + c.group + j;
    mu[i] = a.mean[g];
    r[i] = a.rstd[g];
    w[i] = param<T>(a, a.scale, c.first + col, 1.0f);
    b[i] = param<T>(a, a.offset, c.first + col, 0.0f);
    rw[i] = r[i] * w[i];
    m0[i] = r[i] * mean_h[j];
    m1[i] = r[i] * mean_hx[j];
  }
  const T* const at[2] = {(const T*)a.x + c.n * a.x_b + c.first + tx * V, (const T*)a.dy + c.n * a.dy_b + c.first + tx * V};
  const int64_t stride[2] = {a.x_p, a.dy_p};
  T* out = (T*)a.out + c.n * a.places * a.channels + c.first + tx * V;
  const int64_t p0 = c.split * a.per, p1 = min(a.places, p0 + a.per);
  over_places<T, 2>(at, stride, p0, p1, ty, rows, left, [&](int64_t place, const Pack<T>(&p)[2]) {
    Pack<T> dx;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = to_f(p[0][i]), xh = (x - mu[i]) * r[i];
      const float h = through<T, ACT>(to_f(p[1][i]), x, xh, mu[i], r[i], w[i], b[i]);
      dx.set(i, from_f<T>(h * rw[i] - (m0[i] + xh * m1[i])));
    }
    store_pack(out + place * a.channels, dx, left);
  });
}

// ---- resident: all places of a chunk of whole groups in a block's registers ----------------------------------

constexpr int kFour = 4;   // channels a thread takes of a place

// four channels of a place, as the words they are loaded as
template <typename T>
struct Quad {
  unsigned w[sizeof(T)];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(w, p, 4 * sizeof(T)); }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return to_f(__builtin_bit_cast(T, w[i]));
    else return to_f(__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1)))));
  }
};
template <typename T>
__device__ __forceinline__ void store_quad(T* p, const float (&f)[4]) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = from_f<T>(f[i]);
  __builtin_memcpy(p, t, sizeof(t));
}

// The chunk of a block, whose neighbours share the lines of memory that its places lie in: the chunks of a sequence are one XCD's.  (Blocks are dealt
// to the 8 XCDs in turn.)
struct Resident {
  int n, first;        // sequence, first channel
  int quads, rows;     // threads of a place; places at a time
  int tx, ty;
};
__device__ __forceinline__ Resident resident_of(const GroupArgs& a) {
  const int64_t id = blockIdx.x, whole = (int64_t)a.batch / 8 * 8 * a.chunks;
  Resident c;
  int k;
  if (id < whole) {
    c.n = (int)(id / 8 / a.chunks * 8 + id % 8);
    k = (int)(id / 8 % a.chunks);
  } else {
    c.n = (int)(a.batch / 8 * 8 + (id - whole) / a.chunks);
    k = (int)((id - whole) % a.chunks);
  }
  c.first = k * a.width;
  c.quads = a.width / kFour;
  c.rows = blockDim.x / c.quads;
  c.tx = threadIdx.x % c.quads;
  c.ty = threadIdx.x / c.quads;
  return c;
}

// Sums over the rows of a block, and the channels of each of its groups, of two numbers a thread and channel; sums[j]: of group j, for all threads.  Waves take
// the groups in turn, or share one; the order is fixed.  columns(col, s, q): the sums of a channel, for who wants them.
template <typename N, class Columns>
__device__ __forceinline__ void resident_sums(const GroupArgs& a, const Resident& c, const N (&s)[kFour], const N (&q)[kFour], char* lds, double (*sums)[2],
                                              Columns columns) {
  N* one = (N*)lds;                                  // [rows][width]
  N* two = one + (int64_t)c.rows * a.width;
  if (c.ty < c.rows)
#pragma unroll
    for (int i = 0; i < kFour; ++i) {
      one[c.ty * a.width + c.tx * kFour + i] = s[i];
      two[c.ty * a.width + c.tx * kFour + i] = q[i];
    }
  __syncthreads();
  // channels first: every 8 threads (or fewer) add one channel's rows
  for (int e = threadIdx.x; e < a.width * 8; e += blockDim.x) {
    const int col = e >> 3;
    N x = 0, y = 0;
    for (int k = e & 7; k < c.rows; k += 8) {
      x += one[k * a.width + col];
      y += two[k * a.width + col];
    }
    // (the 8 threads are of one wave, and all of them are here: blocks have a multiple of 64 threads, and so has their work)
#pragma unroll
    for (int k = 4; k > 0; k >>= 1) {
      x += __shfl_xor(x, k, 64);
      y += __shfl_xor(y, k, 64);
    }
    if ((e & 7) == 0) {
      columns(col, x, y);
      one[col] = x;   // (row 0 of this channel: its reader is among these threads, and done)
      two[col] = y;
    }
  }
  __syncthreads();
  const int groups = a.width / a.each, lanes = a.each > 64 ? 64 : 8, at = threadIdx.x % lanes;   // of a group
  for (int j = threadIdx.x / lanes; j < groups; j += blockDim.x / lanes) {
    double x = 0, y = 0;
    for (int e = at; e < a.each; e += lanes) {
      x += (double)one[j * a.each + e];
      y += (double)two[j * a.each + e];
    }
    for (int k = lanes >> 1; k > 0; k >>= 1) {
      x += __shfl_xor(x, k, 64);
      y += __shfl_xor(y, k, 64);
    }
    if (at == 0) {
      sums[j][0] = x;
      sums[j][1] = y;
    }
  }
  __syncthreads();
}

constexpr int kResidentWide = 512;   // channels of a resident chunk, at most: its threads

template <typename T, int NP>
__global__ __launch_bounds__(1024) void group_resident_kernel(const GroupArgs a, int activation) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ double sums[kResidentWide][2];
  const Resident c = resident_of(a);
  const bool on = c.ty < c.rows;
  const int places = (int)a.places;
  const T* x = (const T*)a.x + c.n * a.x_b + c.first + c.tx * kFour;
  Quad<T> in[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) in[k].load(x + min(c.ty + k * c.rows, places - 1) * a.x_p);
  float w[kFour], b[kFour], mu[kFour], from[kFour];
#pragma unroll
  for (int i = 0; i < kFour; ++i) from[i] = origin_of<T>(a, c.n, (c.first + c.tx * kFour + i) / a.each);
  double s[kFour] = {}, q[kFour] = {};
#pragma unroll
  for (int k = 0; k < NP; ++k)
    if (on && c.ty + k * c.rows < places)
#pragma unroll
      for (int i = 0; i < kFour; ++i) {
        const double v = (double)in[k][i] - (double)from[i];
        s[i] += v;
        q[i] = fma(v, v, q[i]);
      }
  resident_sums(a, c, s, q, lds, sums, [](int, double&, double&) {});
  const double inv = 1.0 / ((double)a.places * a.each);
  const int groups = a.width / a.each;
  for (int j = threadIdx.x; j < groups; j += blockDim.x) {
    const double off = sums[j][0] * inv, var = sums[j][1] * inv - off * off, m = (double)origin_of<T>(a, c.n, c.first / a.each + j) + off;
    const int64_t g = (int64_t)c.n * a.groups + c.first / a.each + j;
    a.mean[g] = (float)m;
    a.rstd[g] = (float)(1.0 / sqrt((var < 0 ? 0.0 : var) + a.eps));   // (NaN stays)
    sums[j][0] = m;
    sums[j][1] = (double)a.rstd[g];
  }
  __syncthreads();
  if (!on) return;
  // (the parameters are read here: ahead of the sums they take registers that the places need; 16 x 32 x 32 x 640 in bf16: 21.3 us instead of 17.1)
#pragma unroll
  for (int i = 0; i < kFour; ++i) {
    const int j = (c.tx * kFour + i) / a.each;
    mu[i] = (float)sums[j][0];
    w[i] = param<T>(a, a.scale, c.first + c.tx * kFour + i, 1.0f) * (float)sums[j][1];
    b[i] = param<T>(a, a.offset, c.first + c.tx * kFour + i, 0.0f);
  }
  T* out = (T*)a.out + (c.n * a.places * a.channels + c.first + c.tx * kFour);
  auto write = [&](auto act) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int place = c.ty + k * c.rows;
      if (place < places) {
        float y[kFour];
#pragma unroll
        for (int i = 0; i < kFour; ++i) y[i] = activate<T, decltype(act)::value>((in[k][i] - mu[i]) * w[i] + b[i]);
        store_quad(out + (int64_t)place * a.channels, y);
      }
    }
  };
  if (activation == kSilu) write(std::integral_constant<int, kSilu>());
  else if (activation == kRelu) write(std::integral_constant<int, kRelu>());
  else write(std::integral_constant<int, kNone>());
}

template <typename T, int NP>
__global__ __launch_bounds__(1024) void group_grad_resident_kernel(const GroupArgs a, int activation) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ double sums[kResidentWide][2];
  const Resident c = resident_of(a);
  const bool on = c.ty < c.rows;
  const int places = (int)a.places;
  const T* x = (const T*)a.x + c.n * a.x_b + c.first + c.tx * kFour;
  const T* dy = (const T*)a.dy + c.n * a.dy_b + c.first + c.tx * kFour;
  Quad<T> in[NP], go[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    in[k].load(x + min(c.ty + k * c.rows, places - 1) * a.x_p);
    go[k].load(dy + min(c.ty + k * c.rows, places - 1) * a.dy_p);
  }
  float w[kFour], b[kFour], mu[kFour], r[kFour];
#pragma unroll
  for (int i = 0; i < kFour; ++i) {
    const int col = c.first + c.tx * kFour + i;
    const int64_t g = (int64_t)c.n * a.groups + col / a.each;
    mu[i] = a.mean[g];
    r[i] = a.rstd[g];
    w[i] = param<T>(a, a.scale, col, 1.0f);
    b[i] = param<T>(a, a.offset, col, 0.0f);
  }
  T* out = (T*)a.out + (c.n * a.places * a.channels + c.first + c.tx * kFour);
  auto all = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    float s[kFour] = {}, q[kFour] = {};
#pragma unroll
    for (int k = 0; k < NP; ++k)
      if (on && c.ty + k * c.rows < places)
#pragma unroll
        for (int i = 0; i < kFour; ++i) {
          const float v = in[k][i], xh = (v - mu[i]) * r[i], h = through<T, ACT>(go[k][i], v, xh, mu[i], r[i], w[i], b[i]);
          s[i] += h;
          q[i] += h * xh;
        }
    float* columns = a.columns + ((int64_t)c.n * a.channels + c.first) * 2;
    // (the groups' sums are of h w: the weight of a channel times its sums)
    resident_sums(a, c, s, q, lds, sums, [&](int col, float& sum, float& product) {
      columns[col * 2] = sum;
      columns[col * 2 + 1] = product;
      const float weight = param<T>(a, a.scale, c.first + col, 1.0f);
      sum *= weight;
      product *= weight;
    });
    if (!on) return;
    const double inv = 1.0 / ((double)a.places * a.each);
    float rw[kFour], m0[kFour], m1[kFour];
#pragma unroll
    for (int i = 0; i < kFour; ++i) {
      const int j = (c.tx * kFour + i) / a.each;
      rw[i] = r[i] * w[i];
      m0[i] = r[i] * (float)(sums[j][0] * inv);
      m1[i] = r[i] * (float)(sums[j][1] * inv);
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int place = c.ty + k * c.rows;
      if (place < places) {
        float dx[kFour];
#pragma unroll
        for (int i = 0; i < kFour; ++i) {
          const float v = in[k][i], xh = (v - mu[i]) * r[i], h = through<T, ACT>(go[k][i], v, xh, mu[i], r[i], w[i], b[i]);
          dx[i] = h * rw[i] - (m0[i] + xh * m1[i]);
        }
        store_quad(out + (int64_t)place * a.channels, dx);
      }
    }
  };
  if (activation == kSilu) all(std::integral_constant<int, kSilu>());
  else if (activation == kRelu) all(std::integral_constant<int, kRelu>());
  else all(std::integral_constant<int, kNone>());
}
template <typename T, int>
__global__ __launch_bounds__(kThreads) void group_columns_kernel(const GroupArgs a) {
  add_columns<T>(a, blockIdx.x);
}

constexpr int kMostPlaces = 128;   // that a thread adds, in f32 in the backward pass

// The resident form takes a call where a chunk of whole groups, of four channels' multiples and 32 bytes at least, leaves a thread few enough places to
// hold, and where there are many chunks, or short ones.  Forward, 16 x 64 x 64 x 320 in bf16, 21 places a thread: 28 us, in two launches 33.  Of x and dy
// a thread holds ten places each (twice as many take more registers than 1024 threads have: 57 us, in two launches 54); 40 chunks of 21 places
// (5 x 53 x 79 x 96 in f32) take 26 us.
constexpr int kPacks = 22, kGradPacks = 10;
bool plan_resident(GroupArgs* a, int type, bool backward) {
  const int size = type_size(type);
  a->each = a->channels / a->groups;
  for (int together = 1; together <= 16 && together <= a->groups; ++together) {
    const int64_t width = (int64_t)together * a->each;
    if (a->groups % together || width % kFour || width * size < 32) continue;
    if (width > kResidentWide || (int64_t)a->batch * (a->groups / together) >= (1 << 21)) return false;   // (of 1024 threads: a grid has fewer than 2^32)
    const int quads = (int)width / kFour;
    const int64_t rows = std::min<int64_t>(1024 / quads, a->places), packs = ceil_div(a->places, rows);
    if (packs > (backward ? kGradPacks : kPacks) || (packs > 5 && a->batch * (a->groups / together) < 128)) return false;
    a->width = (int)width;
    a->chunks = a->groups / together;
    a->per_group = a->splits = 1;
    a->per = a->places;
    a->resident = (int)packs;
    a->threads = (int)round_up(rows * quads, 64);
    return true;
  }
  return false;
}

// Sizes to chunks and splits.  A block a CU, whose start (the parts' sums, the channels' parameters) costs as much as some
// ten places a thread (the gradient of 16 x 64 x 64 x 320: 22 + 28 us; two blocks a CU 23 + 31, eight of 256 threads 30 + 51), and no thread with fewer places than it has
// on the way or more than kMostPlaces.
void plan(GroupArgs* a, int type) {
  const int64_t v = 16 / type_size(type);
  a->each = a->channels / a->groups;
  a->per_group = (int)ceil_div(a->each, kWide);
  if (a->per_group > 1) {
    a->width = (int)(ceil_div(ceil_div(a->each, a->per_group), v) * v);
    a->per_group = (int)ceil_div(a->each, a->width);
    a->chunks = a->groups * a->per_group;
  } else {
    const int together = std::min(a->groups, kWide / a->each);
    a->width = together * a->each;
    a->chunks = (int)ceil_div(a->groups, together);
  }
  const int64_t rows = kThreads / ceil_div(std::min(a->width, a->channels), v), blocks = std::max<int64_t>(1, (int64_t)a->batch * a->chunks);
  const int64_t most = std::max<int64_t>(1, ceil_div(a->places, rows * kAhead));
  const int64_t splits = std::max(std::min(std::max<int64_t>(1, ceil_div(256, blocks)), most), ceil_div(a->places, rows * kMostPlaces));
  a->per = std::max<int64_t>(1, ceil_div(a->places, splits));
  a->splits = (int)std::max<int64_t>(1, ceil_div(a->places, a->per));
}

int group_args(const char* what, const nnvhip_group_norm_args* d, bool backward, GroupArgs* a) {
  if (!d) NNV_FAIL(NNVHIP_ERR_ARG, "%s: null pointer", what);
  if (d->type < 0 || d->type > 2 || !known_type((int)d->type) || !(d->param_type == d->type || d->param_type == NNVHIP_TYPE_F32))
    NNV_FAIL(NNVHIP_ERR_ARG, "%s: the values are f32, bf16 or f16, scale and offset of the same type or f32", what);
  if (d->activation < kNone || d->activation > kSilu) NNV_FAIL(NNVHIP_ERR_ARG, "%s: the activation is none, relu or silu", what);
  if (d->batch < 0 || d->places < 1 || d->channels < 1 || d->groups < 1 || d->channels % d->groups)
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: at least one place and channel are expected, the channels in equal groups", what);
  if (d->channels >= (1 << 24) || d->batch >= (1 << 23) || d->places >= (int64_t(1) << 36))
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many values", what);
  a->batch = (int)d->batch;
  a->places = d->places;
  a->channels = (int)d->channels;
  a->groups = (int)d->groups;
  if (!plan_resident(a, (int)d->type, backward)) plan(a, (int)d->type);
  // (a grid has fewer than 2^32 threads, and the backward pass has blocks for its columns' sums)
  if ((int64_t)a->batch * a->chunks * a->splits + ceil_div(a->channels, kColumns) >= (int64_t(1) << 23)) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many values", what);
  a->x = d->x;
  a->x_b = d->x_stride[0];
  a->x_p = d->x_stride[1];
  a->dy = d->dy;
  a->dy_b = d->dy_stride[0];
  a->dy_p = d->dy_stride[1];
  a->out = backward ? d->dx : d->y;
  a->scale = d->scale;
  a->offset = d->offset;
  a->dscale = d->dscale;
  a->doffset = d->doffset;
  a->mean = d->mean;
  a->rstd = d->rstd;
  a->wide_params = d->param_type == NNVHIP_TYPE_F32;
  a->eps = d->epsilon;
  return NNVHIP_OK;
}

int64_t part_bytes(const GroupArgs& a) { return a.resident ? 0 : (int64_t)a.batch * a.splits * a.per_group * a.groups * 2 * (int64_t)sizeof(double); }
int64_t column_bytes(const GroupArgs& a) { return (int64_t)a.batch * a.splits * a.channels * 2 * (int64_t)sizeof(float); }

template <typename T, int NP>
void launch_resident(const GroupArgs& a, int activation, bool backward, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.chunks)), block(a.threads);
  const int rows = a.threads / (a.width / kFour);
  const size_t lds = (size_t)rows * a.width * 2 * (backward ? sizeof(float) : sizeof(double));
  if (!backward) hipLaunchKernelGGL((group_resident_kernel<T, NP>), grid, block, lds, st, a, activation);
  else if constexpr (NP <= kGradPacks) hipLaunchKernelGGL((group_grad_resident_kernel<T, NP>), grid, block, lds, st, a, activation);
}
template <typename T>
void resident(const GroupArgs& a, int activation, bool backward, hipStream_t st) {
  if (a.batch > 0) {
    if (a.resident <= 1) launch_resident<T, 1>(a, activation, backward, st);
    else if (a.resident <= 2) launch_resident<T, 2>(a, activation, backward, st);
    else if (a.resident <= 5) launch_resident<T, 5>(a, activation, backward, st);
    else if (a.resident <= 10) launch_resident<T, 10>(a, activation, backward, st);
    else launch_resident<T, 22>(a, activation, backward, st);
  }
  if (backward && (a.dscale || a.doffset))
    hipLaunchKernelGGL((group_columns_kernel<T, 0>), dim3((unsigned)ceil_div(a.channels, kColumns)), dim3(kThreads), 0, st, a);
}

template <typename T, int ACT>
void forward(const GroupArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.chunks * a.splits));
  hipLaunchKernelGGL((group_sums_kernel<T>), grid, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL((group_apply_kernel<T, ACT>), grid, dim3(kThreads), 0, st, a);
}
template <typename T, int ACT>
void backward(const GroupArgs& a, hipStream_t st) {
  const unsigned blocks = (unsigned)((int64_t)a.batch * a.chunks * a.splits), adders = a.dscale || a.doffset ? (unsigned)ceil_div(a.channels, kColumns) : 0;
  if (blocks) hipLaunchKernelGGL((group_grad_sums_kernel<T, ACT>), dim3(blocks), dim3(kThreads), 0, st, a);
  if (blocks + adders) hipLaunchKernelGGL((group_grad_apply_kernel<T, ACT>), dim3(blocks + adders), dim3(kThreads), 0, st, a, (int)adders);
}

#define GROUP_BY_ACTIVATION(CALL, T, act, ...)          \
  do {                                                  \
    if ((act) == kNone) CALL<T, kNone>(__VA_ARGS__);    \
    else if ((act) == kRelu) CALL<T, kRelu>(__VA_ARGS__); \
    else CALL<T, kSilu>(__VA_ARGS__);                   \
  } while (0)
#define GROUP_BY_TYPE(CALL, type, act, ...)                                            \
  do {                                                                                 \
    if ((type) == NNVHIP_TYPE_F32) GROUP_BY_ACTIVATION(CALL, float, act, __VA_ARGS__); \
    else if ((type) == NNVHIP_TYPE_BF16) GROUP_BY_ACTIVATION(CALL, bf16_t, act, __VA_ARGS__); \
    else GROUP_BY_ACTIVATION(CALL, f16_t, act, __VA_ARGS__);                           \
  } while (0)

#define GROUP_RESIDENT(type, ...)                                     \
  do {                                                                \
    if ((type) == NNVHIP_TYPE_F32) resident<float>(__VA_ARGS__);      \
    else if ((type) == NNVHIP_TYPE_BF16) resident<bf16_t>(__VA_ARGS__); \
    else resident<f16_t>(__VA_ARGS__);                                \
  } while (0)

}  // namespace
}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_group_norm_workspace(const nnvhip_group_norm_args* d, int64_t* bytes) {
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  GroupArgs a{};
  NNV_TRY(group_args("nnvhip_group_norm_workspace", d, false, &a));
  *bytes = part_bytes(a);
  return NNVHIP_OK;
}

int nnvhip_group_norm(nnvhip_ctx* ctx, const nnvhip_group_norm_args* d, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  GroupArgs a{};
  NNV_TRY(group_args("nnvhip_group_norm", d, false, &a));
  if (a.batch == 0) return NNVHIP_OK;
  if (!a.x || !a.out || !a.mean || !a.rstd) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_group_norm: null pointer");
  if (!(d->epsilon >= 0)) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_group_norm: epsilon must not be negative");
  if (workspace_bytes < part_bytes(a) || (part_bytes(a) && !workspace))
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_group_norm: a workspace of %lld bytes is needed", (long long)part_bytes(a));
  a.part = (double*)workspace;
  if (a.resident) GROUP_RESIDENT(d->type, a, (int)d->activation, false, (hipStream_t)stream);
  else GROUP_BY_TYPE(forward, d->type, d->activation, a, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

int nnvhip_group_norm_backward_workspace(const nnvhip_group_norm_args* d, int64_t* bytes) {
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  GroupArgs a{};
  NNV_TRY(group_args("nnvhip_group_norm_backward_workspace", d, true, &a));
  *bytes = part_bytes(a) + column_bytes(a);
  return NNVHIP_OK;
}

int nnvhip_group_norm_backward(nnvhip_ctx* ctx, const nnvhip_group_norm_args* d, void* workspace, int64_t workspace_bytes, void* stream) {
  ENTER_POINT_CALL(ctx);
  GroupArgs a{};
  NNV_TRY(group_args("nnvhip_group_norm_backward", d, true, &a));
  if (a.batch > 0) {
    if (!a.x || !a.dy || !a.out || !a.mean || !a.rstd) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_group_norm_backward: null pointer");
    const int64_t need = part_bytes(a) + column_bytes(a);
    if (!workspace || workspace_bytes < need)
      NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_group_norm_backward: a workspace of %lld bytes is needed", (long long)need);
    a.part = (double*)workspace;
    a.columns = (float*)((char*)workspace + part_bytes(a));
  }
  if (a.resident) GROUP_RESIDENT(d->type, a, (int)d->activation, true, (hipStream_t)stream);
  else GROUP_BY_TYPE(backward, d->type, d->activation, a, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
