// Layer normalization of points, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b        (per row of `size` values)
//   g = dy w;  dx = r (g - mean(g) - xh mean(g xh));  dw = sum over rows of dy xh;  db = sum over rows of dy
//
// Both are bound by memory: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx, and
// everything else they do fits under that.  A row is read once: its values stay in the registers of the lanes that hold it,
// so the variance is a second sum over registers around the mean already known (no difference of large squares).  All
// sums are f32; what is written in 16 bits is rounded once, at the store.
#include "points.h"

#include <algorithm>

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

constexpr int kThreads = 512;       // of the kernels for long rows
constexpr int kGradThreads = 512;   // of the backward pass

// Sum of N values over the LPR consecutive lanes that share a row, in a block of THREADS.  Rows of more than a wave add through LDS;
// `slot` alternates between two sets of partial sums, so that one barrier per sum is enough (a wave can be at most one
// sum ahead of another, and that one writes the other set).
template <int LPR, int THREADS, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* lds, int& slot) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lanes_sum<(LPR < 64 ? LPR : 64)>(v[k]);
  if constexpr (LPR > 64) {
    constexpr int kWaves = LPR / 64;
    const int wave = threadIdx.x >> 6;
    float* part = lds + slot * (THREADS / 64 * N);
    slot ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) part[wave * N + k] = v[k];
    __syncthreads();
    const int first = wave / kWaves * kWaves;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float s = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += part[(first + w) * N + k];
      v[k] = s;
    }
  }
}

// A lane's scales or offsets for a pack of T.  W: their type (T, or float).
template <typename T, typename W>
struct Params {
  Pack<W> p[kVec<T> / kVec<W>];
  __device__ __forceinline__ void load(const W* from, int64_t c, int64_t size) {
#pragma unroll
    for (int k = 0; k < kVec<T> / kVec<W>; ++k) p[k] = load_pack(from + c + k * kVec<W>, from ? size - c - k * kVec<W> : 0);
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f(p[i / kVec<W>][i % kVec<W>]); }
};

// LPR lanes a row, NV packs a lane, as many rows a block as its threads hold; a block takes rows in turn.  A group's next row
// is asked for as soon as the last one is out of the registers that it comes to, and the scales and offsets stay in registers over all rows.
//
// Bound by memory: 16384 x 4096 in bf16 takes 53 us, 5.0 TB/s (a copy of 256 MiB: 5.4), 10176 x 2944 in f32 49 us.  One row ahead is enough: with
// three, which the turn's end asked for, the latter took 59.
template <typename T, typename W, int LPR, int NV>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void norm_kernel(const T* __restrict__ x, int64_t x_stride, const W* __restrict__ scale,
                                                                     const W* __restrict__ offset, float eps, int64_t rows, int size,
                                                                     T* __restrict__ y, float* __restrict__ mean,
                                                                     float* __restrict__ rstd) {
  constexpr int V = kVec<T>, THREADS = LPR > 256 ? LPR : 256, kRows = THREADS / LPR;
  __shared__ float lds[2 * THREADS / 64];
  int slot = 0;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  Pack<T> next[NV];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
      next[j] = ask_pack(x + (row < rows ? row : 0) * x_stride, c, size);
    }
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + group;
  fetch(row);
  Params<T, W> w[NV], b[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    w[j].load(scale, (j * LPR + lane) * V, size);
    b[j].load(offset, (j * LPR + lane) * V, size);
  }
  const float per = 1.0f / size;
  const bool full = size == LPR * NV * V;   // every pack exists
  // every row of a block's turn takes part in its barriers
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < rows; first += step, row += step) {
    Pack<T> in[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) in[j] = full ? next[j] : settle_pack(next[j], (j * LPR + lane) * V, size);
    fetch(row + step);
    float s[1] = {0};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += to_f(in[j][i]);
    row_sum<LPR, THREADS, 1>(s, lds, slot);
    const float mu = s[0] / size;   // (times 1 / size, the mean of equal values would not be that value)
    float q[1] = {0};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = to_f(in[j][i]) - mu;
        q[0] += (j * LPR + lane) * V + i < size ? d * d : 0.0f;
      }
    row_sum<LPR, THREADS, 1>(q, lds, slot);
    const float r = 1.0f / sqrtf(q[0] * per + eps);
    if (row < rows) {
      if (lane == 0) {
        mean[row] = mu;
        rstd[row] = r;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
        if (c >= size) break;
        Pack<T> out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float v = (to_f(in[j][i]) - mu) * r;
          if (scale) v *= w[j][i];
          if (offset) v += b[j][i];
          out.set(i, from_f<T>(v));
        }
        store_pack(y + row * (int64_t)size + c, out, size - c);
      }
    }
  }
}

// A block's passes over rows too long for its registers: use(c, packs at c of the N rows), four packs of each on their way.
template <typename T, int N, class Use>
__device__ __forceinline__ void over_long_rows(const T* const (&row)[N], int64_t size, Use use) {
  constexpr int V = kVec<T>, STEP = kThreads * V, MANY = 4;
  int64_t c = (int64_t)threadIdx.x * V;
  for (int64_t first = 0; first + MANY * STEP <= size; first += MANY * STEP, c += MANY * STEP) {
    Pack<T> p[MANY][N];
#pragma unroll
    for (int k = 0; k < MANY; ++k)
#pragma unroll
      for (int n = 0; n < N; ++n) __builtin_memcpy(p[k][n].w, row[n] + c + k * STEP, 16);
#pragma unroll
    for (int k = 0; k < MANY; ++k) use(c + k * STEP, p[k]);
  }
  for (; c < size; c += STEP) {
    Pack<T> p[N];
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] = load_pack(row[n] + c, size - c);
    use(c, p);
  }
}

// Rows too long for the registers of a block: three passes over the row, the later ones out of the caches: 4096 x 16384 in f32
// takes 162 us, 3.3 TB/s of x and y (a pack at a time, its scales one by one: 233).
template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void norm_long_kernel(const T* __restrict__ x, int64_t x_stride, const W* __restrict__ scale,
                                                             const W* __restrict__ offset, float eps, int64_t size,
                                                             T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int V = kVec<T>;
  __shared__ float lds[2 * kThreads / 64];
  int slot = 0;
  const int64_t row = blockIdx.x;
  const T* const xr[1] = {x + row * x_stride};
  float s[1] = {0}, q[1] = {0};
  over_long_rows(xr, size, [&](int64_t, const Pack<T>(&in)[1]) {   // (what is behind the row is zero)
#pragma unroll
    for (int i = 0; i < V; ++i) s[0] += to_f(in[0][i]);
  });
  row_sum<kThreads, kThreads, 1>(s, lds, slot);
  const float mu = s[0] / size;
  over_long_rows(xr, size, [&](int64_t c, const Pack<T>(&in)[1]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = to_f(in[0][i]) - mu;
      q[0] += c + i < size ? d * d : 0.0f;
    }
  });
  row_sum<kThreads, kThreads, 1>(q, lds, slot);
  const float r = 1.0f / sqrtf(q[0] / size + eps);
  if (threadIdx.x == 0) {
    mean[row] = mu;
    rstd[row] = r;
  }
  over_long_rows(xr, size, [&](int64_t c, const Pack<T>(&in)[1]) {
    Params<T, W> w, b;
    w.load(scale, c, size);
    b.load(offset, c, size);
    Pack<T> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = (to_f(in[0][i]) - mu) * r;
      if (scale) v *= w[i];
      if (offset) v += b[i];
      out.set(i, from_f<T>(v));
    }
    store_pack(y + row * size + c, out, size - c);
  });
}

// The backward pass.  A block's kGradThreads / LPR groups take rows in turn, the next one on its way; every lane keeps the sums of its
// own columns of dw and db in registers over all rows it sees.  At the end the groups of a block add theirs up in LDS, one
// after the other, and the block writes one row of partial sums (or the result, when there is one block); column_sum_kernel
// adds those in order.  No atomics: the same inputs give the same bits.  One block a CU: every block more would leave
// 8 * size bytes of partial sums more, and with a row ahead two waves a SIMD keep the memory busy (12345 x 768 in f32: 30.6 us with 256
// blocks, 39 with 512, 41 with 128; 16384 x 4096 in bf16: 85, 89 and 132 with the next row asked for at a turn's end).
//
// Bound by memory: 16384 x 4096 in bf16 takes 77 us, 5.2 TB/s.  Where rows have more than a wave, the next one is asked for in front of
// the sums, whose barriers no load is moved across (77 us; at the end of the turn 85).  Where a wave or less has them, the compiler moves the
// loads itself, and asked for early a row would take registers twice (12345 x 768 in f32: 32.0 us; at the end 30.6).
template <typename T, typename W, int LPR, int NV>
__global__ __launch_bounds__(kGradThreads) void norm_grad_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x,
                                                             int64_t x_stride, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const W* __restrict__ scale,
                                                             int64_t rows, int size, T* __restrict__ dx, W* __restrict__ dscale,
                                                             W* __restrict__ doffset, float* __restrict__ part) {
  constexpr int V = kVec<T>, kRows = kGradThreads / LPR, E = NV * V;
  __shared__ float lds[4 * kGradThreads / 64];
  __shared__ float sums[2 * LPR * E];
  int slot = 0;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  struct Row {
    Pack<T> x[NV], g[NV];
    float mu, r;
  } next;
  auto fetch = [&](int64_t row) {
    const bool here = row < rows;
    const int64_t at = here ? row : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * LPR + lane) * V;
      next.x[j] = ask_pack(x + at * x_stride, c, size);
      next.g[j] = ask_pack(dy + at * dy_stride, c, size);
    }
    next.mu = mean[at];
    next.r = rstd[at];
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + group;
  fetch(row);
  Params<T, W> w[NV];
  float dw[E], db[E];
#pragma unroll
  for (int j = 0; j < NV; ++j) w[j].load(scale, (j * LPR + lane) * V, size);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
  const float per = 1.0f / size;
  const bool full = size == LPR * NV * V && rows % step == 0;   // every pack exists, and every row of every turn
  // every row of a block's turn takes part in its barriers
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < rows; first += step, row += step) {
    Row now;
    now.mu = next.mu;
    now.r = row < rows ? next.r : 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      now.x[j] = full ? next.x[j] : settle_pack(next.x[j], (j * LPR + lane) * V, size);
      now.g[j] = full ? next.g[j] : settle_pack(next.g[j], row < rows ? (j * LPR + lane) * V : size, size);   // (a row that is not there: all zero)
    }
    const float mu = now.mu, r = now.r;
    if constexpr (LPR > 64) fetch(row + step);
    float s[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float g = to_f(now.g[j][i]), xh = (to_f(now.x[j][i]) - mu) * r, gw = scale ? g * w[j][i] : g;
        dw[j * V + i] += g * xh;   // g is zero where there is no column or no row
        db[j * V + i] += g;
        s[0] += gw;
        s[1] += gw * xh;
      }
    row_sum<LPR, kGradThreads, 2>(s, lds, slot);
    const float m0 = s[0] * per, m1 = s[1] * per;
    if (row < rows) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
        if (c >= size) break;
        Pack<T> out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float g = to_f(now.g[j][i]), xh = (to_f(now.x[j][i]) - mu) * r;
          out.set(i, from_f<T>(r * ((scale ? g * w[j][i] : g) - m0 - xh * m1)));
        }
        store_pack(dx + row * (int64_t)size + c, out, size - c);
      }
    }
    if constexpr (LPR <= 64) fetch(row + step);
  }
  if (dscale == nullptr && doffset == nullptr) return;
  for (int g = 0; g < kRows; ++g) {
    if (group == g)
#pragma unroll
      for (int e = 0; e < E; ++e) {   // (a lane's values lie apart, so that neighbouring lanes meet neighbouring banks)
        const int at = e * LPR + lane;
        sums[at] = (g ? sums[at] : 0.0f) + dw[e];
        sums[LPR * E + at] = (g ? sums[LPR * E + at] : 0.0f) + db[e];
      }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < size; c += kGradThreads) {
    const int at = (c / V / LPR * V + c % V) * LPR + c / V % LPR;
    if (gridDim.x == 1) {
      if (dscale) dscale[c] = from_f<W>(sums[at]);
      if (doffset) doffset[c] = from_f<W>(sums[LPR * E + at]);
    } else {
      part[((int64_t)blockIdx.x * 2 + 0) * size + c] = sums[at];
      part[((int64_t)blockIdx.x * 2 + 1) * size + c] = sums[LPR * E + at];
    }
  }
}

// Rows too long for registers: dx with the row read twice, the second time out of the caches (4096 x 16384 in bf16: 144 us with the sums, 2.8 TB/s
// of x, dy and dx) ...
template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void norm_grad_long_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x,
                                                                  int64_t x_stride, const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, const W* __restrict__ scale,
                                                                  int64_t size, T* __restrict__ dx) {
  constexpr int V = kVec<T>;
  __shared__ float lds[4 * kThreads / 64];
  int slot = 0;
  const int64_t row = blockIdx.x;
  const float mu = mean[row], r = rstd[row];
  const T* const at[2] = {x + row * x_stride, dy + row * dy_stride};
  float s[2] = {0, 0};
  over_long_rows(at, size, [&](int64_t c, const Pack<T>(&p)[2]) {   // (what is behind the rows is zero)
    Params<T, W> w;
    w.load(scale, c, size);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float g = to_f(p[1][i]), gw = scale ? g * w[i] : g;
      s[0] += gw;
      s[1] += gw * ((to_f(p[0][i]) - mu) * r);
    }
  });
  row_sum<kThreads, kThreads, 2>(s, lds, slot);
  const float m0 = s[0] / size, m1 = s[1] / size;
  over_long_rows(at, size, [&](int64_t c, const Pack<T>(&p)[2]) {
    Params<T, W> w;
    w.load(scale, c, size);
    Pack<T> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float g = to_f(p[1][i]), gw = scale ? g * w[i] : g;
      out.set(i, from_f<T>(r * (gw - m0 - (to_f(p[0][i]) - mu) * r * m1)));
    }
    store_pack(dx + row * size + c, out, size - c);
  });
}

// ... and the sums over rows by a thread per column and chunk of rows.
template <typename T>
__global__ __launch_bounds__(256) void norm_grad_columns_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ x,
                                                                int64_t x_stride, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, int64_t rows, int64_t size,
                                                                float* __restrict__ part) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= size) return;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
  float dw = 0, db = 0;
#pragma unroll 8
  for (int64_t row = r0; row < r1; ++row) {
    const float g = to_f(dy[row * dy_stride + c]);
    dw += g * ((to_f(x[row * x_stride + c]) - mean[row]) * rstd[row]);
    db += g;
  }
  part[((int64_t)blockIdx.y * 2 + 0) * size + c] = dw;
  part[((int64_t)blockIdx.y * 2 + 1) * size + c] = db;
}

// dscale / doffset = the partial sums added over `parts` rows.  64 columns a block, 16 threads a column with up to 8 loads on the way;
// blockIdx.y: which of the two.
template <typename W>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ part, int64_t parts, int64_t size,
                                                          W* __restrict__ dscale, W* __restrict__ doffset) {
  __shared__ float lds[16][64];
  W* out = blockIdx.y ? doffset : dscale;
  if (out == nullptr) return;
  const int cx = threadIdx.x % 64, py = threadIdx.x / 64;
  const int64_t c = (int64_t)blockIdx.x * 64 + cx;
  float s = 0;
  if (c < size)
    for (int64_t p = py; p < parts; p += 16 * 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p + 16 * k < parts ? part[((p + 16 * k) * 2 + blockIdx.y) * size + c] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  lds[py][cx] = s;
  __syncthreads();
  if (py == 0 && c < size) {
    s = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += lds[k][cx];
    out[c] = from_f<W>(s);
  }
}

constexpr int64_t kLongest = 8192;  // values of a row that the registers of a block hold

// Blocks of the backward pass: one a CU (see norm_grad_kernel), and none that would see less than four turns (of few rows, every block's partial
// sums are read again: 300 x 512 and 2048 x 1024 take as long with a turn each).
int64_t grad_blocks(int64_t rows, int64_t size, int type) {
  if (size > kLongest) return std::min<int64_t>(64, std::max<int64_t>(1, ceil_div(rows, 32)));
  const int64_t per = type == NNVHIP_TYPE_F32 ? 4 : 8;
  int64_t lpr = per == 8 ? 8 : 16;   // as NORM_BY_SIZE has it
  while (lpr < 16 && lpr * per < size) lpr *= 2;
  while (lpr < 64 && lpr * per * (per == 8 ? 2 : 1) < size) lpr *= 2;
  while (lpr * 16 < size) lpr *= 2;
  return std::max<int64_t>(1, std::min<int64_t>(256, ceil_div(rows, kGradThreads / lpr * 4)));
}

template <typename T, typename W, int LPR, int NV>
void launch_norm(const void* x, int64_t xs, const void* scale, const void* offset, float eps, int64_t rows, int64_t size, void* y,
                 float* mean, float* rstd, hipStream_t st) {
  constexpr int THREADS = LPR > 256 ? LPR : 256;
  const int64_t blocks = std::min<int64_t>(ceil_div(rows, THREADS / LPR), 256 * (1024 / THREADS));   // as many as the chip holds at once
  hipLaunchKernelGGL((norm_kernel<T, W, LPR, NV>), dim3((unsigned)blocks), dim3(THREADS), 0, st, (const T*)x, xs, (const W*)scale,
                     (const W*)offset, eps, rows, (int)size, (T*)y, mean, rstd);
}
template <typename T, typename W, int LPR, int NV>
void launch_norm_grad(const void* dy, int64_t dys, const void* x, int64_t xs, const float* mean, const float* rstd, const void* scale,
                      int64_t rows, int64_t size, void* dx, void* dscale, void* doffset, float* part, int64_t blocks, hipStream_t st) {
  hipLaunchKernelGGL((norm_grad_kernel<T, W, LPR, NV>), dim3((unsigned)blocks), dim3(kGradThreads), 0, st, (const T*)dy, dys, (const T*)x,
                     xs, mean, rstd, (const W*)scale, rows, (int)size, (T*)dx, (W*)dscale, (W*)doffset, part);
}

// The lanes that share a row, and the 16-byte packs a lane takes of it: up to a wave one pack of f32, two of 16 bits (from 129 values on); then
// up to 16 values a lane, and more waves.  Measured, forward, 2^25 values of 16 bits, 2^24 of f32: rows of 512 in bf16 25.5 us (64 lanes with a pack each:
// 28.8), of 200 29.1 (32 lanes: 33.6), of 256 in f32 26.8 (32 lanes, two packs: 30.8), of 1024 in bf16 25.3 (32 lanes, four packs: 26.8; 128 with one: 26.4);
// 16384 rows of 4096 in bf16 54 us (512 lanes with a pack each: 64; the gradient 78 and 99).
#define NORM_BY_SIZE(CALL, T, W, ...)                                         \
  do {                                                                        \
    constexpr int V_ = kVec<T>, P_ = V_ == 8 ? 2 : 1;                         \
    if (size <= 16 * V_ / 2 && V_ == 8) CALL<T, W, 8, 1>(__VA_ARGS__);        \
    else if (size <= 16 * V_) CALL<T, W, 16, 1>(__VA_ARGS__);                 \
    else if (size <= 32 * V_) CALL<T, W, 32 / P_, P_>(__VA_ARGS__);           \
    else if (size <= 64 * V_) CALL<T, W, 64 / P_, P_>(__VA_ARGS__);           \
    else if (size <= 128 * V_) CALL<T, W, 64, 2>(__VA_ARGS__);                \
    else if (size <= 1024) CALL<T, W, 64, 16 / V_>(__VA_ARGS__);              \
    else if (size <= 2048) CALL<T, W, 128, 16 / V_>(__VA_ARGS__);             \
    else if (size <= 4096) CALL<T, W, 256, 16 / V_>(__VA_ARGS__);             \
    else CALL<T, W, 512, 16 / V_>(__VA_ARGS__);                               \
  } while (0)

template <typename T, typename W>
void norm_forward(const void* x, int64_t xs, const void* scale, const void* offset, float eps, int64_t rows, int64_t size, void* y,
                  float* mean, float* rstd, hipStream_t st) {
  if (size > kLongest) {
    hipLaunchKernelGGL((norm_long_kernel<T, W>), dim3((unsigned)rows), dim3(kThreads), 0, st, (const T*)x, xs, (const W*)scale,
                       (const W*)offset, eps, size, (T*)y, mean, rstd);
    return;
  }
  NORM_BY_SIZE(launch_norm, T, W, x, xs, scale, offset, eps, rows, size, y, mean, rstd, st);
}

template <typename T, typename W>
void norm_backward(const void* dy, int64_t dys, const void* x, int64_t xs, const float* mean, const float* rstd, const void* scale,
                   int64_t rows, int64_t size, void* dx, void* dscale, void* doffset, float* part, int type, hipStream_t st) {
  const int64_t blocks = rows > 0 ? grad_blocks(rows, size, type) : 0;   // no rows: nothing to read, and sums of no parts
  if (size > kLongest && rows > 0) {
    hipLaunchKernelGGL((norm_grad_long_kernel<T, W>), dim3((unsigned)rows), dim3(kThreads), 0, st, (const T*)dy, dys, (const T*)x, xs,
                       mean, rstd, (const W*)scale, size, (T*)dx);
    if (dscale || doffset)
      hipLaunchKernelGGL((norm_grad_columns_kernel<T>), dim3((unsigned)ceil_div(size, 256), (unsigned)blocks), dim3(256), 0, st,
                         (const T*)dy, dys, (const T*)x, xs, mean, rstd, rows, size, part);
  } else if (rows > 0) {
    NORM_BY_SIZE(launch_norm_grad, T, W, dy, dys, x, xs, mean, rstd, scale, rows, size, dx, dscale, doffset, part, blocks, st);
    if (blocks == 1) return;
  }
  if (dscale || doffset)
    hipLaunchKernelGGL((column_sum_kernel<W>), dim3((unsigned)ceil_div(size, 64), 2), dim3(1024), 0, st, part, blocks, size, (W*)dscale,
                       (W*)doffset);
}

#define NORM_BY_TYPE(CALL, ...)                                                                 \
  do {                                                                                          \
    const bool wide = param_type == NNVHIP_TYPE_F32;                                            \
    if (type == NNVHIP_TYPE_F32) CALL<float, float>(__VA_ARGS__);                               \
    else if (type == NNVHIP_TYPE_BF16 && wide) CALL<bf16_t, float>(__VA_ARGS__);                \
    else if (type == NNVHIP_TYPE_BF16) CALL<bf16_t, bf16_t>(__VA_ARGS__);                       \
    else if (wide) CALL<f16_t, float>(__VA_ARGS__);                                             \
    else CALL<f16_t, f16_t>(__VA_ARGS__);                                                       \
  } while (0)

int check_norm(const char* what, int type, int param_type, int64_t rows, int64_t size) {
  if (!known_type(type) || !(param_type == type || param_type == NNVHIP_TYPE_F32))
    NNV_FAIL(NNVHIP_ERR_ARG, "%s: the values are f32, bf16 or f16, scale and offset of the same type or f32", what);
  if (rows < 0 || size < 1) NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: rows of at least one value are expected", what);
  if (rows >= (int64_t(1) << (size > kLongest ? 23 : 31)))   // (a block of kThreads for each long row: a grid has fewer than 2^32 threads)
    NNV_FAIL(NNVHIP_ERR_SHAPE, "%s: too many rows", what);
  return NNVHIP_OK;
}

}  // namespace
}  // namespace nnvhip

using namespace nnvhip;

extern "C" {

int nnvhip_layer_norm(nnvhip_ctx* ctx, int type, int param_type, int64_t rows, int64_t size, const void* x, int64_t x_stride,
                      const void* scale, const void* offset, double eps, void* y, float* mean, float* rstd, void* stream) {
  ENTER_POINT_CALL(ctx);
  NNV_TRY(check_norm("nnvhip_layer_norm", type, param_type, rows, size));
  if (rows == 0) return NNVHIP_OK;
  if (!x || !y || !mean || !rstd) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_layer_norm: null pointer");
  NORM_BY_TYPE(norm_forward, x, x_stride, scale, offset, (float)eps, rows, size, y, mean, rstd, (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

int nnvhip_layer_norm_backward_workspace(int type, int64_t rows, int64_t size, int64_t* bytes) {
  if (!bytes) NNV_FAIL(NNVHIP_ERR_ARG, "null pointer");
  NNV_TRY(check_norm("nnvhip_layer_norm_backward_workspace", type, type, rows, size));
  const int64_t blocks = grad_blocks(rows, size, type);
  *bytes = blocks == 1 && size <= kLongest ? 0 : blocks * 2 * size * (int64_t)sizeof(float);
  return NNVHIP_OK;
}

int nnvhip_layer_norm_backward(nnvhip_ctx* ctx, int type, int param_type, int64_t rows, int64_t size, const void* dy,
                               int64_t dy_stride, const void* x, int64_t x_stride, const float* mean, const float* rstd,
                               const void* scale, void* dx, void* dscale, void* doffset, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  ENTER_POINT_CALL(ctx);
  NNV_TRY(check_norm("nnvhip_layer_norm_backward", type, param_type, rows, size));
  if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_layer_norm_backward: null pointer");
  int64_t need = 0;
  NNV_TRY(nnvhip_layer_norm_backward_workspace(type, rows, size, &need));
  if (need > workspace_bytes || (need && !workspace))
    NNV_FAIL(NNVHIP_ERR_ARG, "nnvhip_layer_norm_backward: a workspace of %lld bytes is needed", (long long)need);
  if (rows == 0 && !dscale && !doffset) return NNVHIP_OK;
  NORM_BY_TYPE(norm_backward, dy, dy_stride, x, x_stride, mean, rstd, scale, rows, size, dx, dscale, doffset, (float*)workspace, type,
               (hipStream_t)stream);
  NNV_HIP_TRY(hipGetLastError());
  return NNVHIP_OK;
}

}  // extern "C"
