// Attention of points in 16 bits, forward, on v_mfma_f32_32x32x16_{bf16,f16} (2.5 PFLOP/s at best).
#include "points_attend16.h"

#pragma clang fp contract(fast)

namespace nnvhip {
namespace {

// FEW = false: WAVES waves of 32 rows each share tiles of 64 keys.  FEW = true: 32 rows for the block, whose waves take tiles of 32
// keys in turn (see attend_kernel, which this is the 16-bit form of).
//
// The next tile is on its way to LDS (no registers in between) while one is worked on; one barrier a tile.  A weight is rounded to T
// before the product with the values.  The running maximum is raised only when a row's has grown by more than 2^8: the sums
// are in f32 and any base serves, so that the accumulators are hardly ever multiplied.
template <typename T, int DP, int WAVES, bool FEW>
__global__ __launch_bounds__(64 * WAVES) void attend16_kernel(const AttendArgs a) {
  constexpr int KEYS = FEW ? 32 : 64, TILE = KEYS * DP, STEP = FEW ? WAVES : 1;
  typedef PairLoad<T, DP, KEYS, FEW ? 1 : WAVES> Load;
  __shared__ __attribute__((aligned(1024))) T lds[(FEW ? WAVES : 1) * 2 * 2 * TILE];   // two pairs (k, v), of every wave if FEW
  __shared__ float row_max[FEW ? WAVES : 1][32], row_total[FEW ? WAVES : 1][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, h = lane >> 5;
  int64_t at = xcd_order(blockIdx.x, gridDim.x);
  const int split = at % a.splits;
  at /= a.splits;
  const int row_tile = at % a.row_tiles;
  const int bkv = at / a.row_tiles, b = bkv / a.kv_heads, kv = bkv % a.kv_heads;
  const int n = keys_that_count(a, b);
  const int tiles = (n + KEYS - 1) / KEYS, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per + (FEW ? wave : 0), t1 = min(tiles, split * per + per);
  const int64_t r = FEW ? (int64_t)row_tile * 32 + col : (int64_t)row_tile * (32 * WAVES) + wave * 32 + col;
  const bool row_here = r < a.rows;
  T* mine = lds + (FEW ? wave * 4 * TILE : 0);
  const unsigned mine_at = lds_addr_of(mine), rows_at = rows_place<T, DP>(lane), columns_at = columns_place<T, DP>(lane);

  if (DP != a.head) {   // the columns behind the head size, for good
    half8<T> zero = {};
    for (int e = threadIdx.x; e < (FEW ? WAVES : 1) * 4 * KEYS * (DP / 8); e += 64 * WAVES) __builtin_memcpy(lds + e * 8, &zero, 16);
    __syncthreads();
  }

  // A negative scale is moved into q's sign: the largest score is then the largest product.  (And one of zero is taken as one that
  // leaves every score next to zero, so that the -inf of a key that does not count stays one.)
  const float unit = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
  half8<T> qf[DP / 16];
  {
    const T* q = (const T*)a.q.p + (row_here ? row_at(a.q, a, b, kv, r) : 0);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      qf[c] = half8<T>{};
      if (row_here && 16 * c + 8 * h < a.head) __builtin_memcpy(&qf[c], q + 16 * c + 8 * h, 16);
      if (a.scale < 0) qf[c] = -qf[c];
    }
  }
  float16_t acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  float base = -INFINITY, total = 0.0f;   // base: of the exponents, in products times unit

  const T* kp = (const T*)a.k.p + b * a.k.b + kv * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + kv * a.v.h;
  Load load;
  load.init(FEW ? 0 : wave, lane, a.head);
  int counts = 0;   // FEW: lane i holds which keys of the i-th tile from here count; else: whether key `lane` of the next tile does
  auto fetch = [&](int t, int buffer) {
    // rows past the last key repeat it: what they hold is not used (see below)
    load.issue([&](int j) { return min(t * KEYS + j, n - 1); }, [&](int key) { return kp + key * a.k.t; },
               [&](int key) { return vp + key * a.v.t; }, mine_at + buffer * (4 * TILE), FEW ? 0 : wave);
    if constexpr (!FEW) counts = key_word(a, b, t * KEYS + lane, n);
  };
  int buffer = 0;
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0, turn = 0; t < t1; t += STEP, buffer ^= 1, ++turn) {
    uint64_t valid;
    if constexpr (FEW) {
      // A mask's bytes are read for 32 tiles at a time: a wait for one of them would be a wait for all transfers behind it.
      if (a.mask == nullptr) {
        const int rest = n - t * KEYS;
        valid = rest >= KEYS ? ~0ull : (1ull << rest) - 1;
      } else {
        if (turn % 32 == 0)
          for (int i = 0; i < 32; ++i) {
            const uint64_t word = __ballot(t + i * STEP < t1 && key_word(a, b, (t + i * STEP) * KEYS + col, n) != 0);
            if (lane == i) counts = (int)word;
          }
        const uint32_t word = __builtin_amdgcn_readlane(counts, turn % 32);
        valid = word == ~0u ? ~0ull : word;
      }
    } else {
      valid = __ballot(counts != 0);
    }
    T* vs = mine + (buffer * 2 + 1) * TILE;
    const unsigned ks_at = hide(mine_at + buffer * (4 * TILE) + rows_at), vs_at = hide(mine_at + (buffer * 4 + 2) * TILE + columns_at);
    if constexpr (FEW) {
      // the other pair was read before; its readers are done
      if (t + STEP < t1) {
        wait_vm_lds<63>();
        fetch(t + STEP, buffer ^ 1);
        wait_vm<Load::COUNT>();
      } else {
        wait_vm<0>();
      }
      __builtin_amdgcn_wave_barrier();
    } else {
      wait_vm_lds<0>();
      block_barrier();
      if (t + STEP < t1) fetch(t + STEP, buffer ^ 1);
    }
    if (valid != ~0ull) {   // v's rows that do not count: a weight of zero must meet a zero
      half8<T> zero = {};
      for (int e = FEW ? lane : threadIdx.x; e < KEYS * (DP / 8); e += FEW ? 64 : 64 * WAVES)
        if (!(valid >> (e / (DP / 8)) & 1)) __builtin_memcpy(vs + e * 8, &zero, 16);
      if constexpr (FEW) {
        wait_vm_lds<63>();
        __builtin_amdgcn_wave_barrier();
      } else {
        wait_vm_lds<63>();
        block_barrier();
      }
    }

    float16_t s[KEYS / 32];
    over_head<T, DP, KEYS / 32>(ks_at, 0, qf, s);
    if (valid != ~0ull) {
#pragma unroll
      for (int k = 0; k < KEYS / 32; ++k) {
        const uint32_t word = (uint32_t)(valid >> (32 * k)) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[k][i] = word >> product_row(i, 0) & 1 ? s[k][i] : -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k)
#pragma unroll
      for (int i = 0; i < 16; i += 2) top = max3(top, s[k][i], s[k][i + 1]);
    top = max_of_halves(top) * unit;
    if (__any(top > base + 8.0f)) {   // also: the first keys of a row that count
      const float next = fmaxf(base, top);
      const float fade = next == -INFINITY ? 1.0f : exp2_(base - next);
      base = next;
      total *= fade;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= fade;
    }
    const float off = base == -INFINITY ? 0.0f : base;
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[k][i] = exp2_(s[k][i] * unit - off);
        sum[i & 1] += s[k][i];
      }
    total += sum[0] + sum[1];
#pragma unroll
    for (int k = 0; k < KEYS / 32; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const half8<T> p = round8<T>(s[k], 8 * c);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = Half8<T>::mfma(columns_operand<T, DP>(vs_at, 32 * k + 16 * c, d), p, acc[d]);
      }
  }
  total = sum_of_halves(total);

  const int64_t heads_rows = (int64_t)a.batch * a.kv_heads * a.rows, flat = (int64_t)bkv * a.rows + r;
  if constexpr (!FEW) {
    if (!row_here) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const float lse = total == 0.0f ? -INFINITY : (base + log2f(total)) * kLn2;
    if (h == 0) (a.splits > 1 ? a.part_lse[split * heads_rows + flat] : a.lse[flat]) = lse;
    float* part = a.splits > 1 ? a.part + (split * heads_rows + flat) * a.head : nullptr;
    T* out = (T*)a.out + dense_row_at(a, b, kv, r);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = acc[d][4 * i4 + i] * inv;
        const int at_d = d * 32 + 8 * i4 + 4 * h;
        if (part) store_four(part, at_d, a.head, f);
        else store_four(out, at_d, a.head, f);
      }
  } else {
    constexpr int LD = DP + 4;
    static_assert(32 * LD * sizeof(float) <= 4 * TILE * sizeof(T), "a wave's result fits its tiles");
    __syncthreads();
    float* all_found = (float*)lds;
    float* found = all_found + wave * (32 * LD);   // [row][value]
    if (h == 0) {
      row_max[wave][col] = base;
      row_total[wave][col] = total;
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = acc[d][4 * i4 + i];
        __builtin_memcpy(found + col * LD + d * 32 + 8 * i4 + 4 * h, f, 16);
      }
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * (DP / 4); e += 64 * WAVES) {
      const int j = e / (DP / 4), d = e % (DP / 4) * 4;
      const int64_t rj = (int64_t)row_tile * 32 + j;
      if (rj >= a.rows) continue;
      float top = row_max[0][j], all = 0.0f, f[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 1; k < WAVES; ++k) top = fmaxf(top, row_max[k][j]);
      const float off = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) {
        const float w = exp2_(row_max[k][j] - off);
        all += w * row_total[k][j];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] += w * all_found[(k * 32 + j) * LD + d + i];
      }
      const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] *= inv;
      const int64_t fj = (int64_t)bkv * a.rows + rj, sj = split * heads_rows + fj;
      if (d == 0) (a.splits > 1 ? a.part_lse[sj] : a.lse[fj]) = all == 0.0f ? -INFINITY : (top + log2f(all)) * kLn2;
      if (d >= a.head) continue;
      if (a.splits > 1) store_four(a.part + sj * a.head, d, a.head, f);
      else store_four((T*)a.out + dense_row_at(a, b, kv, rj), d, a.head, f);
    }
  }
}

template <typename T, int DP>
void launch(const AttendArgs& a, bool few, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.kv_heads * a.row_tiles * a.splits));
  if (few) hipLaunchKernelGGL((attend16_kernel<T, DP, 4, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((attend16_kernel<T, DP, 8, false>), grid, dim3(512), 0, st, a);
}

}  // namespace

bool attend16_takes(const AttendArgs& a, int type) {
  return type != NNVHIP_TYPE_F32 && by_pieces(a.q, a.head) && by_pieces(a.k, a.head) && by_pieces(a.v, a.head);
}

void launch_attend16(const AttendArgs& a, int type, bool few, hipStream_t st) {
  if (type == NNVHIP_TYPE_BF16) ATTEND_BY_HEAD(launch, bf16_t, a, few, st);
  else ATTEND_BY_HEAD(launch, f16_t, a, few, st);
}

}  // namespace nnvhip
