// What the operators on points and gradients share: the element types of a caller's tensors, wide loads and stores at any
// alignment, and the start of their entry points.
#pragma once
#include "internal.h"

#include <type_traits>

namespace nnvhip {

using bf16_t = __bf16;
using f16_t = _Float16;

// 16 bytes of T.  A tensor's rows start at any multiple of its element size (odd row lengths, views), so the wide accesses
// below ask for no more alignment than that: global memory takes them at any address, and a row that happens to be aligned
// loses nothing.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// (The pack is kept as the four words it is loaded as: taken apart where it is loaded, a pack that is asked for ahead would be
// waited for at once.)
template <typename T>
struct Pack {
  unsigned w[4];
  __device__ __forceinline__ T operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, w[i]);
    else return __builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
  __device__ __forceinline__ void set(int i, T x) {   // in ascending order: an even element clears its neighbour
    if constexpr (sizeof(T) == 4) w[i] = __builtin_bit_cast(unsigned, x);
    else w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | (unsigned)__builtin_bit_cast(uint16_t, x) << 16 : (unsigned)__builtin_bit_cast(uint16_t, x);
  }
};

// n of the pack's elements exist (n >= kVec: all); the others read as zero and are not touched in memory.
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p, int64_t n) {
  Pack<T> r;
  if (n >= kVec<T>) {
    __builtin_memcpy(r.w, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.set(i, i < n ? p[i] : (T)0.0f);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack<T>& r, int64_t n) {
  if (n >= kVec<T>) {
    __builtin_memcpy(p, r.w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < n) p[i] = r[i];
  }
}

// The pack from element c of a row of `size` elements on, in two parts: ask() for it with no lane taking another way than its neighbours (a
// lane that had its missing elements set to zero would have to wait for what others are loading into the same registers),
// and settle() when it is used: what lies behind the row is zero then.  A row shorter than a pack is read element by element.
template <typename T>
__device__ __forceinline__ Pack<T> ask_pack(const T* row, int c, int size) {
  if (size < kVec<T>) return load_pack(row + c, size - c);
  Pack<T> r;
  __builtin_memcpy(r.w, row + min(c, size - kVec<T>), 16);
  return r;
}
template <typename T>
__device__ __forceinline__ Pack<T> settle_pack(const Pack<T>& r, int c, int size) {
  Pack<T> s;
  if (size < kVec<T>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s.w[i] = c < size ? r.w[i] : 0u;
    return s;
  }
  const int missing = c + kVec<T> - size;   // elements that do not exist; the others are the last ones of what was read
  if (size % kVec<T> == 0) {                // all or none
#pragma unroll
    for (int i = 0; i < 4; ++i) s.w[i] = missing > 0 ? 0u : r.w[i];
    return s;
  }
  const int bits = min(max(missing, 0), kVec<T>) * 8 * (int)sizeof(T);
  const uint64_t lo = (uint64_t)r.w[1] << 32 | r.w[0], hi = (uint64_t)r.w[3] << 32 | r.w[2];
  const uint64_t down = bits == 0 ? lo : lo >> (bits & 63) | (bits < 64 ? hi << (-bits & 63) : 0);
  const uint64_t l = bits < 64 ? down : bits < 128 ? hi >> (bits & 63) : 0, u = bits < 64 ? hi >> bits : 0;
  s.w[0] = (unsigned)l;
  s.w[1] = (unsigned)(l >> 32);
  s.w[2] = (unsigned)u;
  s.w[3] = (unsigned)(u >> 32);
  return s;
}

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {  // to nearest, ties to even
  return (T)x;
}

// Sum over the W consecutive lanes (a power of two) that a lane is one of; every one of them gets it.  On the vector units alone: through
// LDS the six steps of a wave would take some 100 cycles each.
template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
  auto dpp = [&](auto ctrl) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if constexpr (W >= 2) dpp(std::integral_constant<int, 0xb1>());    // lane ^ 1 (quad_perm)
  if constexpr (W >= 4) dpp(std::integral_constant<int, 0x4e>());    // lane ^ 2
  if constexpr (W >= 8) dpp(std::integral_constant<int, 0x141>());   // the other four of eight (row_half_mirror)
  if constexpr (W >= 16) dpp(std::integral_constant<int, 0x140>());  // the other eight of sixteen (row_mirror)
  const auto both = [](auto r) { return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]); };
  if constexpr (W >= 32) x = both(__builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false));
  if constexpr (W >= 64) x = both(__builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false));
  return x;
}

// Selects the context's device for the life of an entry point.  The operators on points run on the stream the caller names
// and touch none of the context's sets, so nothing that waits on its own stream is sent ahead of them.
class PointCall {
 public:
  int enter(nnvhip_ctx* ctx) {
    NNV_HIP_TRY(hipGetDevice(&before_));
    if (before_ != ctx->device) {
      NNV_HIP_TRY(hipSetDevice(ctx->device));
      changed_ = true;
    }
    return NNVHIP_OK;
  }
  ~PointCall() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

#define ENTER_POINT_CALL(c)                                            \
  nnvhip::PointCall call_;                                             \
  do {                                                                 \
    if (!(c)) NNV_FAIL(NNVHIP_ERR_ARG, "null context");                \
    NNV_TRY(call_.enter(c));                                           \
  } while (0)

inline int type_size(int type) { return type == NNVHIP_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == NNVHIP_TYPE_F32 || type == NNVHIP_TYPE_BF16 || type == NNVHIP_TYPE_F16; }

}  // namespace nnvhip
