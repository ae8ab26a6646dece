// What the operators on points and gradients share: the element types of a caller's tensors, wide loads and stores at any
// alignment, and the start of their entry points.
#pragma once
#include "internal.h"

namespace nnvhip {

using bf16_t = __bf16;
using f16_t = _Float16;

// 16 bytes of T.  A tensor's rows start at any multiple of its element size (odd row lengths, views), so the wide accesses
// below ask for no more alignment than that: global memory takes them at any address, and a row that happens to be aligned
// loses nothing.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
struct Pack {
  T v[kVec<T>];
};

// n of the pack's elements exist (n >= kVec: all); the others read as zero and are not touched in memory.
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p, int64_t n) {
  Pack<T> r;
  if (n >= kVec<T>) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = i < n ? p[i] : (T)0.0f;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack<T>& r, int64_t n) {
  if (n >= kVec<T>) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {  // to nearest, ties to even
  return (T)x;
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
