// Element types of the node-wise operators (embedding, feed-forward block, dropout): float32, bfloat16, float16 in
// memory, float32 in registers.
#pragma once
#include <hip/hip_fp16.h>
#include <string.h>

#include "fc_common.h"

namespace fc {

struct bf16_t {
  uint16_t v;
};
struct f16_t {
  uint16_t v;
};
struct e4m3_t {
  uint8_t v;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((uint32_t)x.v << 16); }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)__builtin_bit_cast(_Float16, x.v); }

// Round to nearest even.
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) {
  return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)x)};
}
template <>
__device__ __forceinline__ f16_t from_f32<f16_t>(float x) {
  return f16_t{__builtin_bit_cast(uint16_t, (_Float16)x)};
}

// N elements that are loaded and stored as one access, at any alignment that the elements have: the hardware takes
// unaligned vector accesses, at full rate where they are aligned.
template <class T, int N>
struct Pack {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  memcpy(&r, p, sizeof(r));
  return r;
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
  memcpy(p, &x, sizeof(x));
}

// 16 bytes of 16-bit elements, stored for a reader that comes much later.
template <class T>
__device__ __forceinline__ void stream_pack(T* p, const Pack<T, 8>& x) {
  typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
  words w;
  memcpy(&w, &x, 16);
  __builtin_nontemporal_store(w, (words*)p);
}

inline bool node_dtype_ok(int32_t dtype) { return dtype == FC_F32 || dtype == FC_BF16 || dtype == FC_F16; }
inline int64_t node_dtype_size(int32_t dtype) { return dtype == FC_F32 ? 4 : 2; }

// A grid has below 2^32 threads a dimension. Work of more blocks than this goes in several launches, f(first block, blocks)
// each, of GBs each.
constexpr int64_t kLaunchBlocks = 1 << 20;
template <class F>
int in_launches(int64_t blocks, F&& f) {
  for (int64_t b = 0; b < blocks; b += kLaunchBlocks) {
    f(b, (unsigned)(blocks - b < kLaunchBlocks ? blocks - b : kLaunchBlocks));
    FC_LAUNCH_CHECK();
  }
  return FC_OK;
}
inline bool grid_fits(int64_t blocks, int threads) { return blocks < (int64_t(1) << 32) / threads; }

// f(T{}) for the element type of a checked dtype code.
template <class F>
int with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case FC_F32: return f(float{});
    case FC_BF16: return f(bf16_t{});
    default: return f(f16_t{});
  }
}

}  // namespace fc
