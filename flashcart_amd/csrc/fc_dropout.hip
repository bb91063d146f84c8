// Residual dropout: out[e] = residual[e] + keep(e) x[e] / (1 - p). keep(e) compares word e % 4 of the Philox4x32-10
// block (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011) of counter (e / 4, offset) and key seed
// with floor(p 2^32), so the mask is a function of the element's index and is never stored: the backward pass forms it
// again (out = keep(e) grad[e] / (1 - p) is the same kernel without a residual). Seed and offset are read on the
// device, so a captured graph sees the values of each replay. A dropped element is written as if x were 0 whatever it
// holds (infinities and NaN included). The sum is formed in float32 and rounded once.
//
// Bound by memory: 16,384 x 4,096 in bf16 70-71 us with a residual (5.7 TB/s), 56-57 us without; the generator's 20 wide products a
// block of four elements run beside the loads.
#include "fc_node.h"

namespace fc {

// floor(p 2^32) takes 33 bits at p = 1.
struct DropoutArgs {
  int64_t n;
  const void* x;
  const void* residual;
  const int64_t* rng;
  void* out;
  uint64_t threshold;
  float factor;
  int64_t first;  // block of this launch
};

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c[0] * 0xD2511F53u, p1 = (uint64_t)c[2] * 0xCD9E8D57u;
    c[0] = (uint32_t)(p1 >> 32) ^ c[1] ^ k0;
    c[1] = (uint32_t)p1;
    c[2] = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[3] = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// A thread takes 16 bytes of each stream: one block of the generator for four float32, two for eight 16-bit elements.
template <class T, bool RESIDUAL, bool ALL>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs g) {
  constexpr int V = 16 / sizeof(T);
  const int64_t e0 = ((g.first + blockIdx.x) * 256 + threadIdx.x) * V;
  if (e0 >= g.n) return;
  const T* x = (const T*)g.x + e0;
  const T* res = (const T*)g.residual + (RESIDUAL ? e0 : 0);
  T* out = (T*)g.out + e0;
  bool keep[V];
  if constexpr (ALL) {
#pragma unroll
    for (int i = 0; i < V; ++i) keep[i] = true;
  } else {
    const uint64_t seed = (uint64_t)g.rng[0], offset = (uint64_t)g.rng[1];
#pragma unroll
    for (int b = 0; b < V / 4; ++b) {
      const uint64_t block = (uint64_t)e0 / 4 + b;
      uint32_t c[4] = {(uint32_t)block, (uint32_t)(block >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
      philox(c, (uint32_t)seed, (uint32_t)(seed >> 32));
#pragma unroll
      for (int i = 0; i < 4; ++i) keep[4 * b + i] = c[i] >= g.threshold;
    }
  }
  if (e0 + V <= g.n) {
    const Pack<T, V> xv = load_pack<T, V>(x);
    Pack<T, V> rv, ov;
    if constexpr (RESIDUAL) rv = load_pack<T, V>(res);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float kept = keep[i] ? to_f32(xv.v[i]) * g.factor : 0.f;
      ov.v[i] = from_f32<T>(RESIDUAL ? kept + to_f32(rv.v[i]) : kept);
    }
    store_pack<T, V>(out, ov);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e0 + i < g.n) {
      const float kept = keep[i] ? to_f32(x[i]) * g.factor : 0.f;
      out[i] = from_f32<T>(RESIDUAL ? kept + to_f32(res[i]) : kept);
    }
}

}  // namespace fc

using namespace fc;

extern "C" int fc_dropout_add(int32_t dtype, int64_t n, const void* x, const void* residual, double p,
                              const int64_t* rng, void* out, void* stream) {
  if (!node_dtype_ok(dtype) || !(p >= 0.0 && p <= 1.0)) return FC_ERR_BAD_DESC;
  if (n < 0) return FC_ERR_SHAPE;
  if (n == 0) return FC_OK;
  if (!x || !rng || !out) return FC_ERR_NULL;
  DropoutArgs g{n, x, residual, rng, out, (uint64_t)(p * 4294967296.0), (float)(1.0 / (1.0 - p)), 0};
  if (n > INT64_MAX / 8) return FC_ERR_SHAPE;
  const int64_t blocks = (n * node_dtype_size(dtype) + 4095) / 4096;
  const dim3 block(256);
  hipStream_t s = (hipStream_t)stream;
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const bool all = g.threshold == 0;
    return in_launches(blocks, [&](int64_t first, unsigned grid) {
      g.first = first;
      if (residual && all) hipLaunchKernelGGL((dropout_kernel<T, true, true>), dim3(grid), block, 0, s, g);
      else if (residual) hipLaunchKernelGGL((dropout_kernel<T, true, false>), dim3(grid), block, 0, s, g);
      else if (all) hipLaunchKernelGGL((dropout_kernel<T, false, true>), dim3(grid), block, 0, s, g);
      else hipLaunchKernelGGL((dropout_kernel<T, false, false>), dim3(grid), block, 0, s, g);
    });
  });
}
