// Root-mean-square norm of rows with the residual's addition: total = x + residual in the tensors' type,
//   y = w total r,  r = 1 / sqrt(mean(total^2) + eps),
// y being the norm of the total as it is stored, so that the backward pass, which reads the stored total, differentiates what
// was computed. With xhat = r total and g the gradient of y
//   dx = g_total + r (w g - xhat mean(w g xhat)),  dw = sum over the rows of g xhat.
// In 8 bits y is written as round(y / s) in e4m3 with s = max(|y|, 2^-100) / 448 for each row. r has no part in the quotient
// y / s = 448 t w / max|t w|, in which 16-bit values often lie on a midpoint of two e4m3 numbers (1 in 8,000): it is formed from
// the products without r, rounded once, so that these go to the even number as they should.
//
// Bound by memory: every tensor is read or written once. A row is held in registers by a group of 16, 64 or 256 lanes, 16
// bytes a lane and load; squares, means and dw are summed in float32. dw: a workgroup adds up the rows it takes, in
// registers, and a second launch adds the workgroups' sums: a fixed order. Rows too wide for that (above 16,384 16-bit or
// 8,192 float32 elements; half as many backward) are read again instead. 16,384 x 4,096 bf16 with a residual: forward 86 us
// (6.2 TB/s), backward 115 + 5 (4.7 TB/s); 8,192 x 5,120 to 8 bits 52 us (5.6 TB/s), its rows alone 20; 25,000 x 128 float32 10 and 12 + 4 us;
// one row of 4,096 3 us.
#include "fc_node.h"

namespace fc {

struct RowNorm {
  const void *x, *residual, *weight;
  void *total, *y;
  float *rstd, *scale;
  int64_t n, width, first;  // first: block of this launch
  float eps;
};

template <class T>
constexpr int kChunk = 16 / sizeof(T);  // elements of a load

// 16 bytes of a row, as they are loaded.
struct Chunk {
  uint32_t w[4];
};

// The elements c .. c + 15 / sizeof(T) of a row, zeros past its end. EVEN: rows of whole chunks (the code for parts of a
// chunk costs registers: forward 143 us instead of 107).
template <class T, bool EVEN>
__device__ __forceinline__ Chunk load_chunk(const T* row, int64_t c, int64_t width) {
  constexpr int V = kChunk<T>;
  Chunk q;
  if (EVEN || c + V <= width) {
    memcpy(&q, row + c, 16);
    return q;
  }
  T e[V];
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = c + i < width ? row[c + i] : T{};
  memcpy(&q, e, 16);
  return q;
}
template <class E, int BYTES, bool EVEN>
__device__ __forceinline__ void store_chunk(E* row, int64_t c, int64_t width, const void* from) {
  constexpr int V = BYTES / sizeof(E);
  if (EVEN || c + V <= width) {
    memcpy(row + c, from, BYTES);
    return;
  }
  E e[V];
  memcpy(e, from, BYTES);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (c + i < width) row[c + i] = e[i];
}
template <class T>
__device__ __forceinline__ void unpack(const Chunk& q, float (&x)[kChunk<T>]) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(q.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, bf16_t>) {
        x[2 * i] = __uint_as_float(q.w[i] << 16);
        x[2 * i + 1] = __uint_as_float(q.w[i] & 0xffff0000u);
      } else {
        x[2 * i] = to_f32(f16_t{(uint16_t)q.w[i]});
        x[2 * i + 1] = to_f32(f16_t{(uint16_t)(q.w[i] >> 16)});
      }
    }
  }
}
// Rounded to nearest even.
template <class T>
__device__ __forceinline__ Chunk pack(const float (&x)[kChunk<T>]) {
  Chunk q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      q.w[i] = __float_as_uint(x[i]);
    } else if constexpr (std::is_same_v<T, f16_t>) {
      q.w[i] = from_f32<f16_t>(x[2 * i]).v | (uint32_t)from_f32<f16_t>(x[2 * i + 1]).v << 16;
    } else {
      asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(q.w[i]) : "v"(x[2 * i]), "v"(x[2 * i + 1]));
    }
  }
  return q;
}

// A sum, or largest value, over the L lanes of a row; every lane gets it. Called by all threads of a workgroup of NT.
template <int L, int NT, bool MAX>
__device__ __forceinline__ float over_row(float v, float* lds) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o > 0; o /= 2) {
    const float w = __shfl_xor(v, o, 64);
    v = MAX ? fmaxf(v, w) : v + w;
  }
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    const int wave = threadIdx.x / 64;
    __syncthreads();  // (the last call's values have been read)
    if (threadIdx.x % 64 == 0) lds[wave] = v;
    __syncthreads();
    const int w0 = wave / W * W;
    v = lds[w0];
#pragma unroll
    for (int k = 1; k < W; ++k) v = MAX ? fmaxf(v, lds[w0 + k]) : v + lds[w0 + k];
  }
  return v;
}

// r = power * rest with power of two `power`, rest in [1, 2): values times `power` have no rounding that others had not. (0,
// infinity and NaN are their own power.)
__device__ __forceinline__ float power_of(float r, float& rest) {
  const uint32_t u = __float_as_uint(r);
  rest = __uint_as_float((u & 0x007fffffu) | 0x3f800000u);
  return r == r ? __uint_as_float(u & 0x7f800000u) : r;
}

// How a row goes to 8 bits whose largest |x| is `most`, its values being rest x: scale = max(rest most, 2^-100) / 448, and
// rest x / scale = x num / den, with num / den = 448 / most unless the least scale or an infinity stands in its place. No
// quotient is above 448; with an infinite scale the finite ones are zero and the others NaN.
struct RowEight {
  float scale, num, den, inv;
  __device__ __forceinline__ RowEight(float most, float rest) {
    const float top = rest * most;
    scale = fmaxf(top, 0x1p-100f) / 448.f;
    const bool finite = top < __builtin_inff(), plain = top >= 0x1p-100f && finite;
    num = plain ? 0.875f : rest;  // (448 / 2^9)
    den = plain ? 0x1p-9f * most : finite ? scale : 1.f;
    inv = finite ? 1.f / den : 0.f;
  }
  // The quotient, rounded once: an estimate, and what is left of it. LONG: with what x num loses, which has no more than 24
  // bits for bfloat16 products and for 16-bit values alone (and float32's is rounded, as its products are).
  template <bool LONG>
  __device__ __forceinline__ float of(float x) const {
    const float n = x * num, q = n * inv;
    float left = fmaf(-q, den, n);
    if constexpr (LONG) left += fmaf(x, num, -n);
    return fmaf(left, inv, q);
  }
};

// e4m3 numbers of V values of a row, to nearest even.
template <bool LONG, int V>
__device__ __forceinline__ Pack<uint8_t, V> to_e4m3(const float (&x)[V], const RowEight& e) {
  Pack<uint8_t, V> p;
  uint32_t w[V / 4];
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const int u = __builtin_amdgcn_cvt_pk_fp8_f32(e.of<LONG>(x[i]), e.of<LONG>(x[i + 1]), 0, false);
    w[i / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e.of<LONG>(x[i + 2]), e.of<LONG>(x[i + 3]), u, true);
  }
  memcpy(&p, w, V);
  return p;
}

enum { NORM = 0, NORM_EIGHT = 1, ROW_EIGHT = 2 };

// L lanes a row, K chunks a lane.
template <class T, int L, int K, int MODE, bool EVEN>
__global__ void __launch_bounds__(256) row_norm_fwd_kernel(RowNorm g) {
  constexpr int V = kChunk<T>, R = 256 / L;
  __shared__ float lds[4];
  const int lane = threadIdx.x % L;
  const int64_t row = (g.first + blockIdx.x) * R + threadIdx.x / L, at = row * g.width;
  const bool on = row < g.n;
  float t[K][V];
  float sum = 0.f;
  Chunk xp[K], rp[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = ((int64_t)k * L + lane) * V;
    xp[k] = rp[k] = Chunk{};
    if (on && c < g.width) {
      xp[k] = load_chunk<T, EVEN>((const T*)g.x + at, c, g.width);
      if (g.residual) rp[k] = load_chunk<T, EVEN>((const T*)g.residual + at, c, g.width);
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = ((int64_t)k * L + lane) * V;
    unpack<T>(xp[k], t[k]);
    if (g.residual) {
      float r[V];
      unpack<T>(rp[k], r);
#pragma unroll
      for (int i = 0; i < V; ++i) t[k][i] += r[i];
      const Chunk stored = pack<T>(t[k]);
      unpack<T>(stored, t[k]);
      if (on && c < g.width) store_chunk<T, 16, EVEN>((T*)g.total + at, c, g.width, &stored);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fmaf(t[k][i], t[k][i], sum);
  }
  float rest = 1.f;
  if constexpr (MODE != ROW_EIGHT) {
    float r = 1.f / sqrtf(over_row<L, 256, false>(sum, lds) / (float)g.width + g.eps);
    if (g.rstd && on && lane == 0) g.rstd[row] = r;
    if constexpr (MODE == NORM_EIGHT) r = power_of(r, rest);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = ((int64_t)k * L + lane) * V;
      if (g.weight) {
        float w[V];
        unpack<T>(c < g.width ? load_chunk<T, EVEN>((const T*)g.weight, c, g.width) : Chunk{}, w);
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] *= r * w[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] *= r;
      }
    }
  }
  if constexpr (MODE == NORM) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = ((int64_t)k * L + lane) * V;
      const Chunk o = pack<T>(t[k]);
      if (on && c < g.width) store_chunk<T, 16, EVEN>((T*)g.y + at, c, g.width, &o);
    }
  } else {
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) most = fmaxf(most, fabsf(t[k][i]));
    const RowEight eight(over_row<L, 256, true>(most, lds), rest);
    if (on && lane == 0) g.scale[row] = eight.scale;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = ((int64_t)k * L + lane) * V;
      const Pack<uint8_t, V> o = to_e4m3<std::is_same_v<T, f16_t> && MODE == NORM_EIGHT>(t[k], eight);
      if (on && c < g.width) store_chunk<uint8_t, V, EVEN>((uint8_t*)g.y + at, c, g.width, &o);
    }
  }
}

// Rows of any width, a workgroup each: the row is read once for each step.
template <class T, int MODE>
__global__ void __launch_bounds__(1024) row_norm_wide_kernel(RowNorm g) {
  constexpr int V = kChunk<T>, NT = 1024;
  __shared__ float lds[NT / 64];
  const int64_t row = g.first + blockIdx.x, at = row * g.width;
  const T* const x = (const T*)g.x + at;
  const T* const t = g.residual ? (const T*)g.total + at : x;
  float r = 1.f, rest = 1.f;
  if (MODE != ROW_EIGHT) {
    float sum = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < g.width; c += NT * V) {
      float v[V];
      unpack<T>(load_chunk<T, false>(x, c, g.width), v);
      if (g.residual) {
        float q[V];
        unpack<T>(load_chunk<T, false>((const T*)g.residual + at, c, g.width), q);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += q[i];
        const Chunk stored = pack<T>(v);
        unpack<T>(stored, v);
        store_chunk<T, 16, false>((T*)g.total + at, c, g.width, &stored);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum = fmaf(v[i], v[i], sum);
    }
    r = 1.f / sqrtf(over_row<NT, NT, false>(sum, lds) / (float)g.width + g.eps);
    if (g.rstd && threadIdx.x == 0) g.rstd[row] = r;
    if constexpr (MODE == NORM_EIGHT) r = power_of(r, rest);
  }
  // (a thread reads back the elements that it wrote)
  auto values = [&](int64_t c, float (&v)[V]) {
    float w[V];
    unpack<T>(load_chunk<T, false>(t, c, g.width), v);
    if (g.weight) unpack<T>(load_chunk<T, false>((const T*)g.weight, c, g.width), w);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= g.weight ? r * w[i] : r;
  };
  if constexpr (MODE == NORM) {
    for (int64_t c = (int64_t)threadIdx.x * V; c < g.width; c += NT * V) {
      float v[V];
      values(c, v);
      const Chunk o = pack<T>(v);
      store_chunk<T, 16, false>((T*)g.y + at, c, g.width, &o);
    }
  } else {
    float most = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < g.width; c += NT * V) {
      float v[V];
      values(c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) most = fmaxf(most, fabsf(v[i]));
    }
    const RowEight eight(over_row<NT, NT, true>(most, lds), rest);
    if (threadIdx.x == 0) g.scale[row] = eight.scale;
    for (int64_t c = (int64_t)threadIdx.x * V; c < g.width; c += NT * V) {
      float v[V];
      values(c, v);
      const Pack<uint8_t, V> o = to_e4m3<std::is_same_v<T, f16_t> && MODE == NORM_EIGHT>(v, eight);
      store_chunk<uint8_t, V, false>((uint8_t*)g.y + at, c, g.width, &o);
    }
  }
}

struct RowNormBwd {
  const void *grad, *grad_total, *total, *weight;
  const float* rstd;
  void* dx;     // or null
  float* sums;  // (blocks, width), or null
  void* dw;     // one workgroup writes it itself
  int64_t n, width;
};

template <class T, int L, int K, bool EVEN>
__global__ void __launch_bounds__(256) row_norm_bwd_kernel(RowNormBwd g) {
  constexpr int V = kChunk<T>, R = 256 / L;
  __shared__ float lds[4];
  __shared__ float part[R > 1 ? 256 * V : 1];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  float dw[K][V];
  Chunk wp[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = ((int64_t)k * L + lane) * V;
    wp[k] = Chunk{};
    if (g.weight && c < g.width) wp[k] = load_chunk<T, EVEN>((const T*)g.weight, c, g.width);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
  }
  for (int64_t first = (int64_t)blockIdx.x * R; first < g.n; first += (int64_t)gridDim.x * R) {
    const int64_t row = first + group, at = row * g.width;
    const bool on = row < g.n;
    Chunk gp[K], tp[K], ap[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = ((int64_t)k * L + lane) * V;
      gp[k] = tp[k] = ap[k] = Chunk{};
      if (on && c < g.width) {
        gp[k] = load_chunk<T, EVEN>((const T*)g.grad + at, c, g.width);
        tp[k] = load_chunk<T, EVEN>((const T*)g.total + at, c, g.width);
        if (g.grad_total && g.dx) ap[k] = load_chunk<T, EVEN>((const T*)g.grad_total + at, c, g.width);
      }
    }
    const float r = on ? g.rstd[row] : 0.f;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float q[V], t[V], w[V];
      unpack<T>(gp[k], q);
      unpack<T>(tp[k], t);
      unpack<T>(wp[k], w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float p = q[i] * (r * t[i]);
        dw[k][i] += p;
        sum = g.weight ? fmaf(p, w[i], sum) : sum + p;
      }
    }
    if (!g.dx) continue;
    const float mean = over_row<L, 256, false>(sum, lds) / (float)g.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = ((int64_t)k * L + lane) * V;
      float q[V], t[V], w[V], a[V];
      unpack<T>(gp[k], q);
      unpack<T>(tp[k], t);
      unpack<T>(wp[k], w);
      unpack<T>(ap[k], a);
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = fmaf(r, (g.weight ? q[i] * w[i] : q[i]) - (r * t[i]) * mean, a[i]);
      const Chunk o = pack<T>(a);
      if (on && c < g.width) store_chunk<T, 16, EVEN>((T*)g.dx + at, c, g.width, &o);
    }
  }
  if (!g.sums) return;
  float* const out = g.sums + (int64_t)blockIdx.x * g.width;
  const bool alone = gridDim.x == 1;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = ((int64_t)k * L + lane) * V;
    if constexpr (R > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) part[threadIdx.x * V + i] = dw[k][i];
      __syncthreads();
      if (group > 0) continue;
      for (int q = 1; q < R; ++q)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] += part[(q * L + lane) * V + i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (c + i >= g.width) continue;
      if (alone) ((T*)g.dw)[c + i] = from_f32<T>(dw[k][i]);
      else out[c + i] = dw[k][i];
    }
  }
}

template <class T>
__global__ void __launch_bounds__(1024) row_norm_wide_bwd_kernel(RowNormBwd g) {
  constexpr int V = kChunk<T>, NT = 1024;
  __shared__ float lds[NT / 64];
  float* const out = g.sums ? g.sums + (int64_t)blockIdx.x * g.width : nullptr;
  for (int64_t row = blockIdx.x; row < g.n; row += gridDim.x) {
    const int64_t at = row * g.width;
    const T *const grad = (const T*)g.grad + at, *const total = (const T*)g.total + at;
    const float r = g.rstd[row];
    float sum = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < g.width; c += NT * V) {
      float q[V], t[V], w[V];
      unpack<T>(load_chunk<T, false>(grad, c, g.width), q);
      unpack<T>(load_chunk<T, false>(total, c, g.width), t);
      if (g.weight) unpack<T>(load_chunk<T, false>((const T*)g.weight, c, g.width), w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float p = q[i] * (r * t[i]);
        sum = g.weight ? fmaf(p, w[i], sum) : sum + p;
        if (out && c + i < g.width) out[c + i] = row == blockIdx.x ? p : out[c + i] + p;
      }
    }
    if (!g.dx) continue;
    const float mean = over_row<NT, NT, false>(sum, lds) / (float)g.width;
    for (int64_t c = (int64_t)threadIdx.x * V; c < g.width; c += NT * V) {
      float q[V], t[V], w[V], a[V] = {};
      unpack<T>(load_chunk<T, false>(grad, c, g.width), q);
      unpack<T>(load_chunk<T, false>(total, c, g.width), t);
      if (g.weight) unpack<T>(load_chunk<T, false>((const T*)g.weight, c, g.width), w);
      if (g.grad_total) unpack<T>(load_chunk<T, false>((const T*)g.grad_total + at, c, g.width), a);
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = fmaf(r, (g.weight ? q[i] * w[i] : q[i]) - (r * t[i]) * mean, a[i]);
      const Chunk o = pack<T>(a);
      store_chunk<T, 16, false>((T*)g.dx + at, c, g.width, &o);
    }
  }
}

// The workgroups' sums added up: 32 columns by 32 lanes that take every 32nd row.
template <class T>
__global__ void __launch_bounds__(1024) row_norm_dw_kernel(const float* sums, int64_t rows, int64_t width, T* out) {
  __shared__ float part[32][33];
  const int cl = threadIdx.x % 32, grp = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + cl;
  float s = 0.f;
  if (c < width) {
#pragma unroll 8
    for (int64_t k = grp; k < rows; k += 32) s += sums[k * width + c];
  }
  part[grp][cl] = s;
  __syncthreads();
  if (grp > 0 || c >= width) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) s += part[k][cl];
  out[c] = from_f32<T>(s);
}

// f(lanes of a row, chunks of a lane, whole chunks) for rows of so many elements, V a chunk; false where they do not fit into
// registers. `most`: chunks of a lane up to which no more lanes are taken. (16,384 x 4,096 bf16 forward: 2 and 4 86 us, 8 101.)
template <int V, int MOST, class F>
static bool with_row(int64_t width, int64_t most, F&& f) {
  const int64_t chunks = (width + V - 1) / V;
  auto lanes = [&](auto l) {
    constexpr int L = decltype(l)::value;
    const int64_t k = (chunks + L - 1) / L;
    if (width % V != 0) {
      if (k <= 2) f(l, std::integral_constant<int, 2>{}, std::false_type{});
      else f(l, std::integral_constant<int, MOST>{}, std::false_type{});
    } else if (k <= 1) {
      f(l, std::integral_constant<int, 1>{}, std::true_type{});
    } else if (k <= 2) {
      f(l, std::integral_constant<int, 2>{}, std::true_type{});
    } else if (k <= 4) {
      f(l, std::integral_constant<int, 4>{}, std::true_type{});
    } else {
      f(l, std::integral_constant<int, MOST>{}, std::true_type{});
    }
  };
  if (chunks > 256 * MOST) return false;
  if (chunks <= 16 * most) lanes(std::integral_constant<int, 16>{});
  else if (chunks <= 64 * most) lanes(std::integral_constant<int, 64>{});
  else lanes(std::integral_constant<int, 256>{});
  return true;
}

static int row_norm_check(int32_t dtype, int64_t n, int64_t width) {
  if (!node_dtype_ok(dtype)) return FC_ERR_BAD_DESC;
  return n < 0 || n > 0x7fffffff || width < 1 || width > (1 << 20) ? FC_ERR_SHAPE : FC_OK;
}

template <int MODE>
static int run_fwd(int32_t dtype, RowNorm g, hipStream_t s) {
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    int st = FC_OK;
    const bool fits = with_row<kChunk<T>, 8>(g.width, 4, [&](auto l, auto k, auto even) {
      constexpr int L = decltype(l)::value, K = decltype(k)::value;
      st = in_launches((g.n + 256 / L - 1) / (256 / L), [&](int64_t first, unsigned grid) {
        g.first = first;
        hipLaunchKernelGGL((row_norm_fwd_kernel<T, L, K, MODE, decltype(even)::value>), dim3(grid), dim3(256), 0, s, g);
      });
    });
    if (fits) return st;
    return in_launches(g.n, [&](int64_t first, unsigned grid) {
      g.first = first;
      hipLaunchKernelGGL((row_norm_wide_kernel<T, MODE>), dim3(grid), dim3(1024), 0, s, g);
    });
  });
}

// Workgroups of a backward pass with dw: each adds a row to the second launch. (16,384 x 4,096 bf16: 512 115 us and 5 for the
// second launch, 1,024 118 and 5, 2,048 117 and 10.)
static int64_t bwd_blocks(int64_t n) { return n < 512 ? n : 512; }

}  // namespace fc

using namespace fc;

extern "C" int fc_row_norm_fwd(int32_t dtype, int64_t n, int64_t width, const void* x, const void* residual,
                               const void* weight, float eps, void* total, void* y, float* rstd, void* stream) {
  const int st = row_norm_check(dtype, n, width);
  if (st != FC_OK) return st;
  if (n == 0) return FC_OK;
  if (!x || !y || (residual && !total)) return FC_ERR_NULL;
  return run_fwd<NORM>(dtype, RowNorm{x, residual, weight, total, y, rstd, nullptr, n, width, 0, eps}, (hipStream_t)stream);
}

extern "C" int fc_row_norm_quantize(int32_t dtype, int32_t norm, int64_t n, int64_t width, const void* x,
                                    const void* residual, const void* weight, float eps, void* total, void* q,
                                    float* scale, void* stream) {
  const int st = row_norm_check(dtype, n, width);
  if (st != FC_OK) return st;
  if (!norm && (residual || weight)) return FC_ERR_BAD_DESC;
  if (n == 0) return FC_OK;
  if (!x || !q || !scale || (residual && !total)) return FC_ERR_NULL;
  const RowNorm g{x, residual, weight, total, q, nullptr, scale, n, width, 0, eps};
  return norm ? run_fwd<NORM_EIGHT>(dtype, g, (hipStream_t)stream) : run_fwd<ROW_EIGHT>(dtype, g, (hipStream_t)stream);
}

extern "C" int64_t fc_row_norm_bwd_workspace(int32_t dtype, int64_t n, int64_t width, int32_t need_weight) {
  const int st = row_norm_check(dtype, n, width);
  if (st != FC_OK) return -st;
  return need_weight ? 4 * bwd_blocks(n) * width : 0;
}

extern "C" int fc_row_norm_bwd(int32_t dtype, int64_t n, int64_t width, const void* grad, const void* grad_total,
                               const void* total, const void* weight, const float* rstd, void* grad_x, void* grad_weight,
                               void* ws, int64_t ws_bytes, void* stream) {
  const int st = row_norm_check(dtype, n, width);
  if (st != FC_OK) return st;
  if (!grad_x && !grad_weight) return FC_OK;
  if (n == 0) return grad_weight ? FC_ERR_SHAPE : FC_OK;
  if (!grad || !total || !rstd) return FC_ERR_NULL;
  const int64_t need = grad_weight ? 4 * bwd_blocks(n) * width : 0;
  if (need > 0 && (!ws || ws_bytes < need || ((uintptr_t)ws & 15))) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const RowNormBwd g{grad, grad_total, total, weight, rstd, grad_x, grad_weight ? (float*)ws : nullptr, grad_weight, n, width};
    int64_t blocks = 0;
    const bool fits = with_row<kChunk<T>, 4>(width, 2, [&](auto l, auto k, auto even) {
      constexpr int L = decltype(l)::value, K = decltype(k)::value;
      blocks = (n + 256 / L - 1) / (256 / L);
      if (grad_weight) blocks = blocks <= 4 ? 1 : bwd_blocks(blocks);  // (few rows: no second launch)
      else if (blocks > kLaunchBlocks) blocks = kLaunchBlocks;
      hipLaunchKernelGGL((row_norm_bwd_kernel<T, L, K, decltype(even)::value>), dim3((unsigned)blocks), dim3(256), 0, s, g);
    });
    if (!fits) {
      blocks = bwd_blocks(n);
      hipLaunchKernelGGL((row_norm_wide_bwd_kernel<T>), dim3((unsigned)blocks), dim3(1024), 0, s, g);
    }
    FC_LAUNCH_CHECK();
    if (!grad_weight || (fits && blocks == 1)) return FC_OK;
    hipLaunchKernelGGL((row_norm_dw_kernel<T>), dim3((unsigned)((width + 31) / 32)), dim3(1024), 0, s, (const float*)ws,
                       blocks, width, (T*)grad_weight);
    FC_LAUNCH_CHECK();
    return FC_OK;
  });
}
