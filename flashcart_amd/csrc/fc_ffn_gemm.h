// Matrix products of the gated feed-forward block (included by fc_ffn.hip): D[m, n] = sum_k A(m, k) B(n, k) on the 16-bit
// matrix instructions with float32 accumulation, with the block's elementwise steps in the epilogues.
//
// Operands lie as (rows, K), or as (K, rows) ("TR"), so that no operand of the backward pass is transposed in memory.
// float32 has two forms. "Native": float32 operands on the float32 matrix instructions. "Planes", for large products: three
// bf16 planes (x = h + m + l, each the nearest bf16 of what the ones before it leave: the split is exact); the K loop then
// runs over the six plane pairs of relative size 1, 2^-8, 2^-16, smallest first, and what is left out is below 2^-24 of a
// product. A float32 result that comes out infinite or NaN is formed again from scaled operands, one product after the
// other: it follows the IEEE rules, and stays finite where only the unscaled sum does not.
//
// Tiles of BM x BN outputs and 64 k (32 in native float32), by waves of 16x16x32 (16x16x4) instructions. Both operand
// tiles go from memory to LDS without passing through registers, ahead of the products. Chunks of 16 bytes are permuted
// on the way so that the reads of the fragments spread over the banks (no conflicts counted): a (rows, 64) tile is read
// 16 bytes a lane, a (64, rows) tile by the transposing LDS read, whose group of 16 lanes takes 4 k x 16 rows and returns 4
// consecutive k of one row to each.
#pragma once

#include "fc_node.h"

namespace fc {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

// The products of two fragments: 32 k of 16-bit operands, 16 k of float32 ones (four instructions; in each, the lanes of a
// group of 16 take one k of their four).
template <class MT>
__device__ __forceinline__ f32x4v mfma16(const s16x8& a, const s16x8& b, f32x4v c) {
  if constexpr (std::is_same_v<MT, float>) {
    const f32x4v u = __builtin_bit_cast(f32x4v, a), v = __builtin_bit_cast(f32x4v, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(u[e], v[e], c, 0, 0, 0);
    return c;
  } else if constexpr (std::is_same_v<MT, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0,
                                                   0);
}

// One operand: `rows` output rows (or columns), k valid up to `k`; element (r, k) at p[r * ld + k], or p[k * ld + r].
// ld is a multiple of 8 and p is aligned to 16 bytes; in the TR form `rows` is a multiple of 8 too.
struct Opnd {
  const char* p;
  int64_t ld, plane;  // elements; plane: from one bf16 plane to the next
  int32_t rows, k;
};

enum { EPI_GATE = 0, EPI_OUT = 1, EPI_DH = 2 };

struct FfnJob {
  Opnd A, B;
  int32_t M, N;          // outputs; for EPI_GATE N is the hidden size of one half, padded to 8
  int32_t tiles_m, tiles_n, splits, steps;  // steps: of 64 k, over all planes; a split takes steps / splits of them
  int32_t a_tr, b_tr;    // forms of A and B
  int32_t finish;        // splits > 1: the epilogue that the sum of the parts goes through
  float scale;
  // EPI_OUT: out (., ld_out) of the operator's type; rows m >= gap_at are written gap rows earlier, rows in between not
  void* out;
  int64_t ld_out;
  int32_t n_out, m_out, gap_at, gap;
  float* partial;        // splits > 1: (splits, M, N)
  // EPI_GATE: h (n, N) and, in training, the factors a = c act(gate), b = c act'(gate) up; EPI_DH: a, b and dpre
  char* h;
  int64_t h_plane;
  void* saved;           // 16-bit types: (3, n, N) uint16; float32: (2, n, N) float
  char* dpre;            // (n, 2 N)
  int64_t dpre_plane;
  int32_t act;
  float act_scale;
};

constexpr uint32_t kOutOfRange = 0x7ffffff0u;  // byte offset that a buffer load answers with zeros

// Planes of the pair i: 0 2, 2 0, 1 1, 0 1, 1 0, 0 0, the smallest products first.
__device__ __forceinline__ void plane_pair(int i, int& a, int& b) {
  a = (0x010120 >> (4 * i)) & 15;
  b = (0x001102 >> (4 * i)) & 15;
}

// act(g) and its derivative; 0 silu, 1 sigmoid, 2 gelu (erf form). The exponential is that of base 2 of a rounded product,
// so its relative error is about 2^-24 (1 + |g|): all of it shows in silu and sigmoid where they vanish (g << 0), less and
// less for larger g.
__device__ __forceinline__ void ffn_act(int act, float g, float& f, float& d) {
  if (act == 2) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    f = g * cdf;
    d = cdf + g * __expf(-0.5f * g * g) * 0.3989422804014327f;
    return;
  }
  const float s = __builtin_amdgcn_rcpf(1.f + __expf(-g));
  f = act == 0 ? g * s : s;
  d = act == 0 ? s * (1.f + g * (1.f - s)) : s * (1.f - s);
}

template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM_ * WN_, NT = 64 * NW;
  static constexpr int TM = BM / WM, TN = BN / WN, MF = TM / 16, NF = TN / 16;
  static constexpr int STAGE = (BM + BN) * 128, STAGES = STAGES_;  // bytes of LDS a stage, stages
};

// The part of a wave in bringing one operand tile of R rows and 128 bytes of k to LDS: R / 8 segments of 1 KB, shared by the
// waves. ES: bytes of an element.
template <int R, int NW, int ES, bool TR>
struct Loader {
  static constexpr int SEGS = R / 8 / NW, CE = 16 / ES, KS = 128 / ES;  // elements of a chunk, k of a step
  static_assert(R % (8 * NW) == 0, "segments");
  const char* base[SEGS];
  uint32_t off[SEGS];
  int kl[TR ? SEGS : 1];  // k of the lane's chunk, counted from the step's first

  // Where 16 bytes of row k are in a (K, rows) tile: how `c`, the index of 32 (float32: 64) bytes of the row, is permuted.
  __device__ static __forceinline__ int permute(int k, int c) {
    if constexpr (ES == 4) return c ^ ((k >> 2) & 3);
    else return c ^ (R >= 128 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2));
  }

  // HALF > 0: rows r with r % (2 HALF) >= HALF come from `up` rows further on (gate and up rows of one weight)
  template <int HALF>
  __device__ __forceinline__ void init(const Opnd& o, int r0, int wave, int lane, int up) {
#pragma unroll
    for (int j = 0; j < SEGS; ++j) {
      const int seg = wave + NW * j;
      if constexpr (!TR) {
        int row = seg * 8 + (lane >> 3);
        int64_t first = r0;
        if constexpr (HALF > 0) {
          const bool second = (seg * 8) % (2 * HALF) >= HALF;
          row = row / (2 * HALF) * HALF + row % HALF;
          if (second) first += up;
        }
        base[j] = o.p + ES * first * o.ld;
        row = min(row, o.rows - 1 - r0);
        off[j] = (uint32_t)row * (uint32_t)(o.ld * ES) + 16 * ((lane & 7) ^ (lane >> 3));
        kl[0] = CE * ((lane & 7) ^ (lane >> 3));
      } else {
        constexpr int CPR = R / CE, CPP = ES == 4 ? 4 : 2;  // chunks of a row, and of what is permuted as one
        const int k = seg * (64 / CPR) + lane / CPR, phys = lane % CPR;
        const int col = min(r0 + CE * (permute(k, phys / CPP) * CPP + phys % CPP), o.rows - CE);
        base[j] = o.p;
        off[j] = (uint32_t)k * (uint32_t)(o.ld * ES) + ES * col;
        kl[j] = k;
      }
    }
  }
  // the step at k0 of the plane that starts `plane` elements behind the first; the segments of the wave in MASK
  template <int MASK>
  __device__ __forceinline__ void load(const Opnd& o, int k0, int64_t plane, lds_char* dst, int wave) const {
    const int64_t shift = ES * (plane + (TR ? (int64_t)k0 * o.ld : k0));
    const int left = o.k - k0;
#pragma unroll
    for (int j = 0; j < SEGS; ++j) {
      if (!(MASK >> j & 1)) continue;
      __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base[j] + shift), 0, kOutOfRange, 0x00020000);
      const uint32_t at = (left >= KS || kl[TR ? j : 0] < left) ? off[j] : kOutOfRange;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + (wave + NW * j) * 1024),
                                               16, at, 0, 0, 0);
    }
  }
};

// Fragments of a wave: F blocks of 16 rows from row `r0` of an operand tile of R rows; s: which half of the step's k.
template <int R, int F, int ES, bool TR>
struct Reader {
  uint32_t at[TR ? F : 2];
  __device__ __forceinline__ void init(int r0, int lane) {
    const int g = lane >> 4, r = lane & 15;
    if constexpr (!TR) {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (r0 + r) * 128 + 16 * ((4 * s + g) ^ (r & 7));
    } else if constexpr (ES == 4) {
      const int k = 4 * g;
#pragma unroll
      for (int j = 0; j < F; ++j) at[j] = k * (R * 4) + Loader<R, 1, ES, TR>::permute(k, (r0 >> 4) + j) * 64 + r * 4;
    } else {
      const int k = 8 * g + (r >> 2);
#pragma unroll
      for (int j = 0; j < F; ++j) at[j] = k * (R * 2) + Loader<R, 1, ES, TR>::permute(k, (r0 >> 4) + j) * 32 + (r & 3) * 8;
    }
  }
  // C of the blocks, from block J on
  template <int J, int C>
  __device__ __forceinline__ void read(const lds_char* tile, int s, s16x8 (&x)[C]) const {
#pragma unroll
    for (int j = J; j < J + C; ++j) {
      if constexpr (!TR) {
        x[j - J] = *(const __attribute__((address_space(3))) s16x8*)(tile + at[s] + j * 16 * 128);
      } else if constexpr (ES == 4) {
        const lds_char* p = tile + at[j] + s * 16 * (R * 4);
        f32x4v v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = *(const __attribute__((address_space(3))) float*)(p + e * (R * 4));
        x[j - J] = __builtin_bit_cast(s16x8, v);
      } else {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const lds_char* p = tile + at[j] + s * 32 * (R * 2);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        // k + 4: for R = 64 bit 1 of k is as before, bit 2 is not part of the permutation
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * (R * 2)));
        x[j - J] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  }
};

// Two values of the 16-bit type, round to nearest even, a in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, f16_t>) {
    return from_f32<f16_t>(a).v | (uint32_t)from_f32<f16_t>(b).v << 16;
  } else {
    uint32_t u;
    asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(u) : "v"(a), "v"(b));
    return u;
  }
}

// Three bf16 numbers whose sum is x. What rounds to infinity is cut off instead, so that only an infinite or NaN x has
// parts that are not finite, and its other parts are zero.
__device__ __forceinline__ void split3(float x, uint16_t& h, uint16_t& m, uint16_t& l) {
  h = from_f32<bf16_t>(x).v;
  if ((h & 0x7fff) == 0x7f80) h = (uint16_t)(__float_as_uint(x) >> 16);
  const float r = (h & 0x7f80) == 0x7f80 ? 0.f : x - to_f32(bf16_t{h});
  m = from_f32<bf16_t>(r).v;
  l = from_f32<bf16_t>(r - to_f32(bf16_t{m})).v;
}

// V (4 or 8) consecutive 16-bit values.
template <int V>
__device__ __forceinline__ void put_words(void* p, const uint32_t (&x)[V / 2]) {
  if constexpr (V == 8) *(uint4*)p = make_uint4(x[0], x[1], x[2], x[3]);
  else *(uint2*)p = make_uint2(x[0], x[1]);
}
template <int V>
__device__ __forceinline__ void put_floats(float* p, const float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) *(float4*)(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}

// V consecutive values, from element `at` on, of a matrix in the operator's operand form.
template <class MT, bool F32, int V>
__device__ __forceinline__ void put(char* matrix, int64_t at, int64_t plane, const float (&x)[V]) {
  if constexpr (std::is_same_v<MT, float>) {
    put_floats((float*)matrix + at, x);
  } else if constexpr (!F32) {
    uint32_t u[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) u[i] = pack2<MT>(x[2 * i], x[2 * i + 1]);
    put_words<V>(matrix + 2 * at, u);
  } else {
    uint32_t h[V / 2], m[V / 2], l[V / 2];
    float most = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      most = fmaxf(most, fabsf(x[i]));
      sum = fmaf(x[i], 0.f, sum);
    }
    if (most < 0x1.fep127f && sum == 0.f) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        h[i] = pack2<bf16_t>(a, b);
        const float ra = a - __uint_as_float(h[i] << 16), rb = b - __uint_as_float(h[i] & 0xffff0000u);
        m[i] = pack2<bf16_t>(ra, rb);
        l[i] = pack2<bf16_t>(ra - __uint_as_float(m[i] << 16), rb - __uint_as_float(m[i] & 0xffff0000u));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        uint16_t u[2], v[2], w[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) split3(x[2 * i + q], u[q], v[q], w[q]);
        h[i] = u[0] | (uint32_t)u[1] << 16;
        m[i] = v[0] | (uint32_t)v[1] << 16;
        l[i] = w[0] | (uint32_t)w[1] << 16;
      }
    }
    uint16_t* p = (uint16_t*)matrix + at;
    put_words<V>(p, h);
    put_words<V>(p + plane, m);
    put_words<V>(p + 2 * plane, l);
  }
}

// Factors kept for the backward pass. For 16-bit types they keep 24 bits (the upper half of a float32 and the next 8 bits
// of each of the pair in one more uint16), so that their rounding does not add to those of dpre and of the gradients.
// (v_perm_b32: bytes 0 to 3 are those of its second operand, 4 to 7 those of the first.)
template <bool F32, int V>
__device__ __forceinline__ void put_factors(void* saved, int64_t at, int64_t count, const float (&a)[V],
                                            const float (&b)[V]) {
  if constexpr (F32) {
    put_floats((float*)saved + at, a);
    put_floats((float*)saved + count + at, b);
  } else {
    uint32_t ah[V / 2], bh[V / 2], lo[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      // (infinite and NaN stay so: the lowest bits of such a value are zero)
      const uint32_t u0 = __float_as_uint(a[2 * i]) + 0x80, u1 = __float_as_uint(a[2 * i + 1]) + 0x80;
      const uint32_t v0 = __float_as_uint(b[2 * i]) + 0x80, v1 = __float_as_uint(b[2 * i + 1]) + 0x80;
      ah[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302);
      bh[i] = __builtin_amdgcn_perm(v1, v0, 0x07060302);
      lo[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(v1, u1, 0x0c0c0501), __builtin_amdgcn_perm(v0, u0, 0x0c0c0501),
                                    0x05040100);
    }
    uint16_t* p = (uint16_t*)saved + at;
    put_words<V>(p, ah);
    put_words<V>(p + count, bh);
    put_words<V>(p + 2 * count, lo);
  }
}
template <bool F32, int V>
struct Factors {
  uint32_t x[F32 ? 2 : 3][F32 ? V : V / 2];
  __device__ __forceinline__ void load(const void* saved, int64_t at, int64_t count) {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 3); ++i) {
      const uint32_t* p = (const uint32_t*)((const char*)saved + (F32 ? 4 : 2) * (at + i * count));
      constexpr int WORDS = sizeof(x[0]) / 4;
      if constexpr (WORDS == 2) {
        const uint2 v = *(const uint2*)p;
        x[i][0] = v.x;
        x[i][1] = v.y;
      } else {
#pragma unroll
        for (int k = 0; k < WORDS; k += 4) {
          const uint4 v = *(const uint4*)(p + k);
          x[i][k] = v.x;
          x[i][k + 1] = v.y;
          x[i][k + 2] = v.z;
          x[i][k + 3] = v.w;
        }
      }
    }
  }
  __device__ __forceinline__ void get(float (&a)[V], float (&b)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (F32) {
        a[i] = __uint_as_float(x[0][i]);
        b[i] = __uint_as_float(x[1][i]);
      } else {
        a[i] = __uint_as_float(__builtin_amdgcn_perm(x[0][i / 2], x[2][i / 2], i % 2 ? 0x0706020c : 0x0504000c));
        b[i] = __uint_as_float(__builtin_amdgcn_perm(x[1][i / 2], x[2][i / 2], i % 2 ? 0x0706030c : 0x0504010c));
      }
    }
  }
};

// The epilogues of the first products, for V columns from `col` on of row `row`; hp: columns of h, padded to 8; pad columns
// take part in the next product as zeros.
template <class MT, bool F32, int V>
__device__ __forceinline__ void finish_gate(const FfnJob& g, int64_t row, int col, int hp, const float (&gate)[V],
                                            const float (&up)[V]) {
  float a[V], b[V], h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float f, d;
    ffn_act(g.act, gate[v], f, d);
    a[v] = g.act_scale * f;
    b[v] = g.act_scale * d * up[v];
    h[v] = col + v < g.n_out ? a[v] * up[v] : 0.f;
  }
  const int64_t at = row * hp + col;
  put<MT, F32, V>(g.h, at, g.h_plane, h);
  if (g.saved) put_factors<F32, V>(g.saved, at, (int64_t)g.M * hp, a, b);
}
template <class MT, bool F32, int V>
__device__ __forceinline__ void finish_dh(const FfnJob& g, int64_t row, int col, const Factors<F32, V>& f,
                                          const float (&dh)[V]) {
  float a[V], b[V], dg[V], du[V];
  f.get(a, b);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    dg[v] = col + v < g.n_out ? dh[v] * b[v] : 0.f;
    du[v] = col + v < g.n_out ? dh[v] * a[v] : 0.f;
  }
  const int64_t at = row * 2 * g.N + col;
  put<MT, F32, V>(g.dpre, at, g.dpre_plane, dg);
  put<MT, F32, V>(g.dpre, at + g.N, g.dpre_plane, du);
}

// A float32 operand's value, native (ES = 4) or in planes.
template <int ES, bool TR>
__device__ __forceinline__ float value_of(const Opnd& o, int64_t r, int k) {
  if (k >= o.k) return 0.f;
  const int64_t at = TR ? (int64_t)k * o.ld + r : r * o.ld + k;
  if constexpr (ES == 4) return ((const float*)o.p)[at];
  const uint16_t* p = (const uint16_t*)o.p + at;
  return to_f32(bf16_t{p[0]}) + (to_f32(bf16_t{p[o.plane]}) + to_f32(bf16_t{p[2 * o.plane]}));
}

template <class T, class MT, bool F32, bool ATR, bool BTR, int EPI>
struct FfnTile {
  using OT = std::conditional_t<F32, float, MT>;
  static constexpr bool PLANES = F32 && !std::is_same_v<MT, float>;
  static constexpr int ES = std::is_same_v<MT, float> ? 4 : 2, KS = 128 / ES;

  __device__ static __forceinline__ void run(const FfnJob& g, int block, lds_char* lds0, lds_char* lds1, lds_char* lds2,
                                         lds_char* lds3) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / T::WN, wn = wave % T::WN;
    // block -> split, tile. Consecutive blocks go to the 8 XCDs in turn: each XCD takes a run of tiles, in groups of 8
    // tile rows, whose operands its L2 then serves.
    const int tiles = g.tiles_m * g.tiles_n;
    int split = 0, tile = block;
    if (g.splits > 1) {
      split = block / tiles;
      tile = block - split * tiles;
    }
    if (tiles >= 64) {
      const int per = tiles / 8, rest = tiles % 8, x = tile % 8;
      tile = x * per + min(x, rest) + tile / 8;
    }
    const int group = tile / (8 * g.tiles_n), in = tile - group * 8 * g.tiles_n;
    const int gm = min(8, g.tiles_m - group * 8);
    const int mt = group * 8 + in % gm, nt = in / gm;
    constexpr int BNO = EPI == EPI_GATE ? T::BN / 2 : T::BN;  // output columns of a tile
    const int m0 = mt * T::BM, n0 = nt * BNO;

    Loader<T::BM, T::NW, ES, ATR> la;
    Loader<T::BN, T::NW, ES, BTR> lb;
    la.template init<0>(g.A, m0, wave, lane, 0);
    lb.template init<EPI == EPI_GATE ? T::TN / 2 : 0>(g.B, n0, wave, lane, g.N);
    Reader<T::BM, T::MF, ES, ATR> ra;
    Reader<T::BN, T::NF, ES, BTR> rb;
    ra.init(wm * T::TM, lane);
    rb.init(wn * T::TN, lane);

    f32x4v acc[T::MF][T::NF];
#pragma unroll
    for (int i = 0; i < T::MF; ++i)
#pragma unroll
      for (int j = 0; j < T::NF; ++j) acc[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};

    const int s0 = __builtin_amdgcn_readfirstlane((int)((int64_t)g.steps * split / g.splits));
    const int s1 = __builtin_amdgcn_readfirstlane((int)((int64_t)g.steps * (split + 1) / g.splits));
    // Where the next load of some segments is: k, and the planes (float32: the pair, smallest products first).
    struct Cursor {
      int left, k, pair;  // left: steps before the end
      int64_t a, b;       // elements to the planes
    };
    const int per_pair = PLANES ? g.steps / 6 : g.steps;
    auto place = [&](Cursor& c) {
      if constexpr (PLANES) {
        int pa, pb;
        plane_pair(c.pair, pa, pb);
        // (in scalar registers: a buffer's base that the compiler takes for different in the lanes costs a loop a load)
        c.a = __builtin_amdgcn_readfirstlane(pa) * g.A.plane;
        c.b = __builtin_amdgcn_readfirstlane(pb) * g.B.plane;
      } else {
        c.a = c.b = 0;
      }
    };
    auto cursor_at = [&](int s) {
      Cursor c;
      c.left = s1 - s;
      c.pair = PLANES ? __builtin_amdgcn_readfirstlane(s / per_pair) : 0;
      c.k = KS * (s - c.pair * per_pair);
      place(c);
      return c;
    };
    // segments MA of A's tile and MB of B's at the cursor, zeros past the end; the cursor goes to the next step
    auto fetch = [&](Cursor& c, lds_char* at, auto ma, auto mb) {
      const int k = c.left > 0 ? c.k : KS * per_pair;
      la.template load<ma>(g.A, k, c.a, at, wave);
      lb.template load<mb>(g.B, k, c.b, at + T::BM * 128, wave);
      --c.left;
      c.k += KS;
      if constexpr (PLANES) {
        if (c.k == KS * per_pair) {
          c.k = 0;
          ++c.pair;
          place(c);
        }
      }
    };
    constexpr std::integral_constant<int, 15> all{};
    // The two LDS stages are separate arrays and every access names one of them, so that no read waits for the loads into
    // the other. As many steps as there are stages without a branch inside: steps past the end multiply zeros.
    if constexpr (T::NW == 8) {
      // Two waves of each SIMD take turns: one multiplies while the other reads LDS, then they change places at a
      // barrier. A step is two such phases. Where A is (rows, K), phase 1 reads the first half of the wave's rows and all
      // its columns and phase 2 the other rows; where A is (K, rows) the phases are the halves of the step's k. What
      // everyone has read in one phase is loaded again from the next phase on, for the step after next: a load has four
      // turns (32 products each) to arrive. It is waited for, by all waves, one turn before it is read. (16,384 x 5,632 by
      // 2,048 columns: 306 us, 1,235 TFLOP/s; with four phases of 16 products 334, without turns 1,377.)
      constexpr int MH = ATR ? T::MF : T::MF / 2, KH = ATR ? 1 : 2;
      constexpr std::integral_constant<int, ATR ? 3 : 5> a1{};
      constexpr std::integral_constant<int, ATR ? 12 : 10> a2{};
      constexpr std::integral_constant<int, ATR ? 3 : 15> b1{};
      constexpr std::integral_constant<int, ATR ? 12 : 0> b2{};
      static_assert(T::MF == 8 && T::NF == 4, "segments of the halves");
      static_assert(!ATR || BTR, "halves of k are separate segments in the (K, rows) form alone");
      s16x8 a[KH][MH], c[KH][T::NF];
      Cursor first = cursor_at(s0), second = first;  // of the segments that phase 1 reads, and phase 2
      auto turn = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      };
      // 8 loads are younger than the oldest that the next turn reads
      auto read_done = [&]() {
        asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
        turn();
        __builtin_amdgcn_s_setprio(1);
      };
      auto multiply = [&](auto m0) {
#pragma unroll
        for (int ks = 0; ks < KH; ++ks)
#pragma unroll
          for (int i = 0; i < MH; ++i)
#pragma unroll
            for (int j = 0; j < T::NF; ++j) acc[m0 + i][j] = mfma16<MT>(c[ks][j], a[ks][i], acc[m0 + i][j]);
        __builtin_amdgcn_s_setprio(0);
        turn();
      };
      constexpr int BO = T::BM * 128;
      auto step = [&](lds_char* at, lds_char* next) {
#pragma unroll
        for (int ks = 0; ks < KH; ++ks) {
          rb.template read<0, T::NF>(at + BO, ks, c[ks]);
          ra.template read<0, MH>(at, ks, a[ks]);
        }
        fetch(second, next, a2, b2);
        read_done();
        multiply(std::integral_constant<int, 0>{});
        if constexpr (ATR) {
          rb.template read<0, T::NF>(at + BO, 1, c[0]);
          ra.template read<0, MH>(at, 1, a[0]);
        } else {
#pragma unroll
          for (int ks = 0; ks < KH; ++ks) ra.template read<MH, MH>(at, ks, a[ks]);
        }
        fetch(first, at, a1, b1);
        read_done();
        multiply(std::integral_constant<int, ATR ? 0 : MH>{});
      };
      fetch(first, lds0, a1, b1);
      fetch(second, lds0, a2, b2);
      fetch(first, lds1, a1, b1);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      turn();
      if (wave >= 4) turn();
#pragma unroll 1
      for (int s = s0; s < s1; s += 2) {
        step(lds0, lds1);
        step(lds1, lds0);
      }
      if (wave < 4) turn();
    } else {
      Cursor next_load = cursor_at(s0);
      // The float32 instructions round after every product: sums of 256 k are kept apart and added (relative error of a
      // sum of 6,000 normal products 1.05e-6 in one chain, 3e-7 so).
      constexpr bool CHUNKS = std::is_same_v<MT, float>;
      constexpr int EVERY = 256 / (KS * T::STAGES);
      f32x4v sum[CHUNKS ? T::MF : 1][T::NF];
      int turn = 0;
      auto flush = [&](bool now) {
        if constexpr (CHUNKS) {
          if (!now) return;
#pragma unroll
          for (int i = 0; i < T::MF; ++i)
#pragma unroll
            for (int j = 0; j < T::NF; ++j) {
              sum[i][j] += acc[i][j];
              acc[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
            }
        }
      };
      if constexpr (CHUNKS)
#pragma unroll
        for (int i = 0; i < T::MF; ++i)
#pragma unroll
          for (int j = 0; j < T::NF; ++j) sum[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
      if constexpr (T::STAGES == 4) {
        // One barrier a step; its products run while the next step's fragments are read, the loads four steps ahead.
        constexpr int LOADS = la.SEGS + lb.SEGS;
        struct Frags {
          s16x8 a[2][T::MF], b[2][T::NF];
        };
        auto read = [&](const lds_char* at, Frags& f) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            rb.template read<0, T::NF>(at + T::BM * 128, ks, f.b[ks]);
            ra.template read<0, T::MF>(at, ks, f.a[ks]);
          }
        };
        auto multiply = [&](const Frags& f) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < T::MF; ++i)
#pragma unroll
              for (int j = 0; j < T::NF; ++j) acc[i][j] = mfma16<MT>(f.b[ks][j], f.a[ks][i], acc[i][j]);
        };
        Frags f, g2;
        auto step = [&](lds_char* at, const lds_char* next, const Frags& now, Frags& then) {
          // the next step's tiles have arrived, and everyone has read this step's
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * LOADS) : "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          read(next, then);
          fetch(next_load, at, all, all);
          multiply(now);
          // reads and loads are issued between the products
          constexpr int PRODUCTS = 2 * T::MF * T::NF * (std::is_same_v<MT, float> ? 4 : 1);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / 8, 0);  // matrix
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);             // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);             // loads
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        fetch(next_load, lds0, all, all);
        fetch(next_load, lds1, all, all);
        fetch(next_load, lds2, all, all);
        fetch(next_load, lds3, all, all);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * LOADS) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read(lds0, f);
#pragma unroll 1
        for (int s = s0; s < s1; s += 4) {
          step(lds0, lds1, f, g2);
          step(lds1, lds2, g2, f);
          step(lds2, lds3, f, g2);
          step(lds3, lds0, g2, f);
          flush(++turn % EVERY == 0);
        }
      } else {
        // One barrier a step; the loads run one step ahead.
        auto step = [&](const lds_char* at, lds_char* next) {
          // this step's tiles have arrived, and everyone has read the other stage
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          fetch(next_load, next, all, all);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            s16x8 a[T::MF], b[T::NF];
            ra.template read<0, T::MF>(at, ks, a);
            rb.template read<0, T::NF>(at + T::BM * 128, ks, b);
#pragma unroll
            for (int i = 0; i < T::MF; ++i)
#pragma unroll
              for (int j = 0; j < T::NF; ++j) acc[i][j] = mfma16<MT>(b[j], a[i], acc[i][j]);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        fetch(next_load, lds0, all, all);
#pragma unroll 1
        for (int s = s0; s < s1; s += 2) {
          step(lds0, lds1);
          step(lds1, lds0);
          flush(++turn % EVERY == 0);
        }
      }
      if constexpr (CHUNKS) {
#pragma unroll
        for (int i = 0; i < T::MF; ++i)
#pragma unroll
          for (int j = 0; j < T::NF; ++j) acc[i][j] += sum[i][j];
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // (anew, so that nothing of it is held in registers through the loop)
    int again_tid = threadIdx.x;
    asm volatile("" : "+v"(again_tid));
    const int end_lane = again_tid & 63;
    float scale = g.scale;
    if constexpr (F32) {
      float probe = 0.f;
#pragma unroll
      for (int i = 0; i < T::MF; ++i)
#pragma unroll
        for (int j = 0; j < T::NF; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) probe = fmaf(acc[i][j][v], 0.f, probe);
      // (a split K loop leaves this to the sum over its parts)
      if (g.splits == 1 && __any(probe != probe)) {
        again(g, m0, n0, wm, wn, end_lane, acc);
        scale = 1.f;
      }
    }
    __builtin_amdgcn_s_barrier();  // (everyone has read the stages, and their last loads have arrived)
    asm volatile("" ::: "memory");
    epilogue(g, scale, split, m0 + wm * T::TM, n0, wave, wn, end_lane, lds0, acc);
  }

  // In plain float32, scaled before the sum, which may stay finite where the sum of the unscaled products does not: lane
  // (r, q) of a 16x16x4 product takes k = 4 t + q of row r.
  __device__ static __forceinline__ void again(const FfnJob& g, int m0, int n0, int wm, int wn, int lane,
                                            f32x4v (&acc)[T::MF][T::NF]) {
    const int r = lane & 15, q = lane >> 4, k_end = max(g.A.k, g.B.k);
#pragma unroll
    for (int j = 0; j < T::NF; ++j) {
      int64_t col;
      if constexpr (EPI == EPI_GATE) {
        constexpr int H = T::TN / 2;
        col = min(n0 + wn * H + (j * 16) % H + r, g.N - 1) + (j * 16 >= H ? g.N : 0);
      } else {
        col = min(n0 + wn * T::TN + j * 16 + r, g.B.rows - 1);
      }
#pragma unroll
      for (int i = 0; i < T::MF; ++i) {
        f32x4v c{0.f, 0.f, 0.f, 0.f};
        const int row = min(m0 + wm * T::TM + i * 16 + r, g.A.rows - 1);
#pragma unroll 1
        for (int k = q; k < k_end + q; k += 4)
          c = __builtin_amdgcn_mfma_f32_16x16x4f32(value_of<ES, BTR>(g.B, col, k),
                                                   g.scale * value_of<ES, ATR>(g.A, row, k), c, 0, 0, 0);
        acc[i][j] = c;
      }
    }
  }

  // 16 rows of the wave's outputs at a time go through LDS, where a lane writes 4 columns of a row and takes 8, so that
  // memory is read and written in whole lines: as they come out of the products, a store would write 32 bytes of each of
  // 16 rows (16,384 x 2,048 x 5,632 in bf16: hidden gradient 640 us, of them 165 of stores).
  __device__ static __forceinline__ void epilogue(const FfnJob& g, float scale, int split, int row0, int n0, int wave,
                                                  int wn, int lane, lds_char* lds, f32x4v (&acc)[T::MF][T::NF]) {
    typedef __attribute__((address_space(3))) f32x4v lds_f32x4;
    constexpr int RS = T::TN * 4 + 16, COLS = EPI == EPI_GATE ? T::TN / 2 : T::TN;
    constexpr int LPR = COLS / 8, RPP = 64 / LPR < 16 ? 64 / LPR : 16, PASSES = 16 / RPP;  // lanes a row, rows a pass
    static_assert(T::NW * 16 * RS <= T::STAGE, "a stage holds 16 rows of each wave");
    lds_char* const mine = lds + wave * 16 * RS;
    lds_char* const to = mine + (lane & 15) * RS + (lane >> 4) * 16;
    const int rl = lane / LPR, cl = lane % LPR * 8;
    const lds_char* const from = mine + rl * RS + cl * 4;
    const int col = n0 + wn * COLS + cl;
    const bool on = rl < RPP;
    auto stage = [&](int i) {
#pragma unroll
      for (int j = 0; j < T::NF; ++j) *(lds_f32x4*)(to + 64 * j) = acc[i][j];
    };
    auto take = [&](const lds_char* p, float (&x)[8]) {
      const f32x4v u = *(const lds_f32x4*)p, v = *(const lds_f32x4*)(p + 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = u[k] * scale;
        x[4 + k] = v[k] * scale;
      }
    };
    if constexpr (EPI == EPI_OUT) {
#pragma unroll
      for (int i = 0; i < T::MF; ++i) {
        stage(i);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          int64_t row = row0 + 16 * i + p * RPP + rl;
          if (row >= g.M || col >= g.N) continue;
          float x[8];
          if (g.splits > 1) {  // unscaled
            const f32x4v u = *(const lds_f32x4*)(from + p * RPP * RS), v = *(const lds_f32x4*)(from + p * RPP * RS + 16);
            float* out = g.partial + ((int64_t)split * g.M + row) * g.N + col;
            *(f32x4v*)out = u;
            *(f32x4v*)(out + 4) = v;
            continue;
          }
          take(from + p * RPP * RS, x);
          if (row >= g.gap_at) {
            if (row < g.gap_at + g.gap) continue;
            row -= g.gap;
          }
          if (row >= g.m_out) continue;
          OT* out = (OT*)g.out + row * g.ld_out + col;
          Pack<OT, 8> o;
#pragma unroll
          for (int v = 0; v < 8; ++v) o.v[v] = from_f32<OT>(x[v]);
          if (col + 8 <= g.n_out) store_pack<OT, 8>(out, o);
          else
            for (int v = 0; v < 8; ++v)
              if (col + v < g.n_out) out[v] = o.v[v];
        }
      }
    } else if constexpr (EPI == EPI_GATE) {
#pragma unroll
      for (int i = 0; i < T::MF; ++i) {
        stage(i);
        const int64_t row = row0 + 16 * i + rl;
        if (!on || row >= g.M || col >= g.N) continue;
        float gate[8], up[8];
        take(from, gate);
        take(from + COLS * 4, up);
        finish_gate<MT, F32, 8>(g, row, col, g.N, gate, up);
      }
    } else {
      // the factors of the next turns are loaded before these rows' results are stored
      constexpr int TURNS = T::MF * PASSES, AHEAD = PLANES ? 1 : TURNS < 5 ? TURNS - 1 : 4;
      const int64_t count = (int64_t)g.M * g.N;
      Factors<F32, 8> f[AHEAD + 1];
      auto load = [&](int t) {
        const int64_t row = min(row0 + t * RPP + rl, g.M - 1);
        f[t % (AHEAD + 1)].load(g.saved, row * g.N + min(col, g.N - 8), count);
      };
#pragma unroll
      for (int t = 0; t < AHEAD; ++t) load(t);
#pragma unroll
      for (int t = 0; t < TURNS; ++t) {
        if (t % PASSES == 0) stage(t / PASSES);
        if (t + AHEAD < TURNS) load(t + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
        const int64_t row = row0 + t * RPP + rl;
        if (row >= g.M || col >= g.N) continue;
        float dh[8];
        take(from + t % PASSES * RPP * RS, dh);
        finish_dh<MT, F32, 8>(g, row, col, f[t % (AHEAD + 1)], dh);
      }
    }
  }
};

}  // namespace fc
