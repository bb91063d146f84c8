// Dense layers of few rows (included by fc_dense.hip): bound by reading the weight once, so the weight goes from memory
// straight into the fragments of the matrix instructions. A workgroup forms 16 output columns of up to 32 rows: its 8 waves
// take blocks of 256 bytes of k in turn, their sums meet in LDS, and the epilogue follows there: one launch, no copies of
// operands whose rows are not a multiple of 16 bytes. A lane brings 16 bytes of a row to an instruction; which k those are
// does not matter as long as both operands agree.
#pragma once

#include "fc_dense.h"

namespace fc {

constexpr int kFewWaves = 8, kFewRows = 32;

// 16 bytes, at the alignment of an element.
template <int ES>
__device__ __forceinline__ s16x8 few_load(const char* p) {
  s16x8 v;
  memcpy(&v, p, 16);
  return v;
}
// 16 bytes of a row from element k on, zeros past the end.
template <int ES>
__device__ __forceinline__ s16x8 few_load(const char* row, int k, int end) {
  if (k + 16 / ES <= end) return few_load<ES>(row + (int64_t)k * ES);
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < 16 / ES; ++i) {
    if (k + i >= end) continue;
    const char* const p = row + (int64_t)(k + i) * ES;
    if constexpr (ES == 4) w[i] = *(const uint32_t*)p;
    else if constexpr (ES == 2) w[i / 2] |= (uint32_t)*(const uint16_t*)p << 16 * (i % 2);
    else w[i / 4] |= (uint32_t)*(const uint8_t*)p << 8 * (i % 4);
  }
  return __builtin_bit_cast(s16x8, w);
}

// MF blocks of 16 rows. The operands' rows lie in_features elements apart.
template <class MT, class OT, int MF, bool GROUPS>
__global__ void __launch_bounds__(64 * kFewWaves) dense_few_kernel(DenseJob g) {
  constexpr bool F32 = std::is_same_v<MT, float>, EIGHT = std::is_same_v<MT, e4m3_t>;
  constexpr int ES = F32 ? 4 : EIGHT ? 1 : 2, V = 16 / ES, STEP = 4 * V, U = 4, BLOCK = U * STEP, ROWS = 16 * MF;
  __shared__ f32x4v part[kFewWaves][ROWS][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4, col_blocks = (g.n_out + 15) / 16;
  const int id = g.first + blockIdx.x, n0 = (GROUPS ? id % col_blocks : id) * 16;
  const char *xs = g.A.p, *ws = g.B.p;
  int rows = g.M;
  if constexpr (GROUPS) {
    const int e = id / col_blocks;
    const GroupUnit u = find_unit<true>(g.offsets, g.table, g.groups, g.rows, 1, 0, e, true);
    // rows of no group
    for (int64_t k = id; k < g.rows - (u.end - u.begin); k += g.blocks) {
      OT* const out = (OT*)g.out + (k < u.begin ? k : k + (u.end - u.begin)) * g.ld_out;
      for (int c = threadIdx.x; c < g.n_out; c += 64 * kFewWaves) out[c] = from_f32<OT>(0.f);
    }
    if (u.rows == 0) return;
    rows = (int)u.rows;
    xs += ES * u.row * g.A.ld;
    ws += ES * e * g.b_stride;
    g.out = (OT*)g.out + u.row * g.ld_out;
    if (g.bias) g.bias = (const OT*)g.bias + (int64_t)e * g.n_out;
    g.factor_at = u.row * g.N;
    g.M = rows;
  }
  const int K = g.A.k;
  const char* const w = ws + ES * min(n0 + r, g.n_out - 1) * g.B.ld;
  for (int m0 = 0; m0 < rows; m0 += ROWS) {
    const char* x[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) x[i] = xs + ES * min(m0 + 16 * i + r, rows - 1) * g.A.ld;
    f32x4v acc[MF], sum[F32 ? MF : 1];
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    if constexpr (F32)
#pragma unroll
      for (int i = 0; i < MF; ++i) sum[i] = acc[i];
    auto block = [&](auto load, int k0) {
      s16x8 b[U], a[U][MF];
#pragma unroll
      for (int u = 0; u < U; ++u) b[u] = load(w, k0 + u * STEP + q * V);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < MF; ++i) a[u][i] = load(x[i], k0 + u * STEP + q * V);
#pragma unroll
      for (int u = 0; u < U; u += EIGHT ? 2 : 1)
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          if constexpr (EIGHT) acc[i] = mfma8(b[u], b[u + 1], a[u][i], a[u + 1][i], acc[i]);
          else acc[i] = mfma16<MT>(b[u], a[u][i], acc[i]);
        }
    };
    // (the next block's loads ahead of a block's products cost more in occupancy than they gave: 23.8 us instead of 19.9)
    int k0 = wave * BLOCK, turn = 0;
#pragma unroll 1
    for (; k0 + BLOCK <= K; k0 += kFewWaves * BLOCK) {
      block([&](const char* row, int k) { return few_load<ES>(row + (int64_t)k * ES); }, k0);
      if constexpr (F32) {  // (the float32 instructions round after every product: sums of 256 k are kept apart)
        if (++turn % (256 / BLOCK) == 0)
#pragma unroll
          for (int i = 0; i < MF; ++i) {
            sum[i] += acc[i];
            acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
          }
      }
    }
    if (k0 < K) block([&](const char* row, int k) { return few_load<ES>(row, k, K); }, k0);
    if constexpr (F32)
#pragma unroll
      for (int i = 0; i < MF; ++i) acc[i] += sum[i];
    if (m0 > 0) __syncthreads();  // (the last rows' sums have been read)
#pragma unroll
    for (int i = 0; i < MF; ++i) part[wave][16 * i + r][q] = acc[i];
    __syncthreads();
    const int row = threadIdx.x / 4, c4 = threadIdx.x % 4, col = n0 + 4 * c4;
    if (row < ROWS && m0 + row < rows && col < g.n_out) {
      f32x4v s = part[0][row][c4];
#pragma unroll
      for (int k = 1; k < kFewWaves; ++k) s += part[k][row][c4];
      float y[1][4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        y[0][v] = s[v] * g.scale;
        if constexpr (F32) {
          if (!(fabsf(y[0][v]) < __builtin_inff())) {  // again, scaled before the sum
            const float* const u = (const float*)xs + (m0 + row) * g.A.ld;
            const float* const t = (const float*)ws + min(col + v, g.n_out - 1) * g.B.ld;
            y[0][v] = 0.f;
            for (int k = 0; k < K; ++k) y[0][v] = fmaf(g.scale * u[k], t[k], y[0][v]);
          }
        }
      }
      DenseJob::Line<OT, F32, EIGHT, 4> line;
      line.init(g, m0 + row, col);
      line.template ahead<1>(g, true, m0 + row, 0);
      line.template finish<1>(g, true, m0 + row, 0, y);
    }
  }
}

}  // namespace fc
