// Dense layers (included by fc_dense.hip, fc_dense_bwd.hip): y = residual + c act(s x W^T + b), one weight for all rows or
// one for each group of rows, and
//   dz = c g act'(z),  dx = s dz W,  dW = s dz^T x,  db = sum of the rows of dz,  d residual = g.
// The products are those of fc_ffn_gemm.h; bias, activation and residual are applied in the epilogue, before the one
// rounding of y. In 16-bit types dz is rounded to the type, as operand of the matrix instructions (one rounding more than an
// exact sum's: gradients of x and W are 1.4 times as far off as a rounding).
//
// Groups: the rows offsets[e] .. offsets[e + 1] - 1 have weight e. The offsets stay on the device: a workgroup finds its
// group and tile from them, or of many groups from a table that a launch before it makes of them; the grid is the most that any
// offsets can need.
#pragma once

#include "fc_gemm_plan.h"

namespace fc {

enum { ACT_NONE = 3 };

// act'(z) as it is kept for the backward pass: in float32; beside bfloat16 operands 2^15 act'(z) in float16, which has
// |act'| <= 1.13 inside its range and 11 significant bits (a rounding of an eighth of the operands') down to 2^-29, fewer
// below, none below 2^-40; beside float16 ones with 24 bits, (upper 16, next 8) in two arrays.
template <class OT>
constexpr float kFactorScale = std::is_same_v<OT, bf16_t> ? 0x1p15f : 1.f;

// d: act'(z) times that scale.

template <class OT, int V>
__device__ __forceinline__ void put_factor(char* factor, int64_t at, int64_t count, const float (&d)[V]) {
  if constexpr (std::is_same_v<OT, float>) {
    put_floats((float*)factor + at, d);
  } else if constexpr (std::is_same_v<OT, bf16_t>) {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2<f16_t>(d[2 * i], d[2 * i + 1]);
    put_words<V>(factor + 2 * at, w);
  } else {
    uint32_t hi[V / 2], lo[V / 4];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const uint32_t u0 = __float_as_uint(d[2 * i]) + 0x80, u1 = __float_as_uint(d[2 * i + 1]) + 0x80;
      hi[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302);
      const uint32_t pair = __builtin_amdgcn_perm(u1, u0, 0x0c0c0501);
      if (i % 2 == 0) lo[i / 2] = pair;
      else lo[i / 2] |= pair << 16;
    }
    put_words<V>(factor + 2 * at, hi);
    char* const p = factor + 2 * count + at;
    if constexpr (V == 8) *(uint2*)p = make_uint2(lo[0], lo[1]);
    else *(uint32_t*)p = lo[0];
  }
}
template <class OT>
__device__ __forceinline__ void get_factor(const char* factor, int64_t at, int64_t count, float (&d)[8]) {
  if constexpr (std::is_same_v<OT, float>) {
    const float4 u = *(const float4*)((const float*)factor + at), v = *(const float4*)((const float*)factor + at + 4);
    d[0] = u.x, d[1] = u.y, d[2] = u.z, d[3] = u.w, d[4] = v.x, d[5] = v.y, d[6] = v.z, d[7] = v.w;
  } else if constexpr (std::is_same_v<OT, bf16_t>) {
    const Pack<f16_t, 8> p = *(const Pack<f16_t, 8>*)__builtin_assume_aligned(factor + 2 * at, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = to_f32(p.v[i]);
  } else {
    const uint4 h = *(const uint4*)(factor + 2 * at);
    const uint2 l = *(const uint2*)(factor + 2 * count + at);
    const uint32_t hi[4] = {h.x, h.y, h.z, h.w}, lo[2] = {l.x, l.y};
#pragma unroll
    for (int i = 0; i < 8; ++i)  // (bytes: 4 to 7 of the first operand, 0 to 3 of the second, 0x0c zero)
      d[i] = __uint_as_float(__builtin_amdgcn_perm(hi[i / 2], lo[i / 4],
                                                   (i % 2 ? 0x07060000u : 0x05040000u) | (uint32_t)(i % 4) << 8 | 0x0cu));
  }
}

// The normal distribution's function at z, and e = exp(-z^2 / 2). With t = |z| its tail is e R(t), R(t) = erfcx(t / sqrt 2) / 2:
// R is smooth and falls as 1 / t, so with u = 1 / (1 + t / 4) it is u times a polynomial of u (degree 9, fitted to least relative
// error, 3.4e-8 on [0, 1]). So the tail has the relative error of e, 2^-24 (1 + z^2), where 1 + erf(z / sqrt 2) has only
// absolute bits (at z = -5 off by 5%, at -5.6 nothing), and costs less than erf beside e (16,384 x 512 x 4,096 f16 forward 165 ->
// 129 us). EXACT: by erf above -1, where that is nearer (relative errors 2e-7 and 4e-7).
template <bool EXACT>
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& e) {
  constexpr float c[10] = {0.0997355654835701f,  0.09973642975091934f, 0.09346635639667511f, 0.08160309493541718f,
                           0.058975208550691605f, 0.06369893997907639f, -0.0317172147333622f, 0.09559676796197891f,
                           -0.08087713271379471f, 0.019781969487667084f};
  const float u = __builtin_amdgcn_rcpf(fmaf(0.25f, fabsf(z), 1.f));
  float p = c[9];
#pragma unroll
  for (int i = 8; i >= 0; --i) p = fmaf(p, u, c[i]);
  e = __expf(-0.5f * z * z);
  const float tail = e * (u * p);
  cdf = z > 0.f ? 1.f - tail : tail;
  if constexpr (EXACT) cdf = z > -1.f ? 0.5f * (1.f + erff(z * 0.70710678118654752f)) : cdf;
}

// What find_unit finds by scanning all offsets, made once for the whole call where groups are many: then the scan would take
// longer than the work (find_unit reads 64 offsets at a time, every workgroup all of them).
struct UnitTable {
  const int32_t* ends;    // (groups + 1): the first row of each group, and the end of the last; null: there is no table
  const int32_t* before;  // (groups + 1): units of the groups before each, of all
  const int32_t* slots;   // (groups): the same, of those that have more than one
};

// One product of a dense layer. For groups the pointers are those of the whole call, and a workgroup shifts them.
struct DenseJob : GemmJob {
  const void* bias;              // (groups, n_out), or null
  const void* residual;          // (rows, n_out), or null
  const float *row_scale, *col_scale;  // of 8-bit operands
  char* factor;                  // act'(z), (rows, N), or null
  int64_t factor_at, factor_count;
  int32_t act;
  float act_scale;
  const int64_t* offsets;        // (groups + 1)
  UnitTable table;               // of the units that this product's tiles take
  int32_t groups;
  int32_t halves;                // tiles at the end that are taken as two halves of their columns
  int32_t unit;                  // > 0: sums over a group's rows, in parts of so many
  int64_t rows, b_stride, out_stride;  // rows of the call; elements from one group's B, and output, to the next one's
  int32_t first, blocks;         // first workgroup of this launch, workgroups of all

  // V columns from `col` on of the rows that a lane finishes one after the other:
  // where it is, what its columns have in common in all rows, and the residuals of its next rows, loaded ahead.
  template <class OT, bool F32, bool EIGHT, int V>
  struct Line {
    OT* out;
    const OT* res;
    int64_t factor_at;
    float bias[V], col_scale[V];
    float act_scale;
    int col_at;
    bool whole;
    Pack<OT, V> next[2];

    __device__ __forceinline__ void init(const DenseJob& g, int64_t row, int col) {
      out = (OT*)g.out + row * g.ld_out + col;
      res = g.residual ? (const OT*)g.residual + row * g.ld_out + col : nullptr;
      factor_at = g.factor_at + row * g.N + col;
      col_at = col;
      whole = col + V <= g.n_out;
      act_scale = g.act_scale;
      Pack<OT, V> b{};
      Pack<float, V> c{};
      if (g.bias) b = part(g, (const OT*)g.bias + col);
      if constexpr (EIGHT) c = part(g, g.col_scale + col);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        bias[v] = to_f32(b.v[v]);
        col_scale[v] = EIGHT ? c.v[v] : 1.f;
      }
    }
    // the V elements from p on, as far as there are columns
    template <class E>
    __device__ __forceinline__ Pack<E, V> part(const DenseJob& g, const E* p) const {
      Pack<E, V> r{};
      if (whole) return load_pack<E, V>(p);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (col_at + v < g.n_out) r.v[v] = p[v];
      return r;
    }
    // the residuals of this turn's rows: `row`, row + step, ... of PASSES
    template <int PASSES>
    __device__ __forceinline__ void ahead(const DenseJob& g, bool inside, int64_t row, int step) {
      if (!g.residual) return;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        if (inside && row + p * step < g.M) next[p] = part(g, res + p * step * g.ld_out);
      }
    }
    // y of those rows from their sums, scaled by s; the cursor goes on to the next turn, 16 rows further
    template <int PASSES>
    __device__ __forceinline__ void finish(const DenseJob& g, bool inside, int64_t row, int step,
                                           float (&x)[PASSES][V]) {
      static_assert(PASSES <= 2, "residuals ahead");
      constexpr float KEEP = kFactorScale<OT>;
      const bool keep = !EIGHT && g.factor != nullptr;
      Pack<OT, V> r[PASSES];
      const bool with_res = g.residual != nullptr;
      if (with_res) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) r[p] = next[p];
        res += 16 * g.ld_out;
        ahead<PASSES>(g, inside, row + 16, step);
      }
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const bool ok = inside && row + p * step < g.M;
        float d[V];
        float row_scale = 1.f;
        if constexpr (EIGHT) row_scale = g.row_scale[ok ? row + p * step : 0];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if constexpr (EIGHT) x[p][v] = fmaf(x[p][v] * row_scale, col_scale[v], bias[v]);
          else x[p][v] += bias[v];
        }
        if (g.act == ACT_NONE) {
#pragma unroll
          for (int v = 0; v < V; ++v) x[p][v] *= act_scale;
        } else if (g.act == 2) {
          float cdf[V], e[V];
#pragma unroll
          for (int v = 0; v < V; ++v) normal_cdf<std::is_same_v<OT, float>>(x[p][v], cdf[v], e[v]);
          if (keep) {
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] = fmaf(KEEP, cdf[v], x[p][v] * e[v] * (KEEP * 0.3989422804014327f));
          }
#pragma unroll
          for (int v = 0; v < V; ++v) x[p][v] *= act_scale * cdf[v];
        } else {
          // y = s z, or the logistic function s = 1 / (1 + e) itself (also of an infinite z), and act' = y (1 - s) + s, or
          // y (1 - s). 1 - s = s e keeps its bits where s is near one; where e is infinite, s and y are zero, and the smaller of
          // NaN and one is one.
          float s[V], e[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            e[v] = __expf(-x[p][v]);
            s[v] = __builtin_amdgcn_rcpf(1.f + e[v]);
          }
          if (g.act == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) x[p][v] = s[v];
          } else {
#pragma unroll
            for (int v = 0; v < V; ++v) x[p][v] *= s[v];
          }
          if (keep) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
              s[v] *= KEEP;
              e[v] = fminf(s[v] * e[v], KEEP);
            }
            if (g.act == 1) {
#pragma unroll
              for (int v = 0; v < V; ++v) d[v] = x[p][v] * e[v];
            } else {
#pragma unroll
              for (int v = 0; v < V; ++v) d[v] = fmaf(x[p][v], e[v], s[v]);
            }
          }
#pragma unroll
          for (int v = 0; v < V; ++v) x[p][v] *= act_scale;
        }
        if (with_res) {
#pragma unroll
          for (int v = 0; v < V; ++v) x[p][v] += to_f32(r[p].v[v]);
        }
        if (!ok) continue;
        OT* const to = out + p * step * g.ld_out;
        if (whole) {
          Pack<OT, V> o;
          if constexpr (std::is_same_v<OT, float>) {
#pragma unroll
            for (int v = 0; v < V; ++v) o.v[v] = x[p][v];
          } else {
            uint32_t w[V / 2];
#pragma unroll
            for (int v = 0; v < V / 2; ++v) w[v] = pack2<OT>(x[p][2 * v], x[p][2 * v + 1]);
            memcpy(&o, w, sizeof(o));
          }
          // (past the caches where that is 16 bytes: what is read again while a layer runs, its operands and act'(z), stays in
          // them. us: 16,384 x 2,048 x 5,632 bf16 forward 390 -> 372, dz 113 -> 101; 4,096 x 8,192 x 5,120 in 8 bits 180 ->
          // 151; two layers after each other, the second reading y, 612 and 612, 149 -> 146)
          if constexpr (V == 8 && sizeof(OT) == 2) stream_pack<OT>(to, o);
          else store_pack<OT, V>(to, o);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (col_at + v < g.n_out) to[v] = from_f32<OT>(x[p][v]);
        }
        if constexpr (!EIGHT) {
          if (keep) put_factor<OT, V>(g.factor, factor_at + (int64_t)p * step * g.N, g.factor_count, d);
        }
      }
      out += 16 * g.ld_out;
      factor_at += 16 * (int64_t)g.N;
    }
  };
};

// Where unit `t` of the groups' rows is, or (BY_GROUP) group `t`'s first: of the units of `size` rows (an empty group has
// `least` of them), counted group by group. Offsets are taken into [0, n] and as their running maximum, so that the groups' rows are apart whatever they hold.
struct GroupUnit {
  int group, index;   // -1: there are fewer units than that; index within the group
  int64_t row, rows;  // the group's first row and its rows
  int total;          // units of all groups
  int before;         // units of the groups before it
  int slot;           // the same, of those that have more than one
  int64_t begin, end; // rows of all groups
};
template <bool BY_GROUP = false>
__device__ __forceinline__ GroupUnit find_unit(const int64_t* offsets, const UnitTable& table, int groups, int64_t n, int size,
                                               int least, int t, bool want_total) {
  const int lane = threadIdx.x & 63;
  if (table.ends) {
    GroupUnit u{-1, 0, 0, 0, 0, 0, 0, table.ends[0], table.ends[groups]};
    int e = t;
    if constexpr (!BY_GROUP) {
      u.total = table.before[groups];
      if (t < 0 || t >= u.total) return u;
      // the last group with no more units before it than t, in steps of 64
      e = 0;
      for (int span = groups; span > 1;) {
        const int step = (span + 63) / 64, at = lane * step;
        const uint64_t hit = __ballot(at < span && table.before[e + (at < span ? at : 0)] <= t);
        const int k = (__popcll(hit) - 1) * step;
        e += k;
        span = min(step, span - k);
      }
    }
    u.group = __builtin_amdgcn_readfirstlane(e);
    u.before = table.before ? table.before[u.group] : 0;
    u.index = BY_GROUP ? 0 : t - u.before;
    const int row = __builtin_amdgcn_readfirstlane(table.ends[u.group]);
    u.row = row;
    u.rows = __builtin_amdgcn_readfirstlane(table.ends[u.group + 1]) - row;
    u.slot = table.slots ? table.slots[u.group] : 0;
    return u;
  }
  auto clamped = [&](int64_t v) { return v < 0 ? 0 : v > n ? n : v; };
  GroupUnit u{-1, 0, 0, 0, 0, 0, 0, 0, 0};
  int64_t last = clamped(offsets[0]);
  u.begin = last;
  int units = 0, several = 0;
  for (int b = 0; b < groups; b += 64) {
    int64_t end = b + lane < groups ? clamped(offsets[b + lane + 1]) : 0;
    end = end > last ? end : last;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int64_t v = __shfl_up(end, o, 64);
      if (lane >= o && v > end) end = v;
    }
    int64_t begin = __shfl_up(end, 1, 64);
    if (lane == 0) begin = last;
    int count = (int)((end - begin + size - 1) / size);
    if (count < least) count = least;
    if (b + lane >= groups) count = 0;
    int upto = count, more = count > 1 ? count : 0;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int v = __shfl_up(upto, o, 64), w = __shfl_up(more, o, 64);
      if (lane >= o) {
        upto += v;
        more += w;
      }
    }
    const uint64_t hit = __ballot(BY_GROUP ? b + lane == t : t >= units + upto - count && t < units + upto);
    if (hit && u.group < 0) {
      const int at = __builtin_ctzll(hit);
      const int own = __shfl(count, at, 64);
      u.group = b + at;
      u.before = units + __shfl(upto, at, 64) - own;
      u.index = BY_GROUP ? 0 : t - u.before;
      u.row = __shfl(begin, at, 64);
      u.rows = __shfl(end, at, 64) - u.row;
      u.slot = several + __shfl(more, at, 64) - (own > 1 ? own : 0);
      if (!want_total) break;
    }
    units += __shfl(upto, 63, 64);
    several += __shfl(more, 63, 64);
    last = __shfl(end, 63, 64);
  }
  auto uniform64 = [](int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
  };
  u.group = __builtin_amdgcn_readfirstlane(u.group);
  u.index = __builtin_amdgcn_readfirstlane(u.index);
  u.before = __builtin_amdgcn_readfirstlane(u.before);
  u.slot = __builtin_amdgcn_readfirstlane(u.slot);
  u.total = __builtin_amdgcn_readfirstlane(units);
  u.begin = uniform64(u.begin);
  u.end = uniform64(last);
  u.row = uniform64(u.row);
  u.rows = uniform64(u.rows);
  return u;
}

// One workgroup's tile of a job with groups. A job over rows has a tile for every T::BM rows of a group; one with `unit`
// sums over a group's rows, the parts of a group of more than one to `partial`, in the groups' order.
template <class T, class MT, bool F32, bool ATR, bool BTR, int EPI, class OT_ = void>
struct GroupTile {
  using Base = FfnTile<T, MT, F32, ATR, BTR, EPI, OT_>;
  using OT = typename Base::OT;
  __device__ static __forceinline__ void run(const DenseJob& arg, int block, int blocks, lds_char* l0, lds_char* l1, lds_char* l2,
                                             lds_char* l3) {
    constexpr bool SUMS = ATR;
    DenseJob g = arg;
    const int size = SUMS ? g.unit : T::BM, least = SUMS ? 1 : 0, per = SUMS ? g.tiles_m * g.tiles_n : g.tiles_n;
    // block -> tile as without groups: a run of tiles for each XCD
    const GroupUnit all = find_unit(g.offsets, g.table, g.groups, g.rows, size, least, -1, true);
    const int total = all.total * per;
    if constexpr (!SUMS) {  // rows of no group
      for (int64_t r = block; r < g.rows - (all.end - all.begin); r += blocks) {
        OT* const out = (OT*)g.out + (r < all.begin ? r : r + (all.end - all.begin)) * g.ld_out;
        for (int c = threadIdx.x; c < g.n_out; c += T::NT) out[c] = from_f32<OT>(0.f);
      }
    }
    if (block >= total) return;
    int tile = block;
    if (total >= 64) {
      const int each = total / 8, rest = total % 8, x = tile % 8;
      tile = x * each + min(x, rest) + tile / 8;
    }
    const GroupUnit u = find_unit(g.offsets, g.table, g.groups, g.rows, size, least, tile / per, false);
    int tiles_m = g.tiles_m, in;
    if constexpr (SUMS) {
      const int64_t row = u.row + (int64_t)u.index * g.unit, left = u.rows - (int64_t)u.index * g.unit;
      const int k = (int)(left < g.unit ? left : g.unit);
      g.A.p += Base::ES * row * g.A.ld;
      g.B.p += Base::ES * row * g.B.ld;
      g.A.k = g.B.k = k;
      g.steps = max(1, (k + Base::KS - 1) / Base::KS) * (Base::PLANES ? 6 : 1);
      if (u.rows > g.unit) {
        g.splits = 2;
        g.partial += (int64_t)(u.slot + u.index) * g.M * g.N;
      } else {
        g.splits = 1;
        g.out = (OT*)g.out + u.group * g.out_stride;
      }
      in = tile - tile / per * per;
    } else {
      g.A.p += Base::ES * u.row * g.A.ld;
      g.A.rows = g.M = g.m_out = (int)u.rows;
      g.B.p += Base::ES * u.group * g.b_stride;
      g.out = (OT*)g.out + u.row * g.ld_out;
      if constexpr (EPI == EPI_DENSE) {
        if (g.bias) g.bias = (const OT*)g.bias + (int64_t)u.group * g.n_out;
        g.factor_at = u.row * g.N;
      }
      tiles_m = (int)((u.rows + T::BM - 1) / T::BM);
      in = tile - u.before * per;
    }
    const int group = in / (8 * g.tiles_n), rest = in - group * 8 * g.tiles_n, gm = min(8, tiles_m - group * 8);
    Base::run_tile(g, group * 8 + rest % gm, rest / gm, 0, 0, g.steps, l0, l1, l2, l3);
  }
};

}  // namespace fc
