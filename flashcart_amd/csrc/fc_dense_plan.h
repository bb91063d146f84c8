// What is where in one call of a dense layer: operands, padded copies, workspace; tiles of products with groups.
#pragma once

#include "fc_dense.h"

namespace fc {

// ---- operands whose rows are not a multiple of 16 bytes, and those in planes: a padded copy ----
struct PadItem {
  const void* src;
  char* dst;
  int64_t rows, cols, ld, plane;  // rows, columns of src; of dst
  int64_t block_base;
};
struct PadArgs {
  PadItem it[2];
  int32_t count;
  int64_t first;  // block of this launch
};

template <class T, class MT>
__global__ void __launch_bounds__(256) dense_pad_kernel(PadArgs a) {
  const int64_t block = a.first + blockIdx.x;
  const PadItem& it = a.it[a.count > 1 && block >= a.it[1].block_base ? 1 : 0];
  const int64_t chunks = it.ld / 8, t = (block - it.block_base) * 256 + threadIdx.x;
  if (t >= it.rows * chunks) return;
  const int64_t row = t / chunks, c0 = (t - row * chunks) * 8;
  const T* src = (const T*)it.src + row * it.cols + c0;
  if constexpr (std::is_same_v<T, MT>) {
    Pack<T, 8> v;
    if (c0 + 8 <= it.cols) {
      v = load_pack<T, 8>(src);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = c0 + i < it.cols ? src[i] : T{};
    }
    store_pack<T, 8>((T*)it.dst + row * it.ld + c0, v);
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c0 + i < it.cols ? to_f32(src[i]) : 0.f;
    put<MT, true, 8>(it.dst, row * it.ld + c0, it.plane, x);
  }
}

// ---- tables of units (UnitTable) ----
struct UnitsArgs {
  const int64_t* offsets;
  int32_t* ends;
  int64_t rows;
  int32_t groups, count;
  struct {
    int32_t size, least;  // size 0: the ends alone
    int32_t *before, *slots;
  } table[5];
};

// v of the lanes and waves before this thread's, by f; `none` for the first.
template <class F>
__device__ __forceinline__ int before_thread(int v, int none, int* lds, F&& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int w = __shfl_up(v, o, 64);
    if (lane >= o) v = f(v, w);
  }
  __syncthreads();  // (the last call's values have been read)
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  int all = none;
  for (int k = 0; k < waves; ++k)
    if (k < wave) all = f(all, lds[k]);
  const int up = __shfl_up(v, 1, 64);
  return lane > 0 ? f(all, up) : all;
}

// A workgroup a table. A thread takes a run of groups; the largest offset, and the units, of the runs before it come by a scan.
static __global__ void __launch_bounds__(1024) dense_units_kernel(UnitsArgs a) {
  __shared__ int lds[16];
  const int each = (a.groups + 1023) / 1024, e0 = min((int)threadIdx.x * each, a.groups), e1 = min(e0 + each, a.groups);
  const int n = (int)a.rows;
  auto offset = [&](int e) {
    const int64_t v = a.offsets[e];
    return v < 0 ? 0 : v > n ? n : (int)v;
  };
  auto larger = [](int u, int v) { return u > v ? u : v; };
  auto sum = [](int u, int v) { return u + v; };
  const int start = offset(0);
  int most = start;
  for (int e = e0; e < e1; ++e) most = larger(most, offset(e + 1));
  const int first = before_thread(most, start, lds, larger);  // where group e0 begins
  const auto& t = a.table[blockIdx.x];
  const int least = t.least, size = t.size;
  auto units = [&](int rows) { return larger(least, (rows + size - 1) / size); };
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) a.ends[0] = start;
    for (int e = e0, at = first; e < e1; ++e) a.ends[e + 1] = at = larger(at, offset(e + 1));
  }
  if (size == 0) return;
  int count = 0, several = 0;
  for (int e = e0, at = first; e < e1; ++e) {
    const int end = larger(at, offset(e + 1)), c = units(end - at);
    count += c;
    several += c > 1 ? c : 0;
    at = end;
  }
  int before = before_thread(count, 0, lds, sum), slot = before_thread(several, 0, lds, sum);
  for (int e = e0, at = first; e < e1; ++e) {
    const int end = larger(at, offset(e + 1)), c = units(end - at);
    t.before[e] = before;
    t.slots[e] = slot;
    before += c;
    slot += c > 1 ? c : 0;
    at = end;
  }
  if (e0 < e1 && e1 == a.groups) t.before[a.groups] = before;
}

// f(type of the operands in memory, is the operator's type float32)
template <class F>
int with_operand_form(int32_t dtype, Form form, F&& f) {
  if (form == FORM_NATIVE) return f(float{}, std::true_type{});
  if (form == FORM_PLANES) return f(bf16_t{}, std::true_type{});
  if (dtype == FC_BF16) return f(bf16_t{}, std::false_type{});
  return f(f16_t{}, std::false_type{});
}

// float32 in planes where the products are large and the operands are used often enough for their splitting to pay (as in
// the feed-forward block); with groups, a weight is used by the rows of its group.
inline Form dense_form(const fc_dense_desc& d, int64_t n) {
  if (d.dtype != FC_F32) return FORM_16;
  const int64_t each = d.groups > 0 ? n / d.groups : n;
  const bool large = each >= 512 && d.in >= 512 && d.out >= 512 && (double)n * d.in * d.out >= 2e9;
  return large ? FORM_PLANES : FORM_NATIVE;
}

inline int dense_check(const fc_dense_desc* d, int64_t n) {
  if (!d) return FC_ERR_NULL;
  if (!node_dtype_ok(d->dtype) || d->act < 0 || d->act > ACT_NONE) return FC_ERR_BAD_DESC;
  if (d->in < 1 || d->out < 1 || d->in > (1 << 20) || d->out > (1 << 20) || n < 0 || n > 0x7ffffff || d->groups < 0 ||
      d->groups > (1 << 16) || (int64_t)(d->groups + 1) * d->out > INT32_MAX / 2)
    return FC_ERR_SHAPE;
  return FC_OK;
}

struct Dense {
  const fc_dense_desc& d;
  int64_t n, in, out, ip, op, weights;  // ip, op: padded sizes
  Form form;
  int64_t esize;  // bytes of an element of an operand, over all planes
  char* ws;
  int64_t at = 0;
  PadArgs pad{};
  int64_t pad_blocks = 0;

  Dense(const fc_dense_desc& desc, int64_t rows, void* workspace, bool eight = false)
      : d(desc), n(rows), in(desc.in), out(desc.out), ip(eight ? (in + 15) / 16 * 16 : up8(in)), op(up8(out)),
        weights(desc.groups > 0 ? desc.groups : 1), form(eight ? FORM_8 : dense_form(desc, rows)),
        esize(form == FORM_8 ? 1 : form == FORM_16 ? 2 : form == FORM_NATIVE ? 4 : 6), ws((char*)workspace) {}

  char* take(int64_t bytes) {
    char* p = ws + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
  bool direct(int64_t cols, int64_t ld) const { return form != FORM_PLANES && d.aligned && ld == cols; }
  // (rows, cols) of the caller as an operand of padded rows: itself, or its copy
  Opnd operand(const void* src, int64_t rows, int64_t cols, int64_t ld) {
    Opnd o{};
    o.ld = ld;
    o.plane = rows * ld;
    if (direct(cols, ld)) {
      o.p = (const char*)src;
      return o;
    }
    PadItem& it = pad.it[pad.count++];
    it.src = src;
    it.dst = take(esize * o.plane);
    it.rows = rows;
    it.cols = cols;
    it.ld = ld;
    it.plane = o.plane;
    it.block_base = pad_blocks;
    pad_blocks += (o.plane / 8 + 255) / 256;
    o.p = it.dst;
    return o;
  }
  Opnd x(const void* p) { return operand(p, n, in, ip); }
  Opnd weight(const void* p) { return operand(p, weights * out, in, ip); }
  int run_pad(hipStream_t s) {
    if (pad.count == 0) return FC_OK;
    return in_launches(pad_blocks, [&](int64_t first, unsigned blocks) {
      pad.first = first;
      const dim3 grid(blocks), block(256);
      if (form == FORM_8) hipLaunchKernelGGL((dense_pad_kernel<e4m3_t, e4m3_t>), grid, block, 0, s, pad);
      else if (form == FORM_16) hipLaunchKernelGGL((dense_pad_kernel<bf16_t, bf16_t>), grid, block, 0, s, pad);
      else if (form == FORM_NATIVE) hipLaunchKernelGGL((dense_pad_kernel<float, float>), grid, block, 0, s, pad);
      else hipLaunchKernelGGL((dense_pad_kernel<float, bf16_t>), grid, block, 0, s, pad);
    });
  }
  int64_t factor_bytes() const {
    return d.act == ACT_NONE ? 0 : (d.dtype == FC_F32 ? 4 : d.dtype == FC_BF16 ? 2 : 3) * n * op;
  }
  // Whether the units of groups stand in a table: of more than 64 groups, which a scan takes in one step, where the weights are
  // many workgroups' work, and of more than 256. us, scan / table, forward and backward: 100 groups of 64 x 64, 16,384 rows 9 and
  // 51 / 13 and 53; 100 of 1,024 x 1,024, 512 rows 41 and 182 / 39 and 145, 200 102 and 423 / 90 and 271; 320 of 256 x 256, 16,384
  // rows 30 and 75 / 21 and 54; 4,096 of 64 x 64 522 and 1,700 / 34 and 91; 65,536 78,000 and 336,000 / 370 and 1,060.
  bool tabled() const { return d.groups > 256 || (d.groups > 64 && d.groups * in * out >= 1 << 26); }
  UnitsArgs unit_tables{};
  UnitTable units(int size, int least) {
    if (!tabled()) return UnitTable{};
    UnitsArgs& a = unit_tables;
    if (a.count == 0) a.ends = (int32_t*)take(4 * ((int64_t)d.groups + 1));
    auto& t = a.table[a.count++];
    t.size = size;
    t.least = least;
    t.before = t.slots = nullptr;
    if (size > 0) {
      t.before = (int32_t*)take(4 * ((int64_t)d.groups + 1));
      t.slots = (int32_t*)take(4 * (int64_t)d.groups);
    }
    return UnitTable{a.ends, t.before, t.slots};
  }
  int run_units(const int64_t* offsets, hipStream_t s) {
    UnitsArgs& a = unit_tables;
    if (a.count == 0) return FC_OK;
    a.offsets = offsets;
    a.rows = n;
    a.groups = d.groups;
    hipLaunchKernelGGL(dense_units_kernel, dim3(a.count), dim3(1024), 0, s, a);
    FC_LAUNCH_CHECK();
    return FC_OK;
  }
  void grouped(DenseJob& g, const void* offsets, int64_t b_stride, int64_t out_stride) const {
    g.offsets = (const int64_t*)offsets;
    g.groups = d.groups;
    g.rows = n;
    g.b_stride = b_stride;
    g.out_stride = out_stride;
  }
};

// Tile size of up to two products with groups, and the rows that a sum over rows takes at once (`sums`: a workgroup sums
// over a group's rows; otherwise its rows are outputs). By the costs of plan_launch, with even groups: of a group's rows half
// a tile is empty in the mean.
inline int plan_groups(DenseJob* rows, DenseJob* sums, const Dense& f) {
  const int cus = device_cu_count();
  const double groups = (double)(f.d.groups < f.n ? f.d.groups : f.n), each = f.n / groups;
  const int per = f.form == FORM_NATIVE ? 32 : f.form == FORM_8 ? 128 : 64, planes = f.form == FORM_PLANES ? 6 : 1;
  if (rows) rows->steps = steps_of(rows->A.k > rows->B.k ? rows->A.k : rows->B.k, f.form);
  const PlanKey key{{cus, -1, (int)f.form, (int)f.n, f.d.groups, rows ? rows->N : 0, rows ? rows->steps : 0, sums ? sums->M : 0,
                     sums ? sums->N : 0}};
  const PlanChoice choice = remembered(key, [&]() {
    int best_kind = 0;
    int64_t best_unit = 0;
    double best = 1e30;
    for (int kind = 0; kind < kKinds; ++kind) {
      if (f.form == FORM_NATIVE && kind == 2) continue;
      const TileCost& c = f.form == FORM_NATIVE ? kNativeCost[kind] : kTileCost[kind];
      const int bm = tile_rows(kind);
      double row_blocks = 0, row_load = 0, row_chain = 0, row_alone = 0;
      if (rows) {
        row_blocks = (f.n / (double)bm + 0.5 * groups) * cdiv(rows->N, bm);
        row_chain = rows->steps;
        row_load = row_blocks * (rows->steps * c.full + c.fused);
        row_alone = row_blocks * (rows->steps * c.step + kLatency[kind][!sums]);
      }
      for (int64_t unit = (f.n + per - 1) / per * per;;) {
        double blocks = row_blocks, load = row_load, chain = row_chain, alone = row_alone, extra = 0;
        if (sums) {
          const double tiles = (double)cdiv(sums->M, bm) * cdiv(sums->N, bm);
          const double parts = each > unit ? f.n / (double)unit + 0.5 * groups : groups;
          const double steps = planes * (each > unit ? (double)unit : each) / per;
          // (the groups are not even: the longest sum of an undivided group is taken as twice the mean)
          const double longest = planes * (double)(unit < 2 * each ? unit : 2 * each) / per;
          blocks += parts * tiles;
          load += parts * tiles * (steps * c.full + c.end) + (f.d.groups - groups) * tiles * c.end;
          alone += parts * tiles * (steps * c.step + kLatency[kind][0]);
          if (longest > chain) chain = longest;
          if (each * 2 > unit) extra = 8e-6 / 3 * (2.0 * f.n / unit) * sums->M * sums->N + 3.5;
        }
        const double shared = kShare[kind] * c.full, pace = blocks > cus && shared > c.step ? shared : c.step;
        const double longest = chain * pace + c.fused;
        load /= cus;
        if (blocks > cus) load *= 0.5 + 0.5 * (double)(int64_t)((blocks + cus - 1) / cus) * cus / blocks;
        double time = load > longest ? load : longest;
        const double rounds = (double)(int64_t)(blocks / (cus * kShare[kind]) + 1) / blocks;
        if (alone * rounds > time) time = alone * rounds;
        time += extra;
        if (time < best) {
          best = time;
          best_kind = kind;
          best_unit = unit;
        }
        if (!sums || unit <= 4 * per) break;
        unit = (unit / 2 + per - 1) / per * per;
      }
    }
    return PlanChoice{best_kind, {best_unit, 0}, best};
  });
  if (rows) {
    set_tiles(*rows, choice.kind, false);
    rows->splits = 1;
  }
  if (sums) {
    set_tiles(*sums, choice.kind, false);
    sums->splits = 1;
    sums->unit = (int32_t)choice.split[0];
  }
  return choice.kind;
}
// Workgroups that any offsets can need.
inline int64_t group_blocks(const DenseJob& g, int bm) {
  if (g.M == 0) return 0;
  if (g.unit > 0) return (g.rows / g.unit + g.groups) * g.tiles_m * g.tiles_n;
  return (g.rows / bm + g.groups) * g.tiles_n;
}
// Edge of the tiles of a backward pass with all gradients.
int dense_bwd_tile(const fc_dense_desc& d, int64_t n);
// Partial sums of groups of more than one unit: at most 2 rows / unit of them.
inline int64_t group_partial_bytes(const DenseJob& g) { return 4 * (2 * g.rows / g.unit) * g.M * g.N; }

}  // namespace fc
