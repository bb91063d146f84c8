// Dense layers backward (fc_dense.h): dz and the bias' gradient in one pass over the incoming gradient, then the products
// for dx and dW in one launch, the one with the longer sums first. 16,384 x 2,048 x 5,632 bf16: dz 100 us (5.5 TB/s, bound by
// memory), products 645-661 us (1,149-1,170 TFLOP/s, the matrix cores busy 62%).
#include <algorithm>

#include "fc_dense_plan.h"

namespace fc {

// ---- dz = c g act'(z) as operand of the products, and the sums of its columns over 32 rows each ----
constexpr int kDzRows = 32, kDzCols = 256;

struct DzArgs {
  const void* grad;         // (n, out)
  const char* factor;       // act'(z), or null
  int64_t factor_count;
  char* dz;                 // (n, op) in the operands' form, or null
  int64_t plane;
  float* sums;              // (chunks, op), or null
  int32_t out, op, col_blocks;
  float act_scale;          // over the scale that act'(z) is kept with
  const int64_t* offsets;   // or null
  UnitTable table;
  int32_t groups;
  int64_t rows;
  int64_t first;            // workgroup of this launch
};

// A workgroup takes 32 rows (of one group) by 256 columns, a thread 8 columns of every 8th row, all loaded before the first is
// stored.
template <class T, class MT>
__global__ void __launch_bounds__(256) dense_dz_kernel(DzArgs a) {
  constexpr bool F32 = std::is_same_v<T, float>;
  constexpr int N = kDzRows / 8;
  __shared__ float part[8][kDzCols + 8];
  const int id = (int)(a.first + blockIdx.x), chunk = id / a.col_blocks, cb = id - chunk * a.col_blocks;
  int64_t r0 = (int64_t)chunk * kDzRows, r1 = min(r0 + kDzRows, a.rows);
  if (a.offsets) {
    const GroupUnit u = find_unit(a.offsets, a.table, a.groups, a.rows, kDzRows, 0, chunk, false);
    if (u.group < 0) return;
    r0 = u.row + (int64_t)u.index * kDzRows;
    r1 = min(r0 + kDzRows, u.row + u.rows);
  }
  const int cl = threadIdx.x % 32 * 8, col = cb * kDzCols + cl;
  float sum[8] = {};
  if (col < a.op) {
    const int64_t first = r0 + threadIdx.x / 32;
    Pack<T, 8> v[N];
    float d[N][8];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t r = min(first + 8 * k, r1 - 1);
      const T* p = (const T*)a.grad + r * a.out + col;
      if (col + 8 <= a.out) {
        v[k] = load_pack<T, 8>(p);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k].v[i] = col + i < a.out ? p[i] : T{};
      }
      if (a.factor) get_factor<T>(a.factor, r * a.op + col, a.factor_count, d[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t r = first + 8 * k;
      if (r >= r1) break;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = to_f32(v[k].v[i]);
        // (where act' is kept with a scale, after what takes that off; where not, first: no product leaves the range that stays
        // in it when the other comes first)
        if constexpr (!F32) x[i] *= a.act_scale;
        if (a.factor) x[i] = col + i < a.out ? x[i] * d[k][i] : 0.f;
        if constexpr (F32) x[i] *= a.act_scale;
        sum[i] += x[i];
      }
      if (a.dz) put<MT, F32, 8>(a.dz, r * a.op + col, a.plane, x);
    }
  }
  if (!a.sums) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[threadIdx.x / 32][cl + i] = sum[i];
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += part[k][threadIdx.x];
  const int c = cb * kDzCols + threadIdx.x;
  if (c < a.op) a.sums[(int64_t)chunk * a.op + c] = s;
}

// Sums over `size` rows each (of one group) made into sums over 64 times as many, in a fixed order. Of many rows the bias'
// gradient would be a long chain of additions otherwise, in few workgroups and with an error that grows with it (2^26 rows of 8
// columns 16.3 ms in place of 0.05, 2^20 of 128 0.26 ms in place of 0.008; the sum of 2^22 numbers 0.1 off by 1.5e-4).
constexpr int kFold = 64;
struct FoldArgs {
  const float* in;  // (chunks, op)
  float* out;
  int64_t chunks, rows, first;
  const int64_t* offsets;
  UnitTable from, to;  // of the units that are added, and of those that they become
  int32_t groups, op, col_blocks, size;
};
__global__ void __launch_bounds__(256) dense_fold_kernel(FoldArgs a) {
  const int id = (int)(a.first + blockIdx.x), unit = id / a.col_blocks;
  const int c = (id - unit * a.col_blocks) * 256 + threadIdx.x;
  int64_t c0 = (int64_t)unit * kFold, end = a.chunks;
  if (a.offsets) {
    const GroupUnit u = find_unit(a.offsets, a.to, a.groups, a.rows, a.size * kFold, 0, unit, false);
    if (u.group < 0) return;
    const int before = find_unit<true>(a.offsets, a.from, a.groups, a.rows, a.size, 0, u.group, false).before;
    c0 = before + (int64_t)u.index * kFold;
    end = before + (u.rows + a.size - 1) / a.size;
  }
  if (c >= a.op) return;
  const int64_t c1 = min(c0 + kFold, end);
  float s = 0.f;
#pragma unroll 8
  for (int64_t k = c0; k < c1; ++k) s += a.in[k * a.op + c];
  a.out[(int64_t)unit * a.op + c] = s;
}

// The bias' gradient, from the sums of `size` rows each: a workgroup of NT threads takes 32 columns of a group, whose chunks it
// adds in a fixed order.
struct DbArgs {
  const float* sums;  // (chunks, op)
  void* out;          // (groups, out), or null
  int64_t chunks, rows;
  const int64_t* offsets;
  UnitTable table;
  int32_t groups, n_out, op, size;
};
template <class T, int NT>
__device__ __forceinline__ void db_block(const DbArgs& a, int block, float (&part)[NT / 32][33]) {
  const int blocks = (a.n_out + 31) / 32, e = block / blocks, cl = threadIdx.x % 32, grp = threadIdx.x / 32;
  const int c = (block - e * blocks) * 32 + cl;
  int64_t c0 = 0, c1 = a.chunks;
  if (a.offsets) {
    const GroupUnit u = find_unit<true>(a.offsets, a.table, a.groups, a.rows, a.size, 0, e, false);
    c0 = u.before;
    c1 = c0 + (u.rows + a.size - 1) / a.size;
  }
  float s = 0.f;
  if (c < a.n_out) {
#pragma unroll 8
    for (int64_t k = c0 + grp; k < c1; k += NT / 32) s += a.sums[k * a.op + c];
  }
  part[grp][cl] = s;
  __syncthreads();
  if (grp > 0 || c >= a.n_out) return;
#pragma unroll
  for (int k = 1; k < NT / 32; ++k) s += part[k][cl];
  ((T*)a.out)[(int64_t)e * a.n_out + c] = from_f32<T>(s);
}
// (where neither dx nor dW is asked for; with them it is part of their launch)
template <class T>
__global__ void __launch_bounds__(1024) dense_db_kernel(DbArgs a, int first) {
  __shared__ float part[32][33];
  db_block<T, 1024>(a, first + blockIdx.x, part);
}

// ---- the products: g1 forms dW (sums over rows), g2 dx. The first `front` workgroups take the one with the longer sums; the
// workgroups from `products` on the bias' gradient ----
template <class T, class MT, bool F32, bool GROUPS>
__global__ void __launch_bounds__(T::NT, 2) dense_bwd_kernel(DenseJob g1, DenseJob g2, DbArgs db, int front, int products,
                                                                bool swapped, int first) {
  __shared__ __attribute__((aligned(1024))) char lds0[T::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds1[T::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds2[T::STAGES > 2 ? T::STAGE : 1];
  __shared__ __attribute__((aligned(1024))) char lds3[T::STAGES > 2 ? T::STAGE : 1];
  lds_char *const l0 = (lds_char*)lds0, *const l1 = (lds_char*)lds1, *const l2 = (lds_char*)lds2;
  lds_char* const l3 = (lds_char*)lds3;
  const int id = first + blockIdx.x;
  if (id >= products) {
    static_assert(T::STAGE >= T::NT / 32 * 33 * 4, "sums in a stage");
    db_block<std::conditional_t<F32, float, MT>, T::NT>(db, id - products, *(float (*)[T::NT / 32][33])lds0);
    return;
  }
  const bool in_front = id < front;
  const int block = in_front ? id : id - front, blocks = in_front ? front : products - front;
  if (in_front != swapped) {
    if constexpr (GROUPS) GroupTile<T, MT, F32, true, true, EPI_OUT>::run(g1, block, blocks, l0, l1, l2, l3);
    else FfnTile<T, MT, F32, true, true, EPI_OUT>::run(g1, block, l0, l1, l2, l3);
  } else {
    if constexpr (GROUPS) GroupTile<T, MT, F32, false, true, EPI_OUT>::run(g2, block, blocks, l0, l1, l2, l3);
    else FfnTile<T, MT, F32, false, true, EPI_OUT>::run(g2, block, l0, l1, l2, l3);
  }
}

// ---- sums over the parts of split sums: dW (first; with groups that alone) and dx ----
struct BwdSums {
  DenseJob job[2];
  int64_t base;      // first workgroup of the second
  int64_t first;     // workgroup of this launch
  int32_t lanes[2];  // that share the parts of an output
};
template <class MT, bool F32, bool GROUPS>
__global__ void __launch_bounds__(256) dense_bwd_sum_kernel(BwdSums a) {
  using OT = std::conditional_t<F32, float, MT>;
  constexpr int ES = std::is_same_v<MT, float> ? 4 : 2;
  __shared__ f32x4v part[256];
  const int64_t id = a.first + blockIdx.x;
  const bool dx = !GROUPS && id >= a.base;
  DenseJob g = a.job[dx];
  const int lanes = a.lanes[dx], per = 256 / lanes, grp = threadIdx.x / per;
  const int64_t chunks = g.N / 4;
  int64_t block = dx ? id - a.base : id;
  if constexpr (GROUPS) {
    const int64_t each = (g.M * chunks + per - 1) / per;
    const int e = (int)(block / each);
    block -= e * each;
    const GroupUnit u = find_unit<true>(g.offsets, g.table, g.groups, g.rows, g.unit, 1, e, false);
    if (u.rows <= g.unit) return;
    g.splits = (int)((u.rows + g.unit - 1) / g.unit);
    g.partial += (int64_t)u.slot * g.M * g.N;
    g.A.p += ES * u.row * g.A.ld;
    g.B.p += ES * u.row * g.B.ld;
    g.A.k = g.B.k = (int)u.rows;
    g.out = (OT*)g.out + e * g.out_stride;
  }
  const int64_t t = block * per + threadIdx.x % per;
  const bool ok = t < g.M * chunks;
  const int64_t row = ok ? t / chunks : 0;
  const int col = ok ? (int)(t - row * chunks) * 4 : 0;
  f32x4v s{0.f, 0.f, 0.f, 0.f};
  const float* p = g.partial + row * g.N + col;
#pragma unroll 4
  for (int k = grp; k < g.splits; k += lanes) s += *(const f32x4v*)(p + (int64_t)k * g.M * g.N);
  if (lanes > 1) {
    part[threadIdx.x] = s;
    __syncthreads();
    if (grp == 0)
      for (int k = 1; k < lanes; ++k) s += part[k * per + threadIdx.x];
  }
  if (!ok || grp > 0 || row >= g.m_out) return;
  OT* const out = (OT*)g.out + row * g.ld_out;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    if (col + v >= g.n_out) continue;
    float x = s[v] * g.scale;
    if constexpr (F32) {
      if (!(fabsf(x) < __builtin_inff())) {  // again, scaled before the sum, as where it is not split
        x = 0.f;
        const int k_end = max(g.A.k, g.B.k), m = (int)row, n = col + v;
        for (int k = 0; k < k_end; ++k) {
          const float u = dx ? value_of<ES, false>(g.A, m, k) : value_of<ES, true>(g.A, m, k);
          x = fmaf(g.scale * u, value_of<ES, true>(g.B, n, k), x);
        }
      }
    }
    out[col + v] = from_f32<OT>(x);
  }
}

struct DenseBwd {
  DzArgs dz{};
  bool run_dz = false;
  int64_t chunks = 0;
  FoldArgs fold[2]{};
  int folds = 0;
  DbArgs db{};
  DenseJob dw{}, dx{};  // (absent where M = 0)
  int kind = 0;
};
static DenseBwd plan_dense_bwd(Dense& f, const void* grad, const void* x, const void* weight, const void* saved,
                               const void* offsets, int need, void* gx, void* gw) {
  DenseBwd p;
  const bool nx = need & 1, nw = need & 2, nb = need & 4, groups = f.d.groups > 0;
  const bool factor = f.d.act != ACT_NONE, plain = !factor && f.d.act_scale == 1.f && f.direct(f.out, f.op);
  p.chunks = (f.n + kDzRows - 1) / kDzRows;
  if (groups && nb) p.chunks = f.n / kDzRows + f.d.groups;
  Opnd dz{};
  dz.ld = f.op;
  dz.plane = f.n * f.op;
  dz.p = (const char*)grad;
  DzArgs& a = p.dz;
  if ((nx || nw) && !plain) {
    a.dz = f.take(f.esize * dz.plane);
    dz.p = a.dz;
    p.run_dz = true;
  }
  if (nb) {
    a.sums = (float*)f.take(4 * p.chunks * f.op);
    p.run_dz = true;
    if (groups) {
      a.offsets = (const int64_t*)offsets;
      a.groups = f.d.groups;
      a.table = f.units(kDzRows, 0);
    }
  }
  a.grad = grad;
  a.factor = factor ? (const char*)saved : nullptr;
  a.factor_count = a.plane = f.n * f.op;
  a.out = (int32_t)f.out;
  a.op = (int32_t)f.op;
  a.col_blocks = cdiv(f.op, kDzCols);
  if (nb) {
    DbArgs& b = p.db;
    b = DbArgs{a.sums, nullptr, p.chunks, f.n, a.offsets, a.table, f.d.groups, (int32_t)f.out, (int32_t)f.op, kDzRows};
    // A chain of up to 256 additions for each of 8 lanes is left; two folds are enough for 2^27 rows. Backward without and with a
    // fold, us: 40,000 x 128 x 128 bf16 58 / 61, 60,000 x 64 x 1,024 bf16 125 / 123, 80,000 x 512 x 128 bf16 74 / 69, 131,072 x
    // 128 x 128 float32 140 / 129.
    for (; f.n > 2048 * (int64_t)b.size; ++p.folds) {
      const int64_t chunks = groups ? f.n / (b.size * kFold) + f.d.groups : (b.chunks + kFold - 1) / kFold;
      float* const out = (float*)f.take(4 * chunks * f.op);
      const UnitTable to = groups ? f.units(b.size * kFold, 0) : UnitTable{};
      p.fold[p.folds] = FoldArgs{b.sums, out, b.chunks, f.n, 0, a.offsets, b.table, to, f.d.groups, (int32_t)f.op, a.col_blocks, b.size};
      b.sums = out;
      b.chunks = chunks;
      b.size *= kFold;
      b.table = to;
    }
  }
  a.act_scale = f.d.act_scale / (factor && f.d.dtype == FC_BF16 ? kFactorScale<bf16_t> : 1.f);
  a.rows = f.n;
  if (nx) {
    DenseJob& g = p.dx;
    g.A = view(dz, f.n, f.op);
    g.B = view(f.weight(weight), f.ip, f.out);
    g.M = (int32_t)f.n;
    g.N = (int32_t)f.ip;
    set_out(g, gx, f.n, f.in, f.d.scale);
    g.b_tr = 1;
    if (groups) f.grouped(g, offsets, f.out * f.ip, 0);
  }
  if (nw) {
    DenseJob& g = p.dw;
    g.A = view(dz, f.op, f.n);
    g.B = view(f.x(x), f.ip, f.n);
    g.M = (int32_t)f.op;
    g.N = (int32_t)f.ip;
    set_out(g, gw, f.out, f.in, f.d.scale);
    g.a_tr = g.b_tr = 1;
    if (groups) f.grouped(g, offsets, 0, f.out * f.in);
  }
  if (!nx && !nw) return p;
  if (groups) {
    p.kind = plan_groups(nx ? &p.dx : nullptr, nw ? &p.dw : nullptr, f);
    if (nx) p.dx.table = f.units(tile_rows(p.kind), 0);
    if (nw) p.dw.table = f.units(p.dw.unit, 1);
    if (nw && p.dw.unit < f.n) p.dw.partial = (float*)f.take(group_partial_bytes(p.dw));
    return p;
  }
  DenseJob* jobs[] = {&p.dw, &p.dx};
  const bool yes[] = {true, true};
  double time;
  p.kind = plan_launch(jobs, yes, 2, f.form, false, true, &time);
  for (DenseJob* g : jobs) g->partial = (float*)f.take(g->M > 0 ? partial_bytes(*g) : 0);
  return p;
}

int dense_bwd_tile(const fc_dense_desc& d, int64_t n) {
  Dense f(d, n, nullptr);
  return tile_rows(plan_dense_bwd(f, nullptr, nullptr, nullptr, nullptr, nullptr, 7, nullptr, nullptr).kind);
}

template <class MT, bool F32, bool GROUPS>
static int launch_products(const DenseBwd& p, const DbArgs& db, hipStream_t s) {
  const DenseJob &g1 = p.dw, &g2 = p.dx;
  const int bm = tile_rows(p.kind);
  const int64_t blocks1 = g1.M == 0 ? 0 : GROUPS ? group_blocks(g1, bm) : blocks_of(g1);
  const int64_t blocks2 = g2.M == 0 ? 0 : GROUPS ? group_blocks(g2, bm) : blocks_of(g2), blocks = blocks1 + blocks2;
  const int64_t db_blocks = db.out ? (int64_t)(GROUPS ? db.groups : 1) * cdiv(db.n_out, 32) : 0;
  if (blocks + db_blocks > INT32_MAX) return FC_ERR_SHAPE;
  const int products = (int)blocks;
  // With groups: of one of twice the mean size, in steps of 64 k in every form. (In float32 a step is 32 k, or there are six to
  // 64; priced so, dW goes in front more often, which costs: 16,384 x 128 x 512 over 64 groups 88 -> 98 us, 16,384 x 1,024 x 1,024
  // over 8 516 -> 530; 25,000 x 256 x 256 over 8 91 -> 90.)
  const int64_t most = GROUPS && g1.M > 0 ? std::min<int64_t>(g1.unit, 2 * g1.rows / g1.groups) : 0;
  const int steps1 = g1.M == 0 ? 0 : GROUPS ? (int)most / 64 : g1.steps / g1.splits;
  const bool swapped = blocks2 > 0 && (blocks1 == 0 || g2.steps / g2.splits > steps1);
  const int front = (int)(swapped ? blocks2 : blocks1);
  const int st = in_launches(blocks + db_blocks, [&](int64_t first, unsigned count) {
    const dim3 grid(count);
    if constexpr (!std::is_same_v<MT, float>) {
      if (p.kind == 2)
        hipLaunchKernelGGL((dense_bwd_kernel<TileL, MT, F32, GROUPS>), grid, dim3(TileL::NT), 0, s, g1, g2, db, front,
                           products, swapped, (int)first);
    }
    if (p.kind == 1)
      hipLaunchKernelGGL((dense_bwd_kernel<TileM, MT, F32, GROUPS>), grid, dim3(TileM::NT), 0, s, g1, g2, db, front,
                         products, swapped, (int)first);
    else if (p.kind == 3)
      hipLaunchKernelGGL((dense_bwd_kernel<TileX, MT, F32, GROUPS>), grid, dim3(TileX::NT), 0, s, g1, g2, db, front,
                         products, swapped, (int)first);
    else if (p.kind == 0)
      hipLaunchKernelGGL((dense_bwd_kernel<TileS, MT, F32, GROUPS>), grid, dim3(TileS::NT), 0, s, g1, g2, db, front,
                         products, swapped, (int)first);
  });
  if (st != FC_OK) return st;
  // the sums of split sums
  BwdSums a{};
  int64_t sum_blocks = 0;
  auto add = [&](int q, const DenseJob& g, int splits, int64_t times) {
    int lanes = 1;
    while (lanes < 16 && lanes * 4 <= splits) lanes *= 2;
    a.job[q] = g;
    a.lanes[q] = lanes;
    sum_blocks += times * cdiv((int64_t)g.M * (g.N / 4), 256 / lanes);
  };
  if (GROUPS) {
    if (g1.M > 0 && g1.unit < g1.rows) add(0, g1, cdiv(g1.rows, (int64_t)g1.unit * g1.groups), g1.groups);
    a.base = sum_blocks;
  } else {
    if (g1.M > 0 && g1.splits > 1) add(0, g1, g1.splits, 1);
    a.base = sum_blocks;
    if (g2.M > 0 && g2.splits > 1) add(1, g2, g2.splits, 1);
  }
  return in_launches(sum_blocks, [&](int64_t first, unsigned count) {
    a.first = first;
    hipLaunchKernelGGL((dense_bwd_sum_kernel<MT, F32, GROUPS>), dim3(count), dim3(256), 0, s, a);
  });
}

}  // namespace fc

using namespace fc;

extern "C" int64_t fc_node_dense_bwd_workspace(const fc_dense_desc* d, int64_t n, int32_t need_x, int32_t need_weight,
                                               int32_t need_bias) {
  const int st = dense_check(d, n);
  if (st != FC_OK) return -st;
  if (n == 0) return 0;
  Dense f(*d, n, nullptr);
  plan_dense_bwd(f, nullptr, nullptr, nullptr, nullptr, nullptr,
                 (need_x != 0) | 2 * (need_weight != 0) | 4 * (need_bias != 0), nullptr, nullptr);
  return f.at;
}

extern "C" int fc_node_dense_bwd(const fc_dense_desc* d, int64_t n, const void* grad, const void* x, const void* weight,
                                 const void* saved, const int64_t* offsets, void* gx, void* gw, void* gb, void* ws,
                                 int64_t ws_bytes, void* stream) {
  int st = dense_check(d, n);
  if (st != FC_OK) return st;
  const int need = (gx != nullptr) | 2 * (gw != nullptr) | 4 * (gb != nullptr);
  if (n == 0 || need == 0) return n == 0 && (gw || gb) ? FC_ERR_SHAPE : FC_OK;
  if (!grad || (gx && !weight) || (gw && !x) || (d->act != ACT_NONE && !saved) || (d->groups > 0 && !offsets))
    return FC_ERR_NULL;
  if (d->aligned && !(aligned16(grad) && aligned16(x) && aligned16(weight))) return FC_ERR_BAD_DESC;
  Dense f(*d, n, ws);
  const DenseBwd p = plan_dense_bwd(f, grad, x, weight, saved, offsets, need, gx, gw);
  if (f.at > 0 && (!ws || ws_bytes < f.at)) return FC_ERR_WORKSPACE;
  if (!aligned16(saved) || !aligned16(ws)) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  st = f.run_units((const int64_t*)offsets, s);
  if (st == FC_OK) st = f.run_pad(s);
  if (st != FC_OK) return st;
  return with_operand_form(d->dtype, f.form, [&](auto m, auto is32) -> int {
    using MT = decltype(m);
    constexpr bool F32 = decltype(is32)::value;
    using T = std::conditional_t<F32, float, MT>;
    if (p.run_dz) {
      const int64_t blocks = p.chunks * p.dz.col_blocks;
      if (blocks > INT32_MAX) return FC_ERR_SHAPE;
      DzArgs a = p.dz;
      const int r = in_launches(blocks, [&](int64_t first, unsigned count) {
        a.first = first;
        hipLaunchKernelGGL((dense_dz_kernel<T, MT>), dim3(count), dim3(256), 0, s, a);
      });
      if (r != FC_OK) return r;
    }
    DbArgs db = p.db;
    db.out = gb;
    for (int k = 0; k < p.folds; ++k) {
      FoldArgs a = p.fold[k];
      const int64_t units = k + 1 < p.folds ? p.fold[k + 1].chunks : db.chunks;
      if (units * a.col_blocks > INT32_MAX) return FC_ERR_SHAPE;
      const int r = in_launches(units * a.col_blocks, [&](int64_t first, unsigned count) {
        a.first = first;
        hipLaunchKernelGGL(dense_fold_kernel, dim3(count), dim3(256), 0, s, a);
      });
      if (r != FC_OK) return r;
    }
    if (!gx && !gw) {
      const int64_t blocks = (int64_t)(f.d.groups > 0 ? f.d.groups : 1) * cdiv(f.out, 32);
      return in_launches(blocks, [&](int64_t first, unsigned count) {
        hipLaunchKernelGGL((dense_db_kernel<T>), dim3(count), dim3(1024), 0, s, db, (int)first);
      });
    }
    return d->groups > 0 ? launch_products<MT, F32, true>(p, db, s) : launch_products<MT, F32, false>(p, db, s);
  });
}
