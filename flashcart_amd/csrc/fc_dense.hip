// Dense layers forward (fc_dense.h), in three types, with one weight or one for each group of rows, and in 8 bits:
//   y = residual + c act(s (x_scale x) (w_scale W)^T + b)
// with e4m3 x and W, a float32 scale for each of their rows, and y in 16 bits.
//
// Bound by the matrix cores and the stores of y and act'(z) where n is large (16,384 x 2,048 x 5,632 bf16 372 us, 1,020
// TFLOP/s; 8,192 x 4,096 x 5,120 in 8 bits 159-173 us, 1,990-2,160 TFLOP/s; 16,384 rows over 32 experts of 2,048 x 2,816
// 254 us), by the weights' bytes where it is small (1 x 4,096 x 10,240 bf16 15 us, 5.6 TB/s; 64 rows over 64 experts of
// 2,048 x 1,024 41 us, 4.1 TB/s: repeated calls, whose weights the last-level cache holds in whole or in part; from memory the first
// takes 24 us, 3.5 TB/s).
#include "fc_dense_few.h"
#include "fc_dense_plan.h"

namespace fc {

template <class T, class MT, bool F32, class OT, bool GROUPS>
__global__ void __launch_bounds__(T::NT, 2) dense_fwd_kernel(DenseJob g) {
  __shared__ __attribute__((aligned(1024))) char lds0[T::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds1[T::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds2[T::STAGES > 2 ? T::STAGE : 1];
  __shared__ __attribute__((aligned(1024))) char lds3[T::STAGES > 2 ? T::STAGE : 1];
  lds_char *const l0 = (lds_char*)lds0, *const l1 = (lds_char*)lds1, *const l2 = (lds_char*)lds2;
  lds_char* const l3 = (lds_char*)lds3;
  const int block = g.first + blockIdx.x;
  if constexpr (GROUPS) {
    GroupTile<T, MT, F32, false, false, EPI_DENSE, OT>::run(g, block, g.blocks, l0, l1, l2, l3);
    return;
  }
  const int whole = g.tiles_m * g.tiles_n - g.halves;
  if constexpr (!GROUPS && T::BN == 256) {
    if (g.splits == 1 && block >= whole) {  // (tiles in the order of FfnTile::run)
      const int tile = whole + (block - whole) / 2, group = tile / (8 * g.tiles_n), in = tile - group * 8 * g.tiles_n;
      const int gm = min(8, g.tiles_m - group * 8), nt = in / gm * 2 + ((block - whole) & 1);
      if (nt * TileH::BN < g.N)
        FfnTile<TileH, MT, F32, false, false, EPI_DENSE, OT>::run_tile(g, group * 8 + in % gm, nt, 0, 0, g.steps, l0, l1, l2, l3);
      return;
    }
  }
  if constexpr (!GROUPS) FfnTile<T, MT, F32, false, false, EPI_DENSE, OT>::run(g, block, whole, l0, l1, l2, l3);
}

// ---- sums over the parts of a split K loop, with the epilogue ----
// A workgroup forms 256 / groups times 4 outputs: the lanes of an output add every groups-th part, their sums are added in
// order.
template <class MT, bool F32, class OT>
__global__ void __launch_bounds__(256) dense_sum_kernel(DenseJob g, int groups, int64_t first) {
  constexpr int ES = std::is_same_v<MT, float> ? 4 : 2;
  constexpr bool EIGHT = std::is_same_v<MT, e4m3_t>;
  __shared__ f32x4v part[256];
  const int per = 256 / groups, grp = threadIdx.x / per;
  const int64_t chunks = g.N / 4, t = (first + blockIdx.x) * per + threadIdx.x % per;
  const bool ok = t < g.M * chunks;
  const int64_t row = ok ? t / chunks : 0;
  const int col = ok ? (int)(t - row * chunks) * 4 : 0;
  f32x4v s{0.f, 0.f, 0.f, 0.f};
  const float* p = g.partial + row * g.N + col;
#pragma unroll 4
  for (int k = grp; k < g.splits; k += groups) s += *(const f32x4v*)(p + (int64_t)k * g.M * g.N);
  if (groups > 1) {
    part[threadIdx.x] = s;
    __syncthreads();
    if (grp == 0)
      for (int k = 1; k < groups; ++k) s += part[k * per + threadIdx.x];
  }
  if (!ok || grp > 0) return;
  float y[1][4], (&x)[4] = y[0];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    x[v] = s[v] * g.scale;
    if constexpr (F32) {
      if (!(fabsf(x[v]) < __builtin_inff())) {  // again, scaled before the sum, as where it is not split
        x[v] = 0.f;
        const int k_end = max(g.A.k, g.B.k), n = min(col + v, g.B.rows - 1);
        for (int k = 0; k < k_end; ++k)
          x[v] = fmaf(g.scale * value_of<ES, false>(g.A, row, k), value_of<ES, false>(g.B, n, k), x[v]);
      }
    }
  }
  DenseJob::Line<OT, F32, EIGHT, 4> line;
  line.init(g, row, col);
  line.template ahead<1>(g, true, row, 0);
  line.template finish<1>(g, true, row, 0, y);
}

struct DenseFwd {
  DenseJob job{};
  int kind = 0;
  bool few = false;
};
// Whether the kernel for few rows is faster than tiles. It reads x again for every 16 columns, and has less of the weight on
// its way than the tiles; it needs no copy of operands whose rows are not a multiple of 16 bytes. us, few / tiles, out of
// in -> out: bf16, one row 256 -> 512 3.4 / 4.8, 1,024 -> 4,096 4.4 / 6.8, 2,048 -> 8,192 11.6 / 9.8, 4,096 -> 10,240 20 / 16,
// 1,031 -> 4,096 8.0 / 15.8; 16 rows 4,097 -> 4,096 29 / 28; 32 rows 1,024 -> 4,096 6.1 / 6.8, 2,048 -> 1,024 8.6 / 8.9.
// float32, one row 2,048 -> 8,192 15 / 28, 4,096 -> 10,240 52 / 59, 4,096 -> 64 11.5 / 8.8; 32 rows 4,097 -> 4,096 29 / 53.
// Groups: 16 of 2,048 -> 1,024 with 64 rows 20 / 14, 64 of 1,031 -> 512 with 32 rows 24 / 39 and with 512 41 / 47,
// 8 of 4,099 -> 1,000 with 128 rows 66 / 41. (All with the weight in the last-level cache, from the call before.)
// 8 bits, weights from memory: one row 1,024 -> 10,240 5.6 / 6.5, 4,096 -> 4,096 6.8 / 12, 4,096 -> 10,240 13 / 16; 16 rows
// 2,048 -> 8,192 7.4 / 8.5, 4,096 -> 10,240 15 / 14, 8,192 -> 8,192 19 / 21; 32 rows 4,096 -> 4,096 9.4 / 12.5, 1,024 -> 10,240
// 9.1 / 6.7, 8,192 -> 1,024 14 / 11. Rows that are copied for tiles: 16 rows 4,097 -> 4,096 19 / 22, 8,195 -> 4,096 28 / 31,
// 4,097 -> 10,240 46 / 33; 32 rows 2,055 -> 4,096 13.5 / 17, 4,097 -> 4,096 28 / 23.
static bool few_rows(const Dense& f) {
  if (f.form == FORM_PLANES) return false;
  const bool direct = f.direct(f.in, f.ip);
  if (f.d.groups > 0) return !direct && f.n <= 8 * (int64_t)f.d.groups;
  if (f.n > kFewRows) return false;
  const int64_t blocks = (f.n + 15) / 16, k = blocks * f.in;
  if (f.form == FORM_8) {
    if (direct) return blocks == 1 || (f.in <= 4096 && f.out <= 4096);
    return f.in * f.out <= (blocks == 1 ? 5 << 23 : 1 << 24);
  }
  if (f.form == FORM_NATIVE) return k <= (direct ? 2048 : 16384) || (blocks == 1 && f.out >= 4096);
  return direct ? k <= 2048 && k * f.out <= 1 << 23 : k <= 4096;
}
static DenseFwd plan_dense(Dense& f, const void* x, const void* weight, const void* bias, const void* residual,
                           const void* offsets, void* y, void* saved) {
  DenseFwd p;
  DenseJob& g = p.job;
  p.few = few_rows(f);
  if (p.few) {
    g.A.p = (const char*)x;
    g.B.p = (const char*)weight;
    g.A.ld = g.B.ld = f.in;
    g.A.k = (int32_t)f.in;
  } else {
    g.A = view(f.x(x), f.n, f.ip);
    g.B = view(f.weight(weight), f.out, f.ip);
  }
  g.M = (int32_t)f.n;
  g.N = (int32_t)f.op;
  set_out(g, y, f.n, f.out, f.d.scale);
  g.bias = bias;
  g.residual = residual;
  g.act = f.d.act;
  g.act_scale = f.d.act_scale;
  g.factor = (char*)saved;
  g.factor_count = f.n * f.op;
  if (f.d.groups > 0) {
    f.grouped(g, offsets, f.out * (p.few ? f.in : f.ip), 0);
    if (p.few) g.table = f.units(0, 0);
    if (p.few) return p;
    p.kind = plan_groups(&g, nullptr, f);
    // Few rows a group: tiles of 32 rows, three of which a CU runs at once (64 experts of 2,048 -> 1,024, 64 and 1,024 rows,
    // bf16 45.6 -> 41.3 and 62 -> 56 us, 256 rows float32 146 -> 100; 8 experts of 4,096 -> 4,096, 64 rows, bf16 54 -> 58).
    const bool native = f.form == FORM_NATIVE;
    if (p.kind == 0 && f.n <= (native ? 64 : 16) * (int64_t)f.d.groups && (native || f.d.groups >= 16)) p.kind = 4;
    g.table = f.units(tile_rows(p.kind), 0);
    return p;
  }
  if (p.few) return p;
  DenseJob split = g;
  DenseJob *fused[] = {&g}, *parts[] = {&split};
  const bool no[] = {false}, yes[] = {true};
  double time, split_time;
  p.kind = plan_launch(fused, no, 1, f.form, false, true, &time);
  const int kind = plan_launch(parts, yes, 1, f.form, false, true, &split_time);
  if (split.splits > 1 && split_time < time) {
    g = split;
    p.kind = kind;
    g.partial = (float*)f.take(partial_bytes(g));
  }
  // The tiles of a last round that is at most half full as two halves of their columns each (16,384 x 2,048 x 5,632 bf16, 5.5
  // rounds: 398 -> 382 us; 8,192 x 4,096 x 5,120 in 8 bits, 2.5 rounds: 195 -> 184).
  if (p.kind == 2 && g.splits == 1) {
    const int tiles = g.tiles_m * g.tiles_n, cus = device_cu_count(), last = tiles % cus;
    if (tiles > cus && 2 * last <= cus) g.halves = last;
  }
  return p;
}

template <class MT, bool F32, class OT, bool GROUPS>
static int launch_tiles(DenseJob g, int kind, hipStream_t s) {
  const int64_t blocks = GROUPS ? group_blocks(g, tile_rows(kind)) : blocks_of(g) + g.halves;
  if (blocks > INT32_MAX) return FC_ERR_SHAPE;
  g.blocks = (int32_t)blocks;
  return in_launches(blocks, [&](int64_t first, unsigned count) {
    const dim3 grid(count);
    g.first = (int32_t)first;
    if constexpr (!std::is_same_v<MT, float>) {
      if (kind == 2) hipLaunchKernelGGL((dense_fwd_kernel<TileL, MT, F32, OT, GROUPS>), grid, dim3(TileL::NT), 0, s, g);
    }
    if constexpr (GROUPS) {
      if (kind == 4) hipLaunchKernelGGL((dense_fwd_kernel<TileR, MT, F32, OT, GROUPS>), grid, dim3(TileR::NT), 0, s, g);
    }
    if (kind == 3) hipLaunchKernelGGL((dense_fwd_kernel<TileX, MT, F32, OT, GROUPS>), grid, dim3(TileX::NT), 0, s, g);
    else if (kind == 1) hipLaunchKernelGGL((dense_fwd_kernel<TileM, MT, F32, OT, GROUPS>), grid, dim3(TileM::NT), 0, s, g);
    else if (kind == 0) hipLaunchKernelGGL((dense_fwd_kernel<TileS, MT, F32, OT, GROUPS>), grid, dim3(TileS::NT), 0, s, g);
  });
}

template <class MT, class OT, bool GROUPS>
static int launch_few(DenseJob g, hipStream_t s) {
  const int64_t blocks = (int64_t)(GROUPS ? g.groups : 1) * cdiv(g.n_out, 16);
  g.blocks = (int32_t)blocks;  // (below 2^27)
  return in_launches(blocks, [&](int64_t first, unsigned count) {
    const dim3 grid(count), block(64 * kFewWaves);
    g.first = (int32_t)first;
    if (GROUPS || g.M <= 16) hipLaunchKernelGGL((dense_few_kernel<MT, OT, 1, GROUPS>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((dense_few_kernel<MT, OT, 2, GROUPS>), grid, block, 0, s, g);
  });
}

template <class MT, bool F32, class OT>
static int launch_dense(const DenseFwd& p, hipStream_t s) {
  const DenseJob& g = p.job;
  if (p.few) {
    if constexpr (!(F32 && std::is_same_v<MT, bf16_t>)) {
      if constexpr (!std::is_same_v<MT, e4m3_t>) {
        if (g.groups > 0) return launch_few<MT, OT, true>(g, s);
      }
      return launch_few<MT, OT, false>(g, s);
    }
  }
  if constexpr (!std::is_same_v<MT, e4m3_t>) {
    if (g.groups > 0) return launch_tiles<MT, F32, OT, true>(g, p.kind, s);
  }
  const int r = launch_tiles<MT, F32, OT, false>(g, p.kind, s);
  if (r != FC_OK || g.splits == 1) return r;
  int groups = 1;
  while (groups < 16 && groups * 4 <= g.splits) groups *= 2;
  return in_launches(cdiv((int64_t)g.M * (g.N / 4), 256 / groups), [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL((dense_sum_kernel<MT, F32, OT>), dim3(blocks), dim3(256), 0, s, g, groups, first);
  });
}

}  // namespace fc

using namespace fc;

extern "C" int64_t fc_node_dense_saved(const fc_dense_desc* d, int64_t n) {
  const int st = dense_check(d, n);
  return st != FC_OK ? -st : Dense(*d, n, nullptr).factor_bytes();
}

extern "C" int64_t fc_node_dense_fwd_workspace(const fc_dense_desc* d, int64_t n) {
  const int st = dense_check(d, n);
  if (st != FC_OK) return -st;
  if (n == 0) return 0;
  Dense f(*d, n, nullptr);
  plan_dense(f, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  return f.at;
}

extern "C" int fc_node_dense_fwd(const fc_dense_desc* d, int64_t n, const void* x, const void* weight, const void* bias,
                                 const void* residual, const int64_t* offsets, void* y, void* saved, void* ws,
                                 int64_t ws_bytes, void* stream) {
  int st = dense_check(d, n);
  if (st != FC_OK) return st;
  if (d->groups > 0 && residual) return FC_ERR_BAD_DESC;
  if (n == 0) return FC_OK;
  if (!x || !weight || !y || (d->groups > 0 && !offsets)) return FC_ERR_NULL;
  if (d->aligned && !(aligned16(x) && aligned16(weight))) return FC_ERR_BAD_DESC;
  Dense f(*d, n, ws);
  const DenseFwd p = plan_dense(f, x, weight, bias, residual, offsets, y, d->act == ACT_NONE ? nullptr : saved);
  if (f.at > 0 && (!ws || ws_bytes < f.at)) return FC_ERR_WORKSPACE;
  if (!aligned16(saved) || !aligned16(ws)) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  st = f.run_units(offsets, s);
  if (st == FC_OK) st = f.run_pad(s);
  if (st != FC_OK) return st;
  return with_operand_form(d->dtype, f.form, [&](auto m, auto is32) -> int {
    using MT = decltype(m);
    constexpr bool F32 = decltype(is32)::value;
    return launch_dense<MT, F32, std::conditional_t<F32, float, MT>>(p, s);
  });
}

static int eight_check(const fc_dense_desc* d, int64_t n) {
  const int st = dense_check(d, n);
  return st != FC_OK ? st : d->groups != 0 || d->dtype == FC_F32 ? FC_ERR_BAD_DESC : FC_OK;
}

extern "C" int32_t fc_node_dense_tile(const fc_dense_desc* d, int64_t n, int32_t pass, int32_t* halves) {
  const int st = pass == 1 ? eight_check(d, n) : dense_check(d, n);
  if (st != FC_OK) return -st;
  if (pass < 0 || pass > 2) return -FC_ERR_BAD_DESC;
  if (n == 0) return -FC_ERR_SHAPE;
  if (halves) *halves = 0;
  fc_dense_desc desc = *d;
  desc.aligned = 1;
  if (pass == 2) return dense_bwd_tile(desc, n);
  Dense f(desc, n, nullptr, pass == 1);
  const DenseFwd p = plan_dense(f, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  if (halves && !p.few) *halves = p.job.halves;
  return p.few ? 0 : tile_rows(p.kind);
}

extern "C" int64_t fc_quantized_dense_workspace(const fc_dense_desc* d, int64_t n) {
  const int st = eight_check(d, n);
  if (st != FC_OK) return -st;
  if (n == 0) return 0;
  Dense f(*d, n, nullptr, true);
  plan_dense(f, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  return f.at;
}

extern "C" int fc_quantized_dense(const fc_dense_desc* d, int64_t n, const void* x, const float* x_scale,
                                  const void* weight, const float* weight_scale, const void* bias, const void* residual,
                                  void* y, void* ws, int64_t ws_bytes, void* stream) {
  int st = eight_check(d, n);
  if (st != FC_OK) return st;
  if (n == 0) return FC_OK;
  if (!x || !x_scale || !weight || !weight_scale || !y) return FC_ERR_NULL;
  if (d->aligned && !(aligned16(x) && aligned16(weight))) return FC_ERR_BAD_DESC;
  Dense f(*d, n, ws, true);
  DenseFwd p = plan_dense(f, x, weight, bias, residual, nullptr, y, nullptr);
  p.job.row_scale = x_scale;
  p.job.col_scale = weight_scale;
  if (f.at > 0 && (!ws || ws_bytes < f.at)) return FC_ERR_WORKSPACE;
  if (!aligned16(ws)) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  st = f.run_pad(s);
  if (st != FC_OK) return st;
  return d->dtype == FC_BF16 ? launch_dense<e4m3_t, false, bf16_t>(p, s) : launch_dense<e4m3_t, false, f16_t>(p, s);
}
