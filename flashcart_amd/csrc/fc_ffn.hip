// Gated feed-forward block: [gate | up] = s_in x W_in^T, a = c act(gate), h = a up, y = s_out h W_out^T, and its gradients
//   dh = s_out g W_out,  d up = dh a,  d gate = dh b  with b = c act'(gate) up,
//   dx = s_in [d gate | d up] W_in,  dW_in = s_in [d gate | d up]^T x,  dW_out = s_out g^T h.
// Two products forward (the first forms gate and up of the same hidden columns in one workgroup and applies the
// activation and the product in its epilogue), four backward (the first applies the factors a and b, kept from the
// forward pass, in its epilogue). In 16-bit types h and [d gate | d up] are rounded to the type between the products, as
// operands of the matrix instructions, and the factors a and b are kept with 16 significant bits; everything else is
// float32 until an output is rounded.
//
// Bound by the matrix cores where n is large (16,384 x 2,048 x 5,632 in bf16, forward and backward: 2.83-3.0 ms, 1,130-1,200
// TFLOP/s, the cores busy 57-72%), by the weights' bytes where it is small (1 x 4,096 x 10,240: 61 us, 4.1 TB/s).
#include "fc_gemm_plan.h"

namespace fc {

// ---- operands whose rows are not a multiple of 16 bytes, and those in planes: a padded copy ----
struct PrepItem {
  const void* src;
  char* dst;
  int64_t cols, ld, plane;  // of src; of dst
  int32_t rows, rows_out, gap_at, gap;  // dst row r is src row r (r < gap_at) or r - gap (r >= gap_at + gap), else zeros
  int64_t block_base;
};
struct PrepArgs {
  PrepItem it[4];
  int32_t count;
  int64_t first;  // block of this launch
};

template <class T, class MT>
__global__ void __launch_bounds__(256) ffn_prep_kernel(PrepArgs a) {
  int k = 0;
  const int64_t block = a.first + blockIdx.x;
#pragma unroll
  for (int q = 1; q < 4; ++q)
    if (q < a.count && block >= a.it[q].block_base) k = q;
  const PrepItem& it = a.it[k];
  const int64_t chunks = it.ld / 8, t = (block - it.block_base) * 256 + threadIdx.x;
  if (t >= it.rows_out * chunks) return;
  const int64_t row = t / chunks, c0 = (t - row * chunks) * 8;
  int64_t from = row < it.gap_at ? row : row < it.gap_at + it.gap ? -1 : row - it.gap;
  if (from >= it.rows) from = -1;
  float x[8];
  const T* src = (const T*)it.src + from * it.cols + c0;
  if (from >= 0 && c0 + 8 <= it.cols) {
    const Pack<T, 8> v = load_pack<T, 8>(src);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = from >= 0 && c0 + i < it.cols ? to_f32(src[i]) : 0.f;
  }
  put<MT, std::is_same_v<T, float>, 8>(it.dst, row * it.ld + c0, it.plane, x);
}

// ---- sums over the parts of split K loops ----
struct SumArgs {
  FfnJob job[3];
  int32_t base[3];    // first workgroup of each
  int32_t groups[3];  // lanes that share the parts of an output
  int32_t count;
};

// A workgroup forms 256 / groups times 4 outputs: the lanes of an output add every groups-th part, their sums are added in
// order. Where the product has an epilogue of its own, it follows here; with the gate's, a lane's second output is the other
// projection's.
template <class MT, bool F32>
__global__ void __launch_bounds__(256) ffn_sum_kernel(SumArgs a) {
  using OT = std::conditional_t<F32, float, MT>;
  constexpr int ES = std::is_same_v<MT, float> ? 4 : 2;
  __shared__ f32x4v part[256];
  int which = 0;
#pragma unroll
  for (int q = 1; q < 3; ++q)
    if (q < a.count && (int)blockIdx.x >= a.base[q]) which = q;
  const FfnJob& g = a.job[which];
  const int groups = a.groups[which], per = 256 / groups, grp = threadIdx.x / per;
  const int cols = g.finish == EPI_GATE ? g.N / 2 : g.N;
  const int64_t chunks = cols / 4, t = (int64_t)(blockIdx.x - a.base[which]) * per + threadIdx.x % per;
  const bool ok = t < g.M * chunks;
  int64_t row = ok ? t / chunks : 0;
  const int col = ok ? (int)(t - row * chunks) * 4 : 0;
  // the sums, scaled; every lane of the workgroup takes part
  auto total = [&](int c, float (&x)[4]) {
    f32x4v s{0.f, 0.f, 0.f, 0.f};
    const float* p = g.partial + row * g.N + c;
#pragma unroll 4
    for (int k = grp; k < g.splits; k += groups) s += *(const f32x4v*)(p + (int64_t)k * g.M * g.N);
    if (groups > 1) {
      part[threadIdx.x] = s;
      __syncthreads();
      if (grp == 0)
        for (int k = 1; k < groups; ++k) s += part[k * per + threadIdx.x];
      __syncthreads();
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      x[v] = s[v] * g.scale;
      if constexpr (F32) {
        if (ok && grp == 0 && !(fabsf(x[v]) < __builtin_inff())) {  // again, as where the sum is not split
          x[v] = 0.f;
          const int k_end = max(g.A.k, g.B.k), m = (int)row, n = min(c + v, g.B.rows - 1);
          for (int k = 0; k < k_end; ++k) {
            const float u = g.a_tr ? value_of<ES, true>(g.A, m, k) : value_of<ES, false>(g.A, m, k);
            const float w = g.b_tr ? value_of<ES, true>(g.B, n, k) : value_of<ES, false>(g.B, n, k);
            x[v] = fmaf(g.scale * u, w, x[v]);
          }
        }
      }
    }
  };
  float x[4];
  total(col, x);
  if (g.finish == EPI_GATE) {
    float up[4];
    total(cols + col, up);
    if (ok && grp == 0) finish_gate<MT, F32, 4>(g, row, col, cols, x, up);
    return;
  }
  if (!ok || grp > 0) return;
  if (g.finish == EPI_DH) {
    Factors<F32, 4> f;
    f.load(g.saved, row * g.N + col, (int64_t)g.M * g.N);
    finish_dh<MT, F32, 4>(g, row, col, f, x);
    return;
  }
  if (row >= g.gap_at) {
    if (row < g.gap_at + g.gap) return;
    row -= g.gap;
  }
  if (row >= g.m_out) return;
  OT* out = (OT*)g.out + row * g.ld_out;
#pragma unroll
  for (int v = 0; v < 4; ++v)
    if (col + v < g.n_out) out[col + v] = from_f32<OT>(x[v]);
}

// The products of one launch. The first `front` workgroups take the one with the longer sums, g1 or (swapped) g2, the others
// the other one.
template <class T, class MT, bool F32, bool ATR1, bool BTR1, int EPI1, bool ATR2, bool BTR2, int EPI2>
__global__ void __launch_bounds__(T::NT, 2) ffn_gemm_kernel(FfnJob g1, FfnJob g2, int front, bool swapped) {
  __shared__ __attribute__((aligned(1024))) char lds0[T::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds1[T::STAGE];
  __shared__ __attribute__((aligned(1024))) char lds2[T::STAGES > 2 ? T::STAGE : 1];
  __shared__ __attribute__((aligned(1024))) char lds3[T::STAGES > 2 ? T::STAGE : 1];
  lds_char *const l0 = (lds_char*)lds0, *const l1 = (lds_char*)lds1, *const l2 = (lds_char*)lds2;
  lds_char* const l3 = (lds_char*)lds3;
  constexpr bool SAME = ATR1 == ATR2 && BTR1 == BTR2 && EPI1 == EPI2;
  const bool in_front = (int)blockIdx.x < front;
  const int block = in_front ? blockIdx.x : blockIdx.x - front;
  if (SAME || in_front != swapped) {
    FfnTile<T, MT, F32, ATR1, BTR1, EPI1>::run(g1, block, l0, l1, l2, l3);
  } else {
    if constexpr (!SAME) FfnTile<T, MT, F32, ATR2, BTR2, EPI2>::run(g2, block, l0, l1, l2, l3);
  }
}

// One launch of up to two products (the second may have no outputs).
template <class MT, bool F32, bool ATR1, bool BTR1, int EPI1, bool ATR2 = ATR1, bool BTR2 = BTR1, int EPI2 = EPI1>
static int launch(const FfnJob& g1, const FfnJob& g2, int kind, hipStream_t s) {
  const int64_t blocks1 = g1.M > 0 ? blocks_of(g1) : 0, blocks2 = g2.M > 0 ? blocks_of(g2) : 0, blocks = blocks1 + blocks2;
  if (!grid_fits(blocks, 512)) return FC_ERR_SHAPE;
  if (blocks == 0) return FC_OK;
  const dim3 grid((unsigned)blocks);
  const bool swapped = blocks2 > 0 && (blocks1 == 0 || g2.steps / g2.splits > g1.steps / g1.splits);
  const int front = (int)(swapped ? blocks2 : blocks1);
  if constexpr (!std::is_same_v<MT, float>) {
    if (kind == 2) {
      hipLaunchKernelGGL((ffn_gemm_kernel<TileL, MT, F32, ATR1, BTR1, EPI1, ATR2, BTR2, EPI2>), grid, dim3(TileL::NT), 0,
                         s, g1, g2, front, swapped);
      FC_LAUNCH_CHECK();
      return FC_OK;
    }
  }
  if (kind == 1)
    hipLaunchKernelGGL((ffn_gemm_kernel<TileM, MT, F32, ATR1, BTR1, EPI1, ATR2, BTR2, EPI2>), grid, dim3(TileM::NT), 0, s,
                       g1, g2, front, swapped);
  else
    hipLaunchKernelGGL((ffn_gemm_kernel<TileS, MT, F32, ATR1, BTR1, EPI1, ATR2, BTR2, EPI2>), grid, dim3(TileS::NT), 0, s,
                       g1, g2, front, swapped);
  FC_LAUNCH_CHECK();
  return FC_OK;
}

// The sums of the products with a split K loop, in one launch.
template <class MT, bool F32>
static int launch_sums(const FfnJob* const* jobs, int count, hipStream_t s) {
  SumArgs a{};
  int64_t blocks = 0;
  for (int q = 0; q < count; ++q) {
    const FfnJob& g = *jobs[q];
    if (g.M == 0 || g.splits <= 1) continue;
    int groups = 1;
    while (groups < 16 && groups * 4 <= g.splits) groups *= 2;
    a.base[a.count] = (int32_t)blocks;
    a.groups[a.count] = groups;
    a.job[a.count++] = g;
    blocks += cdiv((int64_t)g.M * ((g.finish == EPI_GATE ? g.N / 2 : g.N) / 4), 256 / groups);
  }
  if (blocks == 0) return FC_OK;
  if (!grid_fits(blocks, 256)) return FC_ERR_SHAPE;
  hipLaunchKernelGGL((ffn_sum_kernel<MT, F32>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  FC_LAUNCH_CHECK();
  return FC_OK;
}

// float32 in planes where the products are large and the operands are used often enough for their splitting to pay.
// Forward and backward, us, planes against native: 8,192 x 2,048 x 4,096 5,850 / 9,100, 2,048 x 1,024 x 2,048 542 / 719,
// 1,024 x 1,024 x 2,048 326 / 373, 4,096 x 512 x 1,024 345 / 377, 583 x 736 x 3,680 352 / 347, 25,000 x 128 x 512 411 / 393,
// 2,520 x 256 x 768 161 / 133, 512 x 512 x 512 84 / 62.
static Form form_of(const fc_ffn_desc& d, int64_t n) {
  if (d.dtype != FC_F32) return FORM_16;
  const bool large = n >= 512 && d.width >= 512 && d.hidden >= 512 && (double)n * d.width * d.hidden >= 2e9;
  return large ? FORM_PLANES : FORM_NATIVE;
}

// What is where, for one call; pointers are null where only sizes are asked for.
struct Ffn {
  const fc_ffn_desc& d;
  int64_t n, w, hid, wp, hp;
  Form form;
  int64_t esize;  // bytes of an element of an operand, over all planes
  char* ws;
  int64_t at = 0;
  PrepArgs prep{};
  int64_t prep_blocks = 0;

  Ffn(const fc_ffn_desc& desc, int64_t rows, void* workspace)
      : d(desc), n(rows), w(desc.width), hid(desc.hidden), wp(up8(w)), hp(up8(hid)), form(form_of(desc, rows)),
        esize(form == FORM_16 ? 2 : form == FORM_NATIVE ? 4 : 6), ws((char*)workspace) {}

  char* take(int64_t bytes) {
    char* p = ws + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
  // (rows, cols) of the caller as an operand: itself, or its padded copy of rows_out rows
  Opnd operand(const void* src, int64_t rows, int64_t cols, int64_t rows_out, int64_t gap_at) {
    const int64_t ld = up8(cols);
    Opnd o{};
    o.ld = ld;
    if (form != FORM_PLANES && d.aligned && ld == cols && rows == rows_out) {
      o.p = (const char*)src;
      return o;
    }
    PrepItem& it = prep.it[prep.count++];
    o.plane = rows_out * ld;
    it.src = src;
    it.dst = take(esize * o.plane);
    it.cols = cols;
    it.ld = ld;
    it.plane = o.plane;
    it.rows = (int32_t)rows;
    it.rows_out = (int32_t)rows_out;
    it.gap_at = (int32_t)gap_at;
    it.gap = (int32_t)(gap_at < rows_out ? (rows_out - rows) / 2 : 0);
    it.block_base = prep_blocks;
    prep_blocks += (o.plane / 8 + 255) / 256;
    o.p = it.dst;
    return o;
  }
  Opnd x(const void* p) { return operand(p, n, w, n, INT32_MAX); }
  Opnd w_out(const void* p) { return operand(p, w, hid, w, INT32_MAX); }
  Opnd w_in(const void* p) { return operand(p, 2 * hid, w, 2 * hp, hid); }
  int run_prep(hipStream_t s) {
    if (prep.count == 0) return FC_OK;
    return in_launches(prep_blocks, [&](int64_t first, unsigned blocks) {
      prep.first = first;
      const dim3 grid(blocks), block(256);
      if (d.dtype == FC_BF16) hipLaunchKernelGGL((ffn_prep_kernel<bf16_t, bf16_t>), grid, block, 0, s, prep);
      else if (d.dtype == FC_F16) hipLaunchKernelGGL((ffn_prep_kernel<f16_t, f16_t>), grid, block, 0, s, prep);
      else if (form == FORM_NATIVE) hipLaunchKernelGGL((ffn_prep_kernel<float, float>), grid, block, 0, s, prep);
      else hipLaunchKernelGGL((ffn_prep_kernel<float, bf16_t>), grid, block, 0, s, prep);
    });
  }
  int64_t h_bytes() const { return esize * n * hp; }
  int64_t factor_bytes() const { return (form == FORM_16 ? 6 : 8) * n * hp; }
};

static int ffn_check(const fc_ffn_desc* d, int64_t n) {
  if (!d) return FC_ERR_NULL;
  if (!node_dtype_ok(d->dtype) || d->act < 0 || d->act > 2) return FC_ERR_BAD_DESC;
  if (d->width < 1 || d->hidden < 1 || d->width > (1 << 20) || d->hidden > (1 << 20) || n < 0 || n > 0x7ffffff)
    return FC_ERR_SHAPE;
  return FC_OK;
}

struct FfnFwd {
  FfnJob gate{}, out{};
  int gate_kind, out_kind;
};
static FfnFwd plan_fwd(Ffn& f, const void* x, const void* w_in, const void* w_out, void* saved, void* y) {
  FfnFwd p;
  const Opnd ox = f.x(x), oi = f.w_in(w_in), oo = f.w_out(w_out);
  char* keep = saved ? (char*)saved : f.take(f.h_bytes());
  FfnJob& g = p.gate;
  g.A = view(ox, f.n, f.wp);
  g.B = view(oi, f.hp, f.wp);
  g.M = (int32_t)f.n;
  g.N = (int32_t)f.hp;
  g.n_out = (int32_t)f.hid;
  g.scale = f.d.scale_in;
  g.h = keep;
  g.h_plane = f.n * f.hp;
  g.saved = saved ? keep + f.h_bytes() : nullptr;
  g.act = f.d.act;
  g.act_scale = f.d.act_scale;
  {
    // few tiles and long sums: as a plain product with a split K loop, the activation after the sum of its parts
    FfnJob plain = g;
    plain.N = (int32_t)(2 * f.hp);
    plain.B.rows = plain.N;
    plain.finish = EPI_GATE;
    FfnJob *fused[] = {&g}, *split[] = {&plain};
    const bool no[] = {false}, yes[] = {true};
    double time, plain_time;
    p.gate_kind = plan_launch(fused, no, 1, f.form, true, false, &time);
    const int kind = plan_launch(split, yes, 1, f.form, false, false, &plain_time);
    if (plain.splits > 1 && plain_time < time) {
      g = plain;
      p.gate_kind = kind;
      g.partial = (float*)f.take(partial_bytes(g));
    }
  }
  FfnJob& o = p.out;
  Opnd h{};
  h.p = keep;
  h.ld = f.hp;
  h.plane = f.n * f.hp;
  o.A = view(h, f.n, f.hp);
  o.B = view(oo, f.w, f.hp);
  o.M = (int32_t)f.n;
  o.N = (int32_t)f.wp;
  set_out(o, y, f.n, f.w, f.d.scale_out);
  o.finish = EPI_OUT;
  {
    FfnJob* jobs[] = {&o};
    const bool yes[] = {true};
    double time;
    p.out_kind = plan_launch(jobs, yes, 1, f.form, false, false, &time);
  }
  o.partial = (float*)f.take(partial_bytes(o));
  return p;
}

struct FfnBwd {
  FfnJob dh{}, dx{}, dwi{}, dwo{};  // (absent where M = 0)
  int first_kind = 0, second_kind = 0;  // dwo and dh run together, and dwi and dx: the long ones first
};
static FfnBwd plan_bwd(Ffn& f, const void* grad, const void* x, const void* w_in, const void* w_out, const void* saved,
                       int need, void* gx, void* gwi, void* gwo) {
  FfnBwd p;
  const bool nx = need & 1, ni = need & 2, no = need & 4;
  const Opnd og = f.x(grad);
  Opnd h{};
  h.p = (const char*)saved;
  h.ld = f.hp;
  h.plane = f.n * f.hp;
  Opnd dpre{};
  if (nx || ni) {
    const Opnd oo = f.w_out(w_out);
    dpre.ld = 2 * f.hp;
    dpre.plane = f.n * 2 * f.hp;
    char* const dpre_at = f.take(f.esize * dpre.plane);
    dpre.p = dpre_at;
    FfnJob& g = p.dh;
    g.A = view(og, f.n, f.wp);
    g.B = view(oo, f.hp, f.w);
    g.M = (int32_t)f.n;
    g.N = (int32_t)f.hp;
    g.n_out = (int32_t)f.hid;
    g.scale = f.d.scale_out;
    g.saved = saved ? (char*)saved + f.h_bytes() : nullptr;
    g.dpre = dpre_at;
    g.dpre_plane = dpre.plane;
  }
  if (nx) {
    const Opnd oi = f.w_in(w_in);
    FfnJob& g = p.dx;
    g.A = view(dpre, f.n, 2 * f.hp);
    g.B = view(oi, f.wp, 2 * f.hp);
    g.M = (int32_t)f.n;
    g.N = (int32_t)f.wp;
    set_out(g, gx, f.n, f.w, f.d.scale_in);
  }
  if (ni) {
    const Opnd ox = f.x(x);
    FfnJob& g = p.dwi;
    g.A = view(dpre, 2 * f.hp, f.n);
    g.B = view(ox, f.wp, f.n);
    g.M = (int32_t)(2 * f.hp);
    g.N = (int32_t)f.wp;
    set_out(g, gwi, 2 * f.hid, f.w, f.d.scale_in);
    g.gap_at = (int32_t)f.hid;
    g.gap = (int32_t)(f.hp - f.hid);
  }
  if (no) {
    FfnJob& g = p.dwo;
    g.A = view(og, f.wp, f.n);
    g.B = view(h, f.hp, f.n);
    g.M = (int32_t)f.wp;
    g.N = (int32_t)f.hp;
    set_out(g, gwo, f.w, f.hid, f.d.scale_out);
    g.a_tr = g.b_tr = 1;
  }
  p.dx.b_tr = p.dwi.a_tr = p.dwi.b_tr = 1;
  p.dwo.finish = p.dwi.finish = p.dx.finish = EPI_OUT;
  p.dh.b_tr = 1;
  double time, plain_time;
  const bool split_dwo[] = {true, false}, split_both[] = {true, true};
  {
    // (as for the gate: the hidden gradient with a split K loop, where that is faster)
    FfnJob dwo = p.dwo, dh = p.dh;
    dh.finish = EPI_DH;
    FfnJob *fused[] = {&p.dwo, &p.dh}, *split[] = {&dwo, &dh};
    p.first_kind = plan_launch(fused, split_dwo, 2, f.form, false, false, &time);
    const int kind = plan_launch(split, split_both, 2, f.form, false, false, &plain_time);
    if (dh.splits > 1 && plain_time + 3.5 < time) {
      p.dwo = dwo;
      p.dh = dh;
      p.first_kind = kind;
    }
  }
  FfnJob* two[] = {&p.dwi, &p.dx};
  p.second_kind = plan_launch(two, split_both, 2, f.form, false, false, &time);
  for (FfnJob* g : {&p.dwo, &p.dh, &p.dwi, &p.dx}) g->partial = (float*)f.take(g->M > 0 ? partial_bytes(*g) : 0);
  return p;
}

// f(type of the operands in memory, is the operator's type float32)
template <class F>
static int with_operand(int32_t dtype, Form form, F&& f) {
  if (form == FORM_NATIVE) return f(float{}, std::true_type{});
  if (form == FORM_PLANES) return f(bf16_t{}, std::true_type{});
  if (dtype == FC_BF16) return f(bf16_t{}, std::false_type{});
  return f(f16_t{}, std::false_type{});
}

}  // namespace fc

using namespace fc;

extern "C" int64_t fc_ffn_saved(const fc_ffn_desc* d, int64_t n) {
  const int st = ffn_check(d, n);
  if (st != FC_OK) return -st;
  Ffn f(*d, n, nullptr);
  return d->dtype == FC_F32 ? 14 * n * f.hp : f.h_bytes() + f.factor_bytes();
}

extern "C" int64_t fc_ffn_fwd_workspace(const fc_ffn_desc* d, int64_t n, int32_t save) {
  const int st = ffn_check(d, n);
  if (st != FC_OK) return -st;
  Ffn f(*d, n, nullptr);
  plan_fwd(f, nullptr, nullptr, nullptr, save ? (void*)16 : nullptr, nullptr);
  return f.at;
}

extern "C" int fc_ffn_fwd(const fc_ffn_desc* d, int64_t n, const void* x, const void* w_in, const void* w_out, void* y,
                          void* saved, void* ws, int64_t ws_bytes, void* stream) {
  int st = ffn_check(d, n);
  if (st != FC_OK) return st;
  if (n == 0) return FC_OK;
  if (!x || !w_in || !w_out || !y) return FC_ERR_NULL;
  if (d->aligned && !(aligned16(x) && aligned16(w_in) && aligned16(w_out))) return FC_ERR_BAD_DESC;
  Ffn f(*d, n, ws);
  FfnFwd p = plan_fwd(f, x, w_in, w_out, saved, y);
  if (f.at > 0 && (!ws || ws_bytes < f.at)) return FC_ERR_WORKSPACE;
  if (!aligned16(saved) || !aligned16(ws)) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  st = f.run_prep(s);
  if (st != FC_OK) return st;
  return with_operand(d->dtype, f.form, [&](auto m, auto is32) -> int {
    using MT = decltype(m);
    constexpr bool F32 = decltype(is32)::value;
    const FfnJob none{}, *gates[] = {&p.gate}, *sums[] = {&p.out};
    int r = p.gate.splits > 1 ? launch<MT, F32, false, false, EPI_OUT>(p.gate, none, p.gate_kind, s)
                              : launch<MT, F32, false, false, EPI_GATE>(p.gate, none, p.gate_kind, s);
    if (r == FC_OK) r = launch_sums<MT, F32>(gates, 1, s);
    if (r == FC_OK) r = launch<MT, F32, false, false, EPI_OUT>(p.out, none, p.out_kind, s);
    return r != FC_OK ? r : launch_sums<MT, F32>(sums, 1, s);
  });
}

extern "C" int64_t fc_ffn_bwd_workspace(const fc_ffn_desc* d, int64_t n, int32_t need_x, int32_t need_w_in,
                                        int32_t need_w_out) {
  const int st = ffn_check(d, n);
  if (st != FC_OK) return -st;
  Ffn f(*d, n, nullptr);
  plan_bwd(f, nullptr, nullptr, nullptr, nullptr, nullptr, (need_x != 0) | 2 * (need_w_in != 0) | 4 * (need_w_out != 0),
           nullptr, nullptr, nullptr);
  return f.at;
}

extern "C" int fc_ffn_bwd(const fc_ffn_desc* d, int64_t n, const void* grad, const void* x, const void* w_in,
                          const void* w_out, const void* saved, void* gx, void* gwi, void* gwo, void* ws,
                          int64_t ws_bytes, void* stream) {
  int st = ffn_check(d, n);
  if (st != FC_OK) return st;
  const int need = (gx != nullptr) | 2 * (gwi != nullptr) | 4 * (gwo != nullptr);
  if (n == 0 || need == 0) return n == 0 && (gwi || gwo) ? FC_ERR_SHAPE : FC_OK;
  if (!grad || !saved || (gx && !w_in) || (gwi && !x) || ((gx || gwi) && !w_out)) return FC_ERR_NULL;
  if (d->aligned && !(aligned16(grad) && aligned16(x) && aligned16(w_in) && aligned16(w_out))) return FC_ERR_BAD_DESC;
  Ffn f(*d, n, ws);
  FfnBwd p = plan_bwd(f, grad, x, w_in, w_out, saved, need, gx, gwi, gwo);
  if (f.at > 0 && (!ws || ws_bytes < f.at)) return FC_ERR_WORKSPACE;
  if (!aligned16(saved) || !aligned16(ws)) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  st = f.run_prep(s);
  if (st != FC_OK) return st;
  return with_operand(d->dtype, f.form, [&](auto m, auto is32) -> int {
    using MT = decltype(m);
    constexpr bool F32 = decltype(is32)::value;
    const FfnJob *hidden[] = {&p.dh}, *sums[] = {&p.dwo, &p.dwi, &p.dx};
    int r = p.dh.splits > 1 ? launch<MT, F32, true, true, EPI_OUT, false, true, EPI_OUT>(p.dwo, p.dh, p.first_kind, s)
                            : launch<MT, F32, true, true, EPI_OUT, false, true, EPI_DH>(p.dwo, p.dh, p.first_kind, s);
    if (r == FC_OK) r = launch_sums<MT, F32>(hidden, 1, s);
    if (r == FC_OK) r = launch<MT, F32, true, true, EPI_OUT, false, true, EPI_OUT>(p.dwi, p.dx, p.second_kind, s);
    if (r == FC_OK) r = launch_sums<MT, F32>(sums, 3, s);
    return r;
  });
}
