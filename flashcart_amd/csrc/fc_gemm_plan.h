// Host side of the matrix products of fc_ffn_gemm.h: tile sizes and splits by their cost, operands, workspaces.
#pragma once

#include "fc_ffn_gemm.h"

namespace fc {

// (native float32 has no 256 x 256 tile: planes take over before it would fill the device)
using TileL = Tile<256, 256, 2, 4, 2>;
using TileH = Tile<256, 128, 2, 4, 2>;  // half a TileL, in its LDS (of the dense layers alone)
using TileM = Tile<128, 128, 2, 2, 2>;
using TileS = Tile<64, 64, 2, 2, 4>;
using TileR = Tile<32, 64, 2, 2, 4>;  // (of groups of few rows alone)
using TileX = Tile<64, 64, 2, 2, 2>;  // (of the dense layers alone)

inline int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

inline Opnd view(Opnd o, int64_t rows, int64_t k) {
  o.rows = (int32_t)rows;
  o.k = (int32_t)k;
  return o;
}

inline void set_out(GemmJob& g, void* out, int64_t m_out, int64_t n_out, float scale) {
  g.out = out;
  g.ld_out = n_out;
  g.m_out = (int32_t)m_out;
  g.n_out = (int32_t)n_out;
  g.gap_at = INT32_MAX;
  g.scale = scale;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

inline int64_t blocks_of(const GemmJob& g) { return (int64_t)g.tiles_m * g.tiles_n * g.splits; }

inline int tile_rows(int kind) { return kind == 2 ? 256 : kind == 1 ? 128 : kind == 4 ? 32 : 64; }

inline void set_tiles(GemmJob& g, int kind, bool gate) {
  const int bm = tile_rows(kind), bn = gate ? bm / 2 : bm;
  g.tiles_m = cdiv(g.M, bm);
  g.tiles_n = cdiv(g.N, bn);
}

// What a workgroup of each tile size takes, in us: a step of 64 k when it has its CU's loads to itself, the CU's time a
// step takes when the device is full, and filling the pipeline and writing the tile. Measured in bf16: chains of steps on
// few CUs (n = 30,000, width = hidden = 64), full devices at 1,024 to 30,000 rows. (Of 14 sizes tried with each tile
// throughout, the choice was within 3% of the best in 13; 128 x 128 tiles alone cost up to 20%, 64 x 64 up to 2 times.) The 64 x 64 tile is bound by what the L2
// caches deliver, the 256 x 256 tile by the matrix cores.
struct TileCost {
  double step, full, end, fused;  // fused: the end with an epilogue of the block's elementwise steps
};
// The last is the 64 x 64 tile with two LDS stages: up to five workgroups share a CU, whose loads run one step ahead. It is
// faster where workgroups are many and their sums short (25,000 x 128 x 128 float32, forward 21.5 -> 20.1 us, dx and dW 27.0
// -> 24.2; 8,192 x 512 x 512 bf16 forward 17.0 -> 14.6), slower where they are few and long (1 x 4,096 x 10,240 15 -> 31).
constexpr int kKinds = 4;
constexpr TileCost kTileCost[kKinds] = {{0.2, 0.26, 0.8, 1.2}, {0.65, 0.55, 2.5, 3.2}, {1.25, 1.5, 9.0, 14.0},
                                        {0.47, 0.25, 0.9, 1.3}};
// native float32, 32 k a step: bound by the matrix cores
constexpr TileCost kNativeCost[kKinds] = {{0.5, 0.56, 1.0, 2.2}, {2.05, 1.85, 5.0, 6.0}, {}, {0.6, 0.48, 0.6, 1.6}};
constexpr int kShare[kKinds] = {2, 2, 1, 5};  // workgroups that a CU runs at once
// What the first load and the epilogue (plain, of a dense layer) take when nothing hides them: rounds of workgroups with short
// sums are bound by that (8,192 x 64 x 512 bf16 forward, tiles of 64, 128 and 64 with two stages: 14.5, 13.7, 10.5 us).
constexpr double kLatency[kKinds][2] = {{2.0, 4.5}, {4.0, 9.0}, {10.0, 18.0}, {2.0, 4.5}};

enum Form { FORM_16, FORM_NATIVE, FORM_PLANES, FORM_8 };

// Steps of a sum over k, in the operands' form.
inline int steps_of(int k, Form form) {
  const int per = form == FORM_NATIVE ? 32 : form == FORM_8 ? 128 : 64;
  return (form == FORM_PLANES ? 6 : 1) * cdiv(k, per);
}

// The answers to the last questions, by sizes alone: a layer asks the same ones call after call, twice in each (for the
// workspace's size, and for the launch), and an answer takes 1 to 3 us of the host's time.
struct PlanKey {
  int32_t v[12];
};
struct PlanChoice {
  int kind;
  int64_t split[2];
  double time;
};
template <class F>
PlanChoice remembered(const PlanKey& key, F&& choose) {
  constexpr int SLOTS = 64;
  struct Slot {
    PlanKey key;
    PlanChoice choice;
    bool used;
  };
  static thread_local Slot slots[SLOTS];
  uint32_t h = 2166136261u;
  for (int32_t v : key.v) h = (h ^ (uint32_t)v) * 16777619u;
  Slot& s = slots[(h ^ h >> 15) % SLOTS];
  if (!s.used || memcmp(&s.key, &key, sizeof(key)) != 0) s = Slot{key, choose(), true};
  return s.choice;
}

// Tile size and splits of the K loops (plain outputs only) of one launch: those of the least time by the costs above, a
// split K loop paying for its partial sums, written and read at 3 TB/s, and for the launch that adds them. `short_tiles`: the
// 64 x 64 tile with two stages is one of the choices.
template <class Job>
int plan_launch(Job* const* jobs, const bool* can_split, int count, Form form, bool gate, bool short_tiles, double* time_us) {
  const int cus = device_cu_count();
  for (int q = 0; q < count; ++q) {
    const int k = jobs[q]->A.k > jobs[q]->B.k ? jobs[q]->A.k : jobs[q]->B.k;
    jobs[q]->steps = steps_of(k, form);
  }
  PlanKey key{{cus, count, (int)form, gate, short_tiles}};
  for (int q = 0; q < count; ++q) {
    key.v[5 + 3 * q] = jobs[q]->M;
    key.v[6 + 3 * q] = jobs[q]->N;
    key.v[7 + 3 * q] = 2 * jobs[q]->steps + can_split[q];
  }
  const PlanChoice choice = remembered(key, [&]() {
    int best_kind = 0, best_splits[2] = {1, 1};
    double best = 1e30;
    for (int kind = 0; kind < (short_tiles ? 4 : 3); ++kind) {
      if (form == FORM_NATIVE && kind == 2) continue;
      const TileCost& c = form == FORM_NATIVE ? kNativeCost[kind] : kTileCost[kind];
      double chain = 0;  // the longest sum that may be split
      for (int q = 0; q < count; ++q)
        if (jobs[q]->M > 0 && can_split[q] && jobs[q]->steps * c.step > chain) chain = jobs[q]->steps * c.step;
      double most = chain + 1;  // of a workgroup's steps
      do {
        double load = 0, sums = 0, steps[2] = {0, 0}, ends[2] = {0, 0};
        int64_t blocks = 0;
        int splits[2] = {1, 1};
        for (int q = 0; q < count; ++q) {
          GemmJob& g = *jobs[q];
          if (g.M == 0) continue;
          set_tiles(g, kind, gate);
          double end = (can_split[q] ? c.end : c.fused) * (form == FORM_PLANES ? 1.5 : 1);
          if (can_split[q] && g.steps * c.step > most) {
            splits[q] = (int)(g.steps * c.step / most) + 1;
            if (splits[q] > g.steps / 4) splits[q] = g.steps / 4 > 1 ? g.steps / 4 : 1;
          }
          if (splits[q] > 1) {
            end *= 1.5;
            sums += 8e-6 / 3 * splits[q] * g.M * g.N;
          }
          const int64_t n = (int64_t)g.tiles_m * g.tiles_n * splits[q];
          steps[q] = (double)g.steps / splits[q];
          ends[q] = end;
          blocks += n;
          load += n * (steps[q] * c.full + end) / cus;
        }
        // the longest workgroup, which shares its CU with another one where the device is full (not the largest tile)
        const double shared = kShare[kind] * c.full, pace = blocks > cus && shared > c.step ? shared : c.step;
        double longest = 0;
        for (int q = 0; q < count; ++q)
          if (steps[q] * pace + ends[q] > longest) longest = steps[q] * pace + ends[q];
        // whole rounds of workgroups where they are few and the matrix cores bound them, something between otherwise
        const double rounds = blocks > 0 ? (double)((blocks + cus - 1) / cus) * cus / blocks : 1;
        if (blocks > cus) load *= form == FORM_NATIVE && blocks <= 2 * cus ? rounds : 0.5 + 0.5 * rounds;
        double time = load > longest ? load : longest;
        if (short_tiles && blocks > 0) {
          double alone = 0;
          for (int q = 0; q < count; ++q)
            if (jobs[q]->M > 0)
              alone += (double)jobs[q]->tiles_m * jobs[q]->tiles_n * splits[q] *
                       (steps[q] * c.step + kLatency[kind][!can_split[q]]);
          alone *= (double)((blocks + cus * kShare[kind] - 1) / (cus * kShare[kind])) / blocks;
          if (alone > time) time = alone;
        }
        if (sums > 0) time += sums + 3.5;
        if (time < best) {
          best = time;
          best_kind = kind;
          for (int q = 0; q < count; ++q) best_splits[q] = splits[q];
        }
        most /= 2;
      } while (most > 2);
    }
    return PlanChoice{best_kind, {best_splits[0], best_splits[1]}, best};
  });
  for (int q = 0; q < count; ++q) {
    set_tiles(*jobs[q], choice.kind, gate);
    jobs[q]->splits = (int)choice.split[q];
  }
  *time_us = choice.time;
  return choice.kind;
}
inline int64_t partial_bytes(const GemmJob& g) { return g.splits > 1 ? 4ll * g.splits * g.M * g.N : 0; }

}  // namespace fc
