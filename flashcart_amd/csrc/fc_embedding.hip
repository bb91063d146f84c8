// Embedding lookup out[i] = scale table[ids[i]] and the table's gradient g[r] = scale sum_{i: ids[i] = r} grad[i].
//
// The gradient is formed without atomics on values, so that it is the same in every run: token numbers are sorted by
// index (a stable radix sort, 8 bits a pass), the sorted list is cut into pieces of equal length, and each piece adds
// the gradient rows of its runs of equal indices in float32, in token order. Runs inside one piece are written at once;
// runs that cross pieces leave one partial sum per piece, which a second kernel joins in piece order. Rows without
// tokens are zero: the table is filled while the sort counts, since most rows of a large table have no token.
// Small tables need no sort: each wave keeps the sums of all rows in LDS, and a second kernel adds the waves' tables.
// With the lookup: 16,384 tokens of 32,000 rows of 1,024 in bf16 66-70 us, 1,083,777 of 4 rows of 16 in float32 36-37 us.
// Indices outside the table (a device-side check cannot raise) give rows of NaN and take no part in the gradient.
#include <math.h>

#include <algorithm>

#include "fc_node.h"

namespace fc {

// Keys of a workgroup in the sort: 256 times the rounds, few where there are few keys.
inline int emb_rounds(int64_t n) { return n <= 65536 ? 4 : 8; }

// The first column of a chunk of V: the last chunk of a row overlaps the one before it, so that chunks are whole wherever a
// row has V columns (the columns in both get the same value from both).
template <int V>
__device__ __forceinline__ int64_t chunk_start(int64_t c, int64_t width) {
  return width >= V && c > width - V ? width - V : c;
}

// ---- forward: one 16-byte chunk of a row per thread ----
template <class T>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(uint32_t total, uint32_t chunks, int64_t rows, int64_t width,
                                                            const int64_t* __restrict__ ids,
                                                            const T* __restrict__ table, float scale,
                                                            T* __restrict__ out) {
  constexpr int V = 16 / sizeof(T);
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  if (t >= total) return;
  const uint32_t row = t / chunks, chunk = t - row * chunks;
  const int64_t c0 = chunk_start<V>((int64_t)chunk * V, width);
  const int64_t id = ids[row];
  const bool ok = id >= 0 && id < rows;
  const T* src = table + (ok ? id : 0) * width + c0;
  T* dst = out + (int64_t)row * width + c0;
  if (c0 + V <= width) {
    const Pack<T, V> v = load_pack<T, V>(src);
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = from_f32<T>(ok ? to_f32(v.v[i]) * scale : __builtin_nanf(""));
    store_pack<T, V>(dst, o);
    return;
  }
  for (int i = 0; i < width - c0; ++i) dst[i] = from_f32<T>(ok ? to_f32(src[i]) * scale : __builtin_nanf(""));
}

// ---- sort ----
struct EmbSort {
  int64_t n, rows, padding;
  int32_t tiles;
  const int64_t* ids;  // first pass
  const uint32_t* keys;
  const int32_t* order;  // later passes
  uint32_t* keys_out;
  int32_t* order_out;
  int32_t* hist;    // (256, tiles): counts, then the keys of the digit in earlier tiles
  int32_t* total;   // (256)
  int32_t shift, passes;
  bool scanned;     // hist holds sums and total is there
  // table to be filled with zeros by the workgroups behind the tiles
  uint8_t* fill;
  int64_t fill_bytes;
  int32_t* counter;  // of the joins, cleared here
};

// Tokens that add to no row (index outside the table, or the padding row) get the key `rows`: they sort last.
__device__ __forceinline__ uint32_t emb_key(const EmbSort& a, int64_t i) {
  if (!a.ids) return a.keys[i];
  const int64_t id = a.ids[i];
  return (id < 0 || id >= a.rows || id == a.padding) ? (uint32_t)a.rows : (uint32_t)id;
}

constexpr int kEmbFillBytes = 64 << 10;  // of a filling workgroup

__device__ void emb_fill(uint8_t* p, int64_t bytes) {
  const int head = (int)min((int64_t)((16 - ((uintptr_t)p & 15)) & 15), bytes);
  if ((int)threadIdx.x < head) p[threadIdx.x] = 0;
  p += head;
  bytes -= head;
  for (int64_t o = threadIdx.x * 16; o + 16 <= bytes; o += blockDim.x * 16) *(uint4*)(p + o) = make_uint4(0, 0, 0, 0);
  const int64_t done = bytes & ~(int64_t)15;
  if (done + threadIdx.x < bytes) p[done + threadIdx.x] = 0;
}

template <int ROUNDS>
__global__ void __launch_bounds__(256) emb_hist_kernel(EmbSort a) {
  __shared__ int32_t cnt[256];
  const int t = threadIdx.x;
  if ((int)blockIdx.x >= a.tiles) {
    const int64_t b0 = (int64_t)(blockIdx.x - a.tiles) * kEmbFillBytes;
    emb_fill(a.fill + b0, min((int64_t)kEmbFillBytes, a.fill_bytes - b0));
    return;
  }
  if (blockIdx.x == 0 && t == 0 && a.counter) *a.counter = 0;
  cnt[t] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * 256 * ROUNDS;
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = i0 + k * 256 + t;
    if (i < a.n) atomicAdd(&cnt[(emb_key(a, i) >> a.shift) & 255], 1);
  }
  __syncthreads();
  a.hist[(int64_t)t * a.tiles + blockIdx.x] = cnt[t];
}

// Exclusive sum over a workgroup of NW waves; every thread gets the total too.
template <int NW>
__device__ __forceinline__ int block_scan(int v, int* wave_sums, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(s, o, 64);
    if (lane >= o) s += u;
  }
  if (lane == 63) wave_sums[w] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < NW; ++k) {
    const int x = wave_sums[k];
    if (k < w) before += x;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + s - v;
}

// One workgroup per digit: its counts become the number of its keys in earlier tiles.
__global__ void __launch_bounds__(256) emb_scan_kernel(EmbSort a) {
  __shared__ int ws[4];
  int32_t* h = a.hist + (int64_t)blockIdx.x * a.tiles;
  int base = 0;
  for (int k = 0; k < a.tiles; k += 256) {
    const int i = k + threadIdx.x;
    const int v = i < a.tiles ? h[i] : 0;
    int all;
    const int ex = block_scan<4>(v, ws, &all);
    if (i < a.tiles) h[i] = base + ex;
    base += all;
  }
  if (threadIdx.x == 0) a.total[blockIdx.x] = base;
}

// Lanes of this wave whose 8-bit digit equals this lane's, among the active ones.
__device__ __forceinline__ uint64_t match_digit(uint32_t d, bool active) {
  uint64_t m = __ballot(active);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const bool bit = (d >> b) & 1;
    const uint64_t v = __ballot(bit);
    m &= bit ? v : ~v;
  }
  return m;
}

// Stable placement: each wave ranks consecutive keys, 64 at a time.
template <int ROUNDS>
__global__ void __launch_bounds__(256) emb_scatter_kernel(EmbSort a) {
  __shared__ int32_t cnt[4][256];
  __shared__ int32_t base[256];
  __shared__ int ws[4];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
#pragma unroll
  for (int k = 0; k < 4; ++k) cnt[k][t] = 0;
  int total, before;
  if (a.scanned) {
    total = a.total[t];
    before = a.hist[(int64_t)t * a.tiles + blockIdx.x];
  } else {  // few tiles: their counts are added here
    total = before = 0;
    for (int k = 0; k < a.tiles; ++k) {
      const int c = a.hist[(int64_t)t * a.tiles + k];
      before += k < (int)blockIdx.x ? c : 0;
      total += c;
    }
  }
  int all;
  base[t] = block_scan<4>(total, ws, &all) + before;
  __syncthreads();
  const int64_t i0 = ((int64_t)blockIdx.x * 4 + w) * 64 * ROUNDS;
  uint32_t key[ROUNDS];
  int rank[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = i0 + k * 64 + lane;
    const bool ok = i < a.n;
    key[k] = ok ? emb_key(a, i) : 0;
    const uint32_t d = (key[k] >> a.shift) & 255;
    const uint64_t m = match_digit(d, ok);
    const int before = __popcll(m & ((1ull << lane) - 1));
    rank[k] = ok ? cnt[w][d] + before : 0;
    __builtin_amdgcn_wave_barrier();
    if (ok && before == 0) cnt[w][d] += __popcll(m);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  {
    int b = base[t];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = cnt[k][t];
      cnt[k][t] = b;
      b += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = i0 + k * 64 + lane;
    if (i >= a.n) continue;
    const int to = cnt[w][(key[k] >> a.shift) & 255] + rank[k];
    a.keys_out[to] = key[k];
    a.order_out[to] = a.ids ? (int32_t)i : a.order[i];
  }
}

// Up to 1024 K tokens: all passes in one workgroup, in LDS; the other workgroups fill the table. 4,000 tokens of 300 rows:
// 11 us, where two launches a pass take 20; at 16,384 tokens (K = 16) it would take 37, the launches 30.
template <int K>
__global__ void __launch_bounds__(1024) emb_sort_kernel(EmbSort a) {
  __shared__ uint32_t skey[1024 * K];
  __shared__ uint16_t sidx[1024 * K];
  __shared__ int32_t cnt[16][256];
  __shared__ int ws[16];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  if (blockIdx.x > 0) {
    const int64_t b0 = (int64_t)(blockIdx.x - 1) * kEmbFillBytes;
    emb_fill(a.fill + b0, min((int64_t)kEmbFillBytes, a.fill_bytes - b0));
    return;
  }
  if (t == 0) *a.counter = 0;
  const int n = (int)a.n, p0 = w * 64 * K + lane;
  uint32_t key[K];
  int idx[K], rank[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = p0 + 64 * k;
    key[k] = p < n ? emb_key(a, p) : 0;
    idx[k] = p;
  }
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = 8 * pass;
#pragma unroll
    for (int k = 0; k < 4; ++k) (&cnt[0][0])[t + 1024 * k] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool ok = p0 + 64 * k < n;
      const uint32_t d = (key[k] >> shift) & 255;
      const uint64_t m = match_digit(d, ok);
      const int before = __popcll(m & ((1ull << lane) - 1));
      rank[k] = ok ? cnt[w][d] + before : 0;
      __builtin_amdgcn_wave_barrier();
      if (ok && before == 0) cnt[w][d] += __popcll(m);
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    int total = 0;
    if (t < 256)
      for (int k = 0; k < 16; ++k) {
        const int c = cnt[k][t];
        cnt[k][t] = total;
        total += c;
      }
    int all;
    const int base = block_scan<16>(total, ws, &all);
    if (t < 256)
      for (int k = 0; k < 16; ++k) cnt[k][t] += base;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (p0 + 64 * k >= n) continue;
      const int to = cnt[w][(key[k] >> shift) & 255] + rank[k];
      skey[to] = key[k];
      sidx[to] = (uint16_t)idx[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int p = p0 + 64 * k;
      if (p >= n) continue;
      key[k] = skey[p];
      idx[k] = sidx[p];
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int p = p0 + 64 * k;
    if (p >= n) continue;
    a.keys_out[p] = key[k];
    a.order_out[p] = idx[k];
  }
}

// ---- sums of runs ----
struct EmbSum {
  int64_t n, rows, width;
  int32_t pieces, len, col_threads;  // col_threads: a power of two, <= 256
  const uint32_t* keys;
  const int32_t* order;
  const void* grad;
  void* out;
  float scale;
  float* head;  // (pieces, width): sum of the run that began in an earlier piece
  float* tail;  // (pieces, width): sum of the run that goes on in the next piece
  int32_t* joins;  // pieces whose last run has to be joined
  int32_t* counter;
};

// A chunk of V elements, of which `valid` are there and more are asked for only where rows are narrower than V (WIDE false).
// Without a branch, so that loads of several rows are under way together: a branch around a load ends in a wait for it
// (32,126 rows of 2,082 in f16: pieces 53 us with one, 33 without).
template <class T, int V, bool WIDE>
__device__ __forceinline__ Pack<T, V> load_chunk(const T* p, int valid) {
  if constexpr (WIDE) return load_pack<T, V>(p);
  Pack<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.v[i] = p[min(i, valid - 1)];
  return v;
}
template <class T, int V>
__device__ __forceinline__ void store_f32(T* p, int valid, const float (&x)[V]) {
  if (valid >= V) {
    Pack<T, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v.v[i] = from_f32<T>(x[i]);
    store_pack<T, V>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) p[i] = from_f32<T>(x[i]);
  }
}

// A group of col_threads lanes sums one piece over V columns each; U gradient rows are loaded ahead.
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) emb_piece_kernel(EmbSum a) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int groups = 256 / a.col_threads;
  const int64_t p = (int64_t)blockIdx.x * groups + threadIdx.x / a.col_threads;
  const int64_t first = ((int64_t)blockIdx.y * a.col_threads + threadIdx.x % a.col_threads) * V;
  if (p >= a.pieces || first >= a.width) return;
  const int64_t c0 = chunk_start<V>(first, a.width);
  const int valid = (int)min((int64_t)V, a.width - c0);
  const int64_t t0 = p * a.len, t1 = min(a.n, t0 + a.len);
  const T* grad = (const T*)a.grad + c0;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  uint32_t run = a.keys[t0];
  bool from_left = p > 0 && a.keys[t0 - 1] == run;
  auto flush = [&](bool to_right) {
    if (run < (uint32_t)a.rows) {
      if (from_left || to_right) {
        store_f32<float, V>((from_left ? a.head : a.tail) + p * a.width + c0, valid, acc);
        if (!from_left && first == 0) a.joins[atomicAdd(a.counter, 1)] = (int32_t)p;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] *= a.scale;
        store_f32<T, V>((T*)a.out + (int64_t)run * a.width + c0, valid, acc);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
  };
  // the rows of the next U tokens are loaded before this U's are added, their numbers one step earlier still
  uint32_t key[2][U], next_key[U];
  int32_t next_row[U];
  Pack<T, V> g[2][U];
  auto load_tokens = [&](int64_t t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = min(t + u, t1 - 1);
      next_key[u] = a.keys[at];
      next_row[u] = a.order[at];
    }
  };
  auto load_rows = [&](int buf) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[buf][u] = next_key[u];
      g[buf][u] = load_chunk<T, V, WIDE>(grad + (int64_t)next_row[u] * a.width, valid);
    }
  };
  auto add = [&](int64_t t, int buf) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= t1) break;
      if (key[buf][u] != run) {
        flush(false);
        run = key[buf][u];
        from_left = false;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += to_f32(g[buf][u].v[i]);
    }
  };
  load_tokens(t0);
  load_rows(0);
  load_tokens(t0 + U);
  for (int64_t t = t0; t < t1; t += 2 * U) {
    load_rows(1);
    load_tokens(t + 2 * U);
    add(t, 0);
    if (t + U >= t1) break;
    load_rows(0);
    load_tokens(t + 3 * U);
    add(t + U, 1);
  }
  flush(t1 < a.n && a.keys[t1] == run);
}

// A run of several pieces: tail of the first, heads of the others. Runs of up to four pieces are added by one group of lanes
// each, as many at once as there are for a workgroup; longer ones by the whole workgroup: its groups add consecutive spans
// of pieces, the groups' sums are added in order. (351,854 tokens of 120,666 rows of 29 in f16, runs of three tokens: 10 us,
// by whole workgroups only 59.)
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) emb_join_kernel(EmbSum a) {
  constexpr int V = 16 / sizeof(T), SHORT = 4;
  __shared__ float part[256 * V];
  __shared__ int32_t longer[256];  // first piece of a group's run, or -1
  __shared__ uint32_t run[256];
  const int groups = 256 / a.col_threads, grp = threadIdx.x / a.col_threads, ct = threadIdx.x % a.col_threads;
  const int64_t first_col = ((int64_t)blockIdx.y * a.col_threads + ct) * V, c0 = chunk_start<V>(first_col, a.width);
  const int valid = first_col < a.width ? (int)min((int64_t)V, a.width - c0) : 0;
  const int count = *a.counter, batch = min(groups, (count + (int)gridDim.x - 1) / (int)gridDim.x);
  auto store = [&](uint32_t key, float (&acc)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] *= a.scale;
    store_f32<T, V>((T*)a.out + (int64_t)key * a.width + c0, valid, acc);
  };
  for (int64_t j0 = (int64_t)blockIdx.x * batch; j0 < count; j0 += (int64_t)gridDim.x * batch) {
    const int here = (int)min((int64_t)batch, count - j0);
    if (grp < here) {
      const int64_t p = a.joins[j0 + grp];
      const uint32_t key = a.keys[(p + 1) * a.len];
      int m = 2;
#pragma unroll
      for (int k = 2; k <= SHORT; ++k)
        m += p + k < a.pieces && a.keys[min(p + k, (int64_t)a.pieces - 1) * a.len] == key;
      if (ct == 0) {
        longer[grp] = m > SHORT ? (int32_t)p : -1;
        run[grp] = key;
      }
      if (m <= SHORT && valid > 0) {
        float acc[V];
        const Pack<float, V> x = load_chunk<float, V, WIDE>(a.tail + p * a.width + c0, valid);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = x.v[i];
        for (int k = 1; k < m; ++k) {
          const Pack<float, V> y = load_chunk<float, V, WIDE>(a.head + (p + k) * a.width + c0, valid);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] += y.v[i];
        }
        store(key, acc);
      }
    }
    __syncthreads();
    for (int e = 0; e < here; ++e) {
      const int64_t p = longer[e];
      if (p < 0) continue;
      const uint32_t key = run[e];
      // The run's pieces are those that begin with its key: the last one lies in [last, hi]; 256 candidates a round, the
      // next ones first, then spread over the rest.
      int64_t last = p + SHORT, hi = a.pieces - 1;
      for (int64_t stride = 1; last < hi; stride = (hi - last + 255) / 256) {
        const int64_t q = last + (threadIdx.x + 1) * stride;
        const int c = __syncthreads_count(q <= hi && a.keys[q * a.len] == key);
        last += c * stride;
        if (c < 256) hi = min(hi, last + stride - 1);
      }
      const int64_t m = last - p + 1, span = (m + groups - 1) / groups;
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
      if (valid > 0)
#pragma unroll 2
        for (int64_t q = p + grp * span; q < min(p + (grp + 1) * span, last + 1); ++q) {
          const Pack<float, V> x = load_chunk<float, V, WIDE>((q == p ? a.tail : a.head) + q * a.width + c0, valid);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] += x.v[i];
        }
#pragma unroll
      for (int i = 0; i < V; ++i) part[threadIdx.x * V + i] = acc[i];
      __syncthreads();
      if (grp == 0 && valid > 0) {
        for (int k = 1; k < groups; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] += part[(k * a.col_threads + ct) * V + i];
        store(key, acc);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// ---- few rows: no sort ----
struct EmbFew {
  int64_t n, rows, width, padding, per;  // per: tokens of a workgroup
  int32_t col_threads;                   // a power of two, <= 64
  const int64_t* ids;
  const void* grad;
  void* out;
  float scale;
  float* part;  // (rows, chunks, workgroups, V)
};

// Each group of col_threads lanes of a wave keeps the sums of all rows over V columns a lane in LDS, and one row more for
// tokens that add to none. A lane's 16-byte words lie at its own banks, whatever the row. Gradient rows are read once, in
// order, not gathered; two batches of U tokens are under way. (LDS float adds instead of read, add and write: 126 us for
// 16 at 1,083,777 of 4 rows of 16 in float32.)
template <class T, bool WIDE>
__global__ void __launch_bounds__(64) emb_few_kernel(EmbFew a) {
  constexpr int V = 16 / sizeof(T), Q = V / 4, U = 4;
  extern __shared__ float4 sums[];  // (rows + 1, Q, 64)
  const int lane = threadIdx.x, groups = 64 / a.col_threads, grp = lane / a.col_threads, ct = lane % a.col_threads;
  const int rows = (int)a.rows;
  const int64_t cols = (a.width + V - 1) / V, chunk = (int64_t)blockIdx.x * a.col_threads + ct;
  const int64_t c0 = chunk_start<V>(min(chunk, cols - 1) * V, a.width);
  const int valid = (int)min((int64_t)V, a.width - c0);
  for (int k = 0; k < (rows + 1) * Q; ++k) sums[k * 64 + lane] = make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t t0 = blockIdx.y * a.per, t1 = min(a.n, t0 + a.per), batch = (int64_t)U * groups;
  uint64_t id[2][U];
  Pack<T, V> g[2][U];
  auto load = [&](const int64_t* ids, const T* grad, int buf) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[buf][u] = (uint64_t)ids[u * groups];
      g[buf][u] = load_chunk<T, V, WIDE>(grad + (int64_t)(u * groups) * a.width, valid);
    }
  };
  auto add_row = [&](uint64_t x, const Pack<T, V>& v) {
    const int row = x < (uint64_t)rows && x != (uint64_t)a.padding ? (int)x : rows;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float4& to = sums[(row * Q + q) * 64 + lane];
      float4 y = to;
      y.x += to_f32(v.v[4 * q]);
      y.y += to_f32(v.v[4 * q + 1]);
      y.z += to_f32(v.v[4 * q + 2]);
      y.w += to_f32(v.v[4 * q + 3]);
      to = y;
    }
  };
  auto add = [&](int buf) {
#pragma unroll
    for (int u = 0; u < U; ++u) add_row(id[buf][u], g[buf][u]);
  };
  const int64_t pairs = (t1 - t0) / (2 * batch);
  const int64_t* ids = a.ids + t0 + grp;
  const T* grad = (const T*)a.grad + (t0 + grp) * a.width + c0;
  if (pairs > 0) load(ids, grad, 0);
  for (int64_t k = 1; k <= pairs; ++k) {
    load(ids + batch, grad + batch * a.width, 1);
    add(0);
    const int64_t on = k < pairs ? 2 * batch : 0;  // (the last pair's first batch is loaded again, and not used)
    ids += on;
    grad += on * a.width;
    load(ids, grad, 0);
    add(1);
  }
  for (int64_t t = t0 + pairs * 2 * batch; t < t1; t += groups) {  // a token behind the last adds to no row
    const int64_t from = min(t + grp, t1 - 1);
    const Pack<T, V> v = load_chunk<T, V, WIDE>((const T*)a.grad + from * a.width + c0, valid);
    add_row(t + grp < t1 ? (uint64_t)a.ids[from] : ~0ull, v);
  }
  __syncthreads();
  if (chunk >= cols) return;
  for (int r = grp; r < rows; r += groups)
    for (int q = 0; q < Q; ++q) {
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < groups; ++k) {
        const float4 x = sums[(r * Q + q) * 64 + k * a.col_threads + ct];
        y.x += x.x;
        y.y += x.y;
        y.z += x.z;
        y.w += x.w;
      }
      *(float4*)(a.part + ((r * cols + chunk) * gridDim.y + blockIdx.y) * V + 4 * q) = y;
    }
}

// One wave per chunk of V columns of a row: its partial sums in consecutive spans, the lanes' sums in a fixed order.
template <class T>
__global__ void __launch_bounds__(64) emb_few_join_kernel(EmbFew a, int64_t parts) {
  constexpr int V = 16 / sizeof(T);
  const int64_t cols = (a.width + V - 1) / V, r = blockIdx.x / cols, chunk = blockIdx.x - r * cols;
  const float* part = a.part + blockIdx.x * parts * V;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int64_t k = threadIdx.x; k < parts; k += 64) {
    const Pack<float, V> x = load_pack<float, V>(part + k * V);
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += x.v[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc[i] += __shfl_xor(acc[i], o, 64);
    acc[i] *= a.scale;
  }
  const int64_t c0 = chunk_start<V>(chunk * V, a.width);
  if (threadIdx.x == 0) store_f32<T, V>((T*)a.out + r * a.width + c0, (int)min((int64_t)V, a.width - c0), acc);
}

struct EmbPlan {
  int64_t tiles, pieces, len;
  int col_threads, col_blocks, passes;
  int64_t keys[2], order[2], hist, total, head, tail, joins, counter, bytes;
  // few rows
  bool few;
  int few_threads, few_lds;
  int64_t few_parts, few_per;
};

// Tables of up to 32 KB whose sums fit a wave's 64 KB of LDS. Backward kernels, us, against sorting: 1,083,777 of 4 rows of
// 16 in float32 19 / 64, 25,000 of 63 of 128 19 / 24, 2,000 of 31 of 512 in bf16 19 / 17; of larger tables the partial sums
// weigh more: 16,384 of 31 of 1,024 in bf16 32 / 30, 65,536 of 16 of 1,024 in float32 118 / 105, of 63 of 4,096 312 / 278.
static void emb_plan_few(EmbPlan& p, int64_t n, int64_t rows, int64_t width, int64_t V) {
  const int64_t cols = (width + V - 1) / V;
  if (n == 0 || rows > 64 || (rows + 1) * V * 256 > (64 << 10) || rows * width * (16 / V) > (32 << 10)) return;
  int ct = 1;
  while (ct < 64 && ct < cols) ct *= 2;
  const int64_t groups = 64 / ct, blocks = (cols + ct - 1) / ct, lds = (rows + 1) * V * 256;
  const int64_t waves = 256 * std::min<int64_t>(8, (160 << 10) / lds);
  // steps of a workgroup: a step's chain through LDS against the partial sums' bytes, and the waves that run at once
  const double bytes = 8.0 * (double)n * rows * width / groups / 4.5e6;
  int64_t steps = std::max<int64_t>({8, (int64_t)sqrt(bytes / 0.12), n * blocks / (groups * waves)});
  steps = (steps + 7) / 8 * 8;  // (a grid of few thousand workgroups: what 2,048 waves at once or 8 steps each leave)
  p.few = true;
  p.few_threads = ct;
  p.few_lds = (int)lds;
  p.few_per = steps * groups;
  p.few_parts = (n + p.few_per - 1) / p.few_per;
  p.bytes = 4 * p.few_parts * rows * cols * V;
}

static EmbPlan emb_plan(int32_t dtype, int64_t n, int64_t rows, int64_t width) {
  EmbPlan p{};
  const int64_t V = 16 / node_dtype_size(dtype), cols = (width + V - 1) / V;
  emb_plan_few(p, n, rows, width, V);
  if (p.few) return p;
  const int64_t tile = 256 * emb_rounds(n);
  p.tiles = (n + tile - 1) / tile;
  int ct = 1;
  while (ct < 256 && ct < cols) ct *= 2;
  p.col_threads = ct;
  p.col_blocks = (int)((cols + ct - 1) / ct);
  p.len = 16;
  while (p.len < 1024 && n / p.len * cols > (1 << 18)) p.len *= 2;
  p.pieces = (n + p.len - 1) / p.len;
  int bits = 1;
  while ((rows >> bits) > 0) ++bits;
  p.passes = (bits + 7) / 8;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  for (int k = 0; k < 2; ++k) {
    p.keys[k] = take(4 * n);
    p.order[k] = take(4 * n);
  }
  p.hist = take(1024 * p.tiles);
  p.total = take(1024);
  p.head = take(4 * p.pieces * width);
  p.tail = take(4 * p.pieces * width);
  p.joins = take(4 * p.pieces);
  p.counter = take(4);
  p.bytes = at;
  return p;
}

static int emb_check(int32_t dtype, int64_t n, int64_t rows, int64_t width) {
  if (!node_dtype_ok(dtype)) return FC_ERR_BAD_DESC;
  if (n < 0 || rows < 1 || width < 1 || n > 0x7fff0000 || rows > 0x7fff0000 || width > 0x7fff0000) return FC_ERR_SHAPE;
  return FC_OK;
}

}  // namespace fc

using namespace fc;

extern "C" int fc_embedding_fwd(int32_t dtype, int64_t n, int64_t rows, int64_t width, const int64_t* ids,
                                const void* table, float scale, void* out, void* stream) {
  const int st = emb_check(dtype, n, rows, width);
  if (st != FC_OK) return st;
  if (n == 0) return FC_OK;
  if (!ids || !table || !out) return FC_ERR_NULL;
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    // (chunks < 2^30; a launch of whole tokens, kLaunchBlocks blocks of them where a row is not longer)
    const int64_t chunks = (width + 16 / sizeof(T) - 1) / (16 / sizeof(T));
    const int64_t tokens = std::max<int64_t>(1, kLaunchBlocks * 256 / chunks);
    for (int64_t i = 0; i < n; i += tokens) {
      const int64_t total = std::min(tokens, n - i) * chunks;
      hipLaunchKernelGGL(embedding_fwd_kernel<T>, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                         (uint32_t)total, (uint32_t)chunks, rows, width, ids + i, (const T*)table, scale,
                         (T*)out + i * width);
      FC_LAUNCH_CHECK();
    }
    return FC_OK;
  });
}

extern "C" int64_t fc_embedding_bwd_workspace(int32_t dtype, int64_t n, int64_t rows, int64_t width) {
  const int st = emb_check(dtype, n, rows, width);
  if (st != FC_OK) return -st;
  return emb_plan(dtype, n, rows, width).bytes;
}

extern "C" int fc_embedding_bwd(int32_t dtype, int64_t n, int64_t rows, int64_t width, const int64_t* ids,
                                const void* grad_out, float scale, int64_t padding, void* grad_table, void* ws,
                                int64_t ws_bytes, void* stream) {
  const int st = emb_check(dtype, n, rows, width);
  if (st != FC_OK) return st;
  if (!grad_table || (n > 0 && (!ids || !grad_out))) return FC_ERR_NULL;
  const EmbPlan p = emb_plan(dtype, n, rows, width);
  if (ws_bytes < p.bytes || !ws) return FC_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  char* w = (char*)ws;
  if (p.few) {
    EmbFew f{};
    f.n = n;
    f.rows = rows;
    f.width = width;
    f.padding = padding;
    f.per = p.few_per;
    f.col_threads = p.few_threads;
    f.ids = ids;
    f.grad = grad_out;
    f.out = grad_table;
    f.scale = scale;
    f.part = (float*)w;
    return with_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      const int64_t cols = (width + 16 / sizeof(T) - 1) / (16 / sizeof(T));
      const dim3 grid((unsigned)((cols + p.few_threads - 1) / p.few_threads), (unsigned)p.few_parts);
      if (width >= (int64_t)(16 / sizeof(T))) hipLaunchKernelGGL((emb_few_kernel<T, true>), grid, dim3(64), p.few_lds, s, f);
      else hipLaunchKernelGGL((emb_few_kernel<T, false>), grid, dim3(64), p.few_lds, s, f);
      FC_LAUNCH_CHECK();
      hipLaunchKernelGGL((emb_few_join_kernel<T>), dim3((unsigned)(rows * cols)), dim3(64), 0, s, f, p.few_parts);
      FC_LAUNCH_CHECK();
      return FC_OK;
    });
  }
  EmbSort a{};
  a.n = n;
  a.rows = rows;
  a.padding = padding;
  a.tiles = (int32_t)p.tiles;
  a.hist = (int32_t*)(w + p.hist);
  a.total = (int32_t*)(w + p.total);
  a.counter = (int32_t*)(w + p.counter);
  const int64_t table_bytes = rows * width * node_dtype_size(dtype);
  const int64_t fills = (table_bytes + kEmbFillBytes - 1) / kEmbFillBytes;
  if (!grid_fits(p.tiles + fills + 1, 1024) || p.col_blocks > 65535) return FC_ERR_SHAPE;
  a.fill = (uint8_t*)grad_table;
  a.fill_bytes = table_bytes;
  a.passes = p.passes;
  int last = 0;
  if (n > 0 && n <= 4096) {
    a.ids = ids;
    a.keys_out = (uint32_t*)(w + p.keys[0]);
    a.order_out = (int32_t*)(w + p.order[0]);
    const dim3 grid((unsigned)(1 + fills)), block(1024);
    if (n <= 1024) hipLaunchKernelGGL((emb_sort_kernel<1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((emb_sort_kernel<4>), grid, block, 0, s, a);
    FC_LAUNCH_CHECK();
  } else {
    last = (p.passes - 1) & 1;
    a.scanned = p.tiles > 64;
    const bool few = emb_rounds(n) == 4;
    for (int k = 0; k < p.passes; ++k) {
      a.ids = k == 0 ? ids : nullptr;
      a.keys = (uint32_t*)(w + p.keys[(k + 1) & 1]);
      a.order = (int32_t*)(w + p.order[(k + 1) & 1]);
      a.keys_out = (uint32_t*)(w + p.keys[k & 1]);
      a.order_out = (int32_t*)(w + p.order[k & 1]);
      a.shift = 8 * k;
      const int64_t blocks = p.tiles + (k == 0 ? fills : 0);
      if (few) hipLaunchKernelGGL((emb_hist_kernel<4>), dim3((unsigned)blocks), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((emb_hist_kernel<8>), dim3((unsigned)blocks), dim3(256), 0, s, a);
      FC_LAUNCH_CHECK();
      if (n == 0) return FC_OK;
      if (a.scanned) {
        hipLaunchKernelGGL(emb_scan_kernel, dim3(256), dim3(256), 0, s, a);
        FC_LAUNCH_CHECK();
      }
      if (few) hipLaunchKernelGGL((emb_scatter_kernel<4>), dim3((unsigned)p.tiles), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((emb_scatter_kernel<8>), dim3((unsigned)p.tiles), dim3(256), 0, s, a);
      FC_LAUNCH_CHECK();
    }
  }
  EmbSum b{};
  b.n = n;
  b.rows = rows;
  b.width = width;
  b.pieces = (int32_t)p.pieces;
  b.len = (int32_t)p.len;
  b.col_threads = p.col_threads;
  b.keys = (uint32_t*)(w + p.keys[last]);
  b.order = (int32_t*)(w + p.order[last]);
  b.grad = grad_out;
  b.out = grad_table;
  b.scale = scale;
  b.head = (float*)(w + p.head);
  b.tail = (float*)(w + p.tail);
  b.joins = (int32_t*)(w + p.joins);
  b.counter = (int32_t*)(w + p.counter);
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const int groups = 256 / p.col_threads;
    const bool whole = width >= (int64_t)(16 / sizeof(T));
    const dim3 grid((unsigned)((p.pieces + groups - 1) / groups), p.col_blocks);
    if (whole) hipLaunchKernelGGL((emb_piece_kernel<T, true>), grid, dim3(256), 0, s, b);
    else hipLaunchKernelGGL((emb_piece_kernel<T, false>), grid, dim3(256), 0, s, b);
    FC_LAUNCH_CHECK();
    // narrow groups: more of them share the pieces of a run
    EmbSum j = b;
    j.col_threads = b.col_threads < 16 ? b.col_threads : 16;
    const int64_t cols = (width + 16 / sizeof(T) - 1) / (16 / sizeof(T)), wide = (cols + j.col_threads - 1) / j.col_threads;
    if (wide > 65535) return FC_ERR_SHAPE;
    const dim3 joins((unsigned)(p.pieces < 4096 ? p.pieces : 4096), (unsigned)wide);
    if (whole) hipLaunchKernelGGL((emb_join_kernel<T, true>), joins, dim3(256), 0, s, j);
    else hipLaunchKernelGGL((emb_join_kernel<T, false>), joins, dim3(256), 0, s, j);
    FC_LAUNCH_CHECK();
    return FC_OK;
  });
}
