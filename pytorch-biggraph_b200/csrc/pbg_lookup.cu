// Rows of a table by id (scaled), and the gradient of that: the rows' gradients summed by id.
//
//   lookup  out[i] = s W[id_i]                         n rows read, n written: HBM
//   grad    dW[v]  = s sum_{i : id_i = v} g_i          n rows read, num_rows written: HBM, and the sort's latency
//
// The gradient sorts (id, i) first, so that the occurrences of an id lie next to each other in the order of i, and no sum
// depends on the order in which anything arrives.  Sums are fp32, rounded to the output's type once.
//
// Measured, calls on other buffers each time: 16,384 rows of 1024 fp32 19 us (134 MB, part of it from L2); gradients of 16,384 x 2048 bf16 into
// 131,072 rows 140 us (604 MB; sort 15, sums and zeros 105 at 64 % of DRAM's peak, join 14), of 10,000 x 400 fp32 into 14,951 rows 29 us,
// three launches of a few dependent steps each.  Five rows: 2 us in a graph.
#include <cooperative_groups.h>

#include "pbg_tokens.cuh"

namespace cg = cooperative_groups;

// N elements of T as one access of N * sizeof(T) bytes
template <class T, int N> struct __align__(sizeof(T) * N) Unit { T e[N]; };

// A group of G threads moves a row, U units per thread in flight.  Bound by HBM where rows are many, else by two loads in a row.
template <class T, int N, int U>
__global__ void __launch_bounds__(256)
lookup_kernel(const T *__restrict__ table, long long row_stride, long long num_rows, int dim, int G, const long long *__restrict__ ids, long long n,
              float scale, T *__restrict__ out, int *errors) {
  const int sub = threadIdx.x % G, units = dim / N;
  const long long r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (r >= n) return;
  const long long id = ids[r];
  const bool bad = id < 0 || id >= num_rows;
  if (bad && sub == 0 && errors) atomicOr(errors, TOK_ERR_ID);
  const Unit<T, N> *src = reinterpret_cast<const Unit<T, N> *>(table + (bad ? 0 : id) * row_stride);
  Unit<T, N> *dst = reinterpret_cast<Unit<T, N> *>(out + r * dim);
  for (int u0 = sub; u0 < units; u0 += U * G) {
    Unit<T, N> v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) if (u0 + k * G < units) v[k] = src[u0 + k * G];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (u0 + k * G >= units) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) v[k].e[i] = bad ? Tok<T>::down(__int_as_float(0x7fc00000)) : Tok<T>::down(Tok<T>::up(v[k].e[i]) * scale);
      dst[u0 + k * G] = v[k];
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------------
// The sorted list is cut into tiles of LG_TILE occurrences; a warp sums those of one tile over 32 units of columns.  Most ids occur once
// or twice.  A run of one id that reaches into the next tiles is summed by the warp of the tile it begins in, unless it goes on for
// LG_LONG or more: then every tile leaves its part as fp32 sums -- that of its first run in slot 0, that of its last in slot 1 -- and
// the join adds a run's parts in the order of the tiles.
#define LG_TILE 8
#define LG_LONG 32
#define LG_JOIN_WARPS 8
#define LG_JOIN_TILES 32

struct GradArgs {
  const unsigned long long *keys;      // sorted ids, those outside of the table behind all others
  const unsigned int *vals;
  float *part;                         // [tiles][2][dim rounded up to 4]
  const unsigned int *named;           // a bit per row: some id names it
  long long grad_stride, out_stride, num_rows;
  int n, dim, part_ld, accumulate;
  int sum_ctas, zero_words;            // CTAs that sum; words of `named` to each of those that write zeros
  FastDiv by_units;
  float scale;
};
template <class T, int N>
__device__ __forceinline__ void grad_store(T *out, const GradArgs &a, unsigned long long row, int unit, const float (&acc)[N]) {
  Unit<T, N> *dst = reinterpret_cast<Unit<T, N> *>(out + (long long)row * a.out_stride) + unit;
  Unit<T, N> v;
  if (a.accumulate) {
    v = *dst;
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = Tok<T>::down(Tok<T>::up(v.e[i]) + acc[i] * a.scale);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v.e[i] = Tok<T>::down(acc[i] * a.scale);
  }
  *dst = v;
}

// how many of 64 flags, 32 to a word, are set from bit `from` of the first on
__device__ __forceinline__ int run_of(unsigned w0, unsigned w1, int from) {
  const unsigned gap0 = ~(w0 >> from) & (0xffffffffu >> from);
  return gap0 ? __ffs(gap0) - 1 : ~w1 ? 32 - from + __ffs(~w1) - 1 : 64 - from;
}

// Zeros into the zero_words x 32 rows from r0 on that no id names.
template <class T, int N>
__device__ __forceinline__ void lookup_zeros(T *out, const GradArgs &a, long long r0, const unsigned *named) {
  Unit<T, N> z;
#pragma unroll
  for (int i = 0; i < N; ++i) z.e[i] = Tok<T>::down(0.f);
  const int units = a.dim / N;
  const long long rows = a.num_rows - r0 < a.zero_words * 32 ? a.num_rows - r0 : a.zero_words * 32;
  const int total = (int)(rows * units);
  for (int i = threadIdx.x; i < total; i += 256) {
    const int r = a.by_units.div(i);
    if (named[r >> 5] >> (r & 31) & 1u) continue;
    reinterpret_cast<Unit<T, N> *>(out + (r0 + r) * a.out_stride)[i - r * units] = z;
  }
}

// The first sum_ctas CTAs sum, the others write the zeros: sums wait for one thing after the other, and the zeros fill the time.  (Zeros
// beside the sort and sums over them: 166 us for the 16,384 x 2048 bf16 above.)
template <class T, int N>
__global__ void __launch_bounds__(256, 3) lookup_grad_kernel(const T *__restrict__ grad, T *__restrict__ out, GradArgs a) {
  pdl_begin();
  if (blockIdx.x >= (unsigned)a.sum_ctas) {
    const long long word = ((long long)blockIdx.x - a.sum_ctas) * a.zero_words;
    lookup_zeros<T, N>(out, a, word * 32, a.named + word);
    return;
  }
  const int lane = threadIdx.x & 31, units = a.dim / N, blocks = (units + 31) / 32;
  const long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int tile = (int)(job / blocks), unit = (int)(job - (long long)tile * blocks) * 32 + lane;
  const int i0 = tile * LG_TILE;
  if (i0 >= a.n) return;
  const int count = a.n - i0 < LG_TILE ? a.n - i0 : LG_TILE;
  const unsigned rows = (unsigned)a.num_rows, all = 0xffffffffu;
  // 64 ids from the tile's first on and 64 in front of it, all asked for at once: LG_LONG + LG_TILE of them say what is to be known
  static_assert(LG_LONG + LG_TILE <= 64, "the ids around a tile");
  unsigned f[2], b[2], val[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int at = i0 + 32 * w + lane, back = i0 - 1 - 32 * w - lane;
    f[w] = at < a.n ? (unsigned)a.keys[at] : all;
    val[w] = at < a.n ? a.vals[at] : 0u;
    b[w] = back >= 0 ? (unsigned)a.keys[back] : all;
  }
  const unsigned first = __shfl_sync(all, f[0], 0), last = __shfl_sync(all, f[0], count - 1);
  // the first run, where it began before this tile: part of a long one, or another warp's
  const int to = run_of(__ballot_sync(all, f[0] == first), __ballot_sync(all, f[1] == first), 0);
  const int from = run_of(__ballot_sync(all, b[0] == first), __ballot_sync(all, b[1] == first), 0);
  const bool lead = from > 0 && first < rows;
  const int owner_end = ((i0 - from) / LG_TILE + 1) * LG_TILE;            // of the tile it began in
  const bool lead_long = lead && (from == 64 || i0 + to - owner_end >= LG_LONG);
  // the last run, where it goes on behind this tile
  const int behind = run_of(__ballot_sync(all, f[0] == last), __ballot_sync(all, f[1] == last), count);
  const bool trail = behind > 0 && last < rows, trail_long = trail && behind >= LG_LONG;
  const unsigned up = __shfl_up_sync(all, f[0], 1), down = __shfl_down_sync(all, f[0], 1);
  const unsigned heads = __ballot_sync(all, f[0] != (lane == 0 ? b[0] : up)), ends = __ballot_sync(all, f[0] != down);
  unsigned used = __ballot_sync(all, lane < count && f[0] < rows);
  if (lead && !lead_long) used &= to >= 32 ? 0u : all << to;
  const bool live = unit < units;
  auto load = [&](unsigned int v) { return reinterpret_cast<const Unit<T, N> *>(grad + (long long)v * a.grad_stride)[unit]; };
  Unit<T, N> g[LG_TILE];
#pragma unroll
  for (int j = 0; j < LG_TILE; ++j) {
    const unsigned int v = __shfl_sync(all, val[0], j);
    if (live && (used >> j & 1u)) g[j] = load(v);
  }
  float acc[N];
  bool opened = false;                               // the run at hand began in this tile
  auto leave = [&](int slot) {
    float *p = a.part + ((long long)tile * 2 + slot) * a.part_ld + unit * N;
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = acc[i];
  };
  auto add = [&](const Unit<T, N> &u) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += Tok<T>::up(u.e[i]);
  };
#pragma unroll
  for (int j = 0; j < LG_TILE; ++j) {
    const unsigned k = __shfl_sync(all, f[0], j);
    if (!live || !(used >> j & 1u)) continue;
    if ((heads >> j & 1u) || j == 0) {
      opened = heads >> j & 1u;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
    }
    add(g[j]);
    if (!(ends >> j & 1u)) continue;
    if (opened) grad_store<T, N>(out, a, k, unit, acc);
    else leave(0);
  }
  if (!trail || !(used >> (count - 1) & 1u)) return;
  opened = to < count || !lead;
  if (!opened || trail_long) {
    if (live) leave(opened ? 1 : 0);
    return;
  }
  for (int at = count; at < count + behind; at += LG_TILE) {       // the rest of the run
#pragma unroll
    for (int u = 0; u < LG_TILE; ++u) {
      const unsigned v0 = __shfl_sync(all, val[0], (at + u) & 31), v1 = __shfl_sync(all, val[1], (at + u) & 31);
      if (live && at + u < count + behind) g[u] = load(at + u < 32 ? v0 : v1);
    }
#pragma unroll
    for (int u = 0; u < LG_TILE; ++u) if (live && at + u < count + behind) add(g[u]);
  }
  if (live) grad_store<T, N>(out, a, last, unit, acc);
}

// A CTA looks through LG_JOIN_TILES tiles for long runs that begin in them, and adds up the parts of each over 32 units of columns: the
// warps take every LG_JOIN_WARPS-th of the run's further tiles, eight parts in flight with the ids that say whether the run reaches them,
// and the warps' sums are added in their order.
template <class T, int N>
__global__ void __launch_bounds__(32 * LG_JOIN_WARPS) lookup_grad_join_kernel(T *__restrict__ out, GradArgs a) {
  __shared__ float sums[LG_JOIN_WARPS][32 * N];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, units = a.dim / N, blocks = (units + 31) / 32;
  const int group = (int)(blockIdx.x / blocks), unit = (int)(blockIdx.x % blocks) * 32 + lane;
  const long long mine = (long long)group * LG_JOIN_TILES + lane, end = (mine + 1) * LG_TILE, far = end + LG_LONG - 1;
  unsigned long long key = ~0ull, before = ~0ull, behind = ~0ull;
  if (far < a.n) {
    key = a.keys[end - 1];
    behind = a.keys[far];                                                // the list is sorted: all between are the same id as well
    if (mine > 0) before = a.keys[end - LG_TILE - 1];
  }
  const bool begins = key < (unsigned long long)a.num_rows && behind == key && before != key;
  const bool live = unit < units;
  for (unsigned todo = __ballot_sync(0xffffffffu, begins); todo; todo &= todo - 1u) {        // (the same in every warp)
    const int src = __ffs(todo) - 1;
    const long long tile = (long long)group * LG_JOIN_TILES + src;
    const unsigned long long k = __shfl_sync(0xffffffffu, key, src);
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    if (w == 0 && live) {
      const float *p = a.part + (tile * 2 + 1) * a.part_ld + unit * N;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = p[i];
    }
    bool on = true;
    for (long long t0 = tile + 1 + w; on; t0 += 8 * LG_JOIN_WARPS) {
      float part[8][N];
      bool in[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const long long t = t0 + u * LG_JOIN_WARPS;
        in[u] = t * LG_TILE < a.n && a.keys[t * LG_TILE < a.n ? t * LG_TILE : 0] == k;
        const float *p = a.part + (t * LG_TILE < a.n ? t : 0) * 2 * a.part_ld + unit * N;
#pragma unroll
        for (int i = 0; i < N; ++i) part[u][i] = live ? p[i] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        on = on && in[u];
        if (on) {
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] += part[u][i];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) sums[w][lane * N + i] = acc[i];
    __syncthreads();
    if (w != 0 || !live) continue;
    for (int o = 1; o < LG_JOIN_WARPS; ++o) {
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += sums[o][lane * N + i];
    }
    grad_store<T, N>(out, a, k, unit, acc);
  }
}

// ---- a short list -------------------------------------------------------------------------------------------
// Up to LS_SMALL occurrences in one launch: a CTA per occurrence looks through the list for the others of its id, and the CTAs of an id's
// first occurrences share out the blocks of 32 units of its row, a CTA to a block where there are as many; the CTAs behind them write the
// zeros of the rows that the list does not name.  The warps of a CTA take blocks, and where it has fewer blocks than warps, parts of the
// occurrences, added in their order.  fp32, against sorting: 512 ids into 12,574 x 516 8 us and
// 14, 1398 11 and 17; all of one id 8 and 16, 15 and 18.
#define LS_SMALL 1536
#define LS_SMALL_WORDS 1024             // most words of named rows of a CTA that writes zeros

template <class T, int N, int PER>
__global__ void __launch_bounds__(256, 3) lookup_grad_small_kernel(const T *__restrict__ grad, const long long *__restrict__ ids, T *__restrict__ out, GradArgs a, int *errors) {
  __shared__ union { float sums[8][32 * N]; unsigned named[LS_SMALL_WORDS]; } sh;
  __shared__ unsigned short list[256 * PER];
  __shared__ int counts[8], place;
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (blockIdx.x >= (unsigned)a.n) {
    const long long cta = (long long)blockIdx.x - a.n, r0 = cta * a.zero_words * 32;
    for (int i = threadIdx.x; i < a.zero_words; i += 256) sh.named[i] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += 256) {
      const long long r = ids[i] - r0;
      if (r >= 0 && r < a.zero_words * 32ll) atomicOr(&sh.named[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    lookup_zeros<T, N>(out, a, r0, sh.named);
    return;
  }
  const int me = blockIdx.x;
  const long long id = ids[me];
  if (id < 0 || id >= a.num_rows) {
    if (threadIdx.x == 0 && errors) atomicOr(errors, TOK_ERR_ID);
    return;
  }
  // thread t looks at occurrences PER t to PER t + PER - 1: the matches of the whole list lie in the order of the threads
  const int i0 = PER * threadIdx.x;
  unsigned match = 0u;
#pragma unroll
  for (int k = 0; k < PER; ++k) match |= i0 + k < a.n && ids[i0 + k] == id ? 1u << k : 0u;
  const int mine = __popc(match);
  int at = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, at, o); if (lane >= o) at += v; }
  if (lane == 31) counts[w] = at;
  at -= mine;
  __syncthreads();
  int total = 0;
  for (int k = 0; k < 8; ++k) { at += k < w ? counts[k] : 0; total += counts[k]; }
  for (unsigned m = match; m; m &= m - 1u) {
    const int i = i0 + __ffs(m) - 1;
    if (i == me) place = at;
    list[at++] = (unsigned short)i;
  }
  __syncthreads();
  const int units = a.dim / N, blocks = (units + 31) / 32;
  const int share = total < blocks ? total : blocks;                     // CTAs of this id that have blocks: place, place + share, ..
  if (place >= share) return;
  const int own = (blocks - place + share - 1) / share;
  const int parts = own > 4 ? 1 : own > 2 ? 2 : own > 1 ? 4 : 8;         // warps to a block
  const int part = w % parts, per = (total + parts - 1) / parts, lo = part * per, hi = lo + per < total ? lo + per : total;
  for (int o = w / parts; o < (parts > 1 ? 8 / parts : own); o += 8 / parts) {                   // (with several parts, once)
    const int b = place + o * share;
    const int unit = b * 32 + lane;
    const bool live = unit < units;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    for (int k = lo; live && k < hi; k += 8) {
      Unit<T, N> g[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) if (k + u < hi) g[u] = reinterpret_cast<const Unit<T, N> *>(grad + (long long)list[k + u] * a.grad_stride)[unit];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (k + u >= hi) break;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += Tok<T>::up(g[u].e[i]);
      }
    }
    if (parts > 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh.sums[w][lane * N + i] = acc[i];
      __syncthreads();
      if (part == 0)
        for (int o = 1; o < parts; ++o)
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] += sh.sums[w + o][lane * N + i];
    }
    if (part == 0 && live) grad_store<T, N>(out, a, (unsigned long long)id, unit, acc);
  }
}

// ---- sorting ------------------------------------------------------------------------------------------------
// Up to LS_MAX occurrences: one cluster of eight CTAs sorts them by id (a stable radix sort, digits of up to nine bits, the list in
// registers and shared memory) and notes which rows are named.  16,384 ids: 15 us, a chain of barriers; the launches of the sort for longer
// lists, seven for two passes, took 57 us.
#define LS_CTAS 8
#define LS_THREADS 1024
#define LS_WARPS 32
#define LS_BINS 512
#define LS_MAX (LS_CTAS * LS_THREADS * 8)

struct SortIds {
  const long long *ids; long long num_rows; int n, bits; unsigned long long *keys; unsigned int *vals; int *errors;
  unsigned int *named;                                     // null: not asked for
};

template <int IPT>
static constexpr size_t ls_smem() { return (size_t)LS_THREADS * IPT * 8 + LS_WARPS * LS_BINS * 2 + LS_CTAS * LS_BINS * 4 + LS_BINS * 4 + 64; }

template <int IPT>
__global__ void __cluster_dims__(LS_CTAS, 1, 1) __launch_bounds__(LS_THREADS) lookup_sort_kernel(SortIds a) {
  extern __shared__ __align__(16) unsigned char ls_smem_raw[];
  cg::cluster_group cluster = cg::this_cluster();
  const int t = threadIdx.x;
  pdl_begin();
  if (a.named) for (long long i = (long long)cluster.block_rank() * LS_THREADS + t; i < (a.num_rows + 31) / 32; i += LS_CTAS * LS_THREADS) a.named[i] = 0u;
  __threadfence();
  cluster.sync();                                                        // no row is named yet, and every CTA of the cluster runs
  uint2 *buf = (uint2 *)ls_smem_raw;                                      // this CTA's part of the list
  unsigned short *cnt = (unsigned short *)(buf + LS_THREADS * IPT);       // [warps][bins]
  unsigned int *all = (unsigned int *)(cnt + LS_WARPS * LS_BINS);         // [CTAs][bins]
  unsigned int *base = all + LS_CTAS * LS_BINS, *wsum = base + LS_BINS;
  const int rank = (int)cluster.block_rank(), lane = t & 31, w = t >> 5;
  const int passes = (a.bits + 8) / 9, db = (a.bits + passes - 1) / passes, bins = 1 << db;
  const unsigned int mask = (unsigned int)bins - 1u, lt = (1u << lane) - 1u;
  uint2 item[IPT];
  unsigned int off[IPT];
#pragma unroll
  for (int i = 0; i < IPT; ++i) {
    const int o = (rank * LS_WARPS + w) * 32 * IPT + i * 32 + lane;
    unsigned int key = 0xffffffffu;                                       // beyond the list: behind everything
    if (o < a.n) {
      const long long id = a.ids[o];
      const bool bad = id < 0 || id >= a.num_rows;
      if (bad && a.errors) atomicOr(a.errors, TOK_ERR_ID);
      key = (unsigned int)(bad ? a.num_rows : id);
      if (a.named && !bad) atomicOr(a.named + (key >> 5), 1u << (key & 31));
    }
    item[i] = make_uint2(key, (unsigned int)o);
  }
  unsigned short *wc = cnt + w * LS_BINS;
  for (int pass = 0, shift = 0; pass < passes; ++pass, shift += db) {
    for (int i = lane; i < LS_BINS / 2; i += 32) reinterpret_cast<unsigned int *>(wc)[i] = 0u;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const unsigned int dg = (item[i].x >> shift) & mask;
      const unsigned int peers = __match_any_sync(0xffffffffu, dg);
      const unsigned int before = wc[dg];
      __syncwarp();
      if ((peers & lt) == 0u) wc[dg] = (unsigned short)(before + __popc(peers));
      __syncwarp();
      off[i] = before + __popc(peers & lt);
    }
    __syncthreads();
    if (t < bins) {
      unsigned int run = 0u;
#pragma unroll 8
      for (int o = 0; o < LS_WARPS; ++o) { const unsigned int c = cnt[o * LS_BINS + t]; cnt[o * LS_BINS + t] = (unsigned short)run; run += c; }
#pragma unroll
      for (int o = 0; o < LS_CTAS; ++o) cluster.map_shared_rank(all, o)[rank * LS_BINS + t] = run;
    }
    cluster.sync();                                                       // the CTAs' counts are everywhere
    unsigned int total = 0u, lower = 0u;
    if (t < bins) {
#pragma unroll
      for (int o = 0; o < LS_CTAS; ++o) { const unsigned int v = all[o * LS_BINS + t]; total += v; lower += o < rank ? v : 0u; }
    }
    if (t < LS_BINS) {
      unsigned int incl = total;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const unsigned int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
      if (lane == 31) wsum[w] = incl;
      base[t] = incl - total + lower;
    }
    __syncthreads();
    if (t < LS_BINS) {
      unsigned int under = 0u;
#pragma unroll
      for (int o = 0; o < LS_BINS / 32; ++o) under += o < w ? wsum[o] : 0u;
      base[t] += under;
    }
    __syncthreads();
    const bool last = pass == passes - 1;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const unsigned int dg = (item[i].x >> shift) & mask, pos = base[dg] + wc[dg] + off[i];
      if (!last) cluster.map_shared_rank(buf, pos / (LS_THREADS * IPT))[pos % (LS_THREADS * IPT)] = item[i];
      else if (pos < (unsigned int)a.n) { a.keys[pos] = item[i].x; a.vals[pos] = item[i].y; }
    }
    if (!last) {
      cluster.sync();
#pragma unroll
      for (int i = 0; i < IPT; ++i) item[i] = buf[(w * IPT + i) * 32 + lane];
    }
  }
}

// What is sorted: (id, occurrence), ids outside of the table as num_rows.
__global__ void __launch_bounds__(256) id_keys_kernel(const long long *__restrict__ ids, long long num_rows, int n, unsigned long long *__restrict__ keys,
                                                      unsigned int *__restrict__ vals, int *errors, unsigned int *named) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long id = ids[i];
  const bool bad = id < 0 || id >= num_rows;
  if (bad && errors) atomicOr(errors, TOK_ERR_ID);
  if (named && !bad) atomicOr(named + (id >> 5), 1u << (id & 31));
  keys[i] = (unsigned long long)(bad ? num_rows : id);
  vals[i] = (unsigned int)i;
}

static bool unit_fits(const void *p, long long stride, int dim, int size, int n) {
  const int b = n * size;
  return dim % n == 0 && (stride * size) % b == 0 && ((uintptr_t)p & (b - 1)) == 0;
}

struct LookupCall {
  const void *table; long long row_stride, num_rows; int dim; const long long *ids; long long n; float scale; void *out; int *errors;
  cudaStream_t st;
};
template <class T, int N, int U>
static void lookup_launch(const LookupCall &c) {
  int G = 1;
  while (G < 256 && G * U < c.dim / N) G *= 2;
  const long long per = 256 / G;
  pbg_launch_in_order(lookup_kernel<T, N, U>, dim3((unsigned)((c.n + per - 1) / per)), 256, 0, c.st, (const T *)c.table, c.row_stride, c.num_rows, c.dim, G,
                      c.ids, c.n, c.scale, (T *)c.out, c.errors);
}
template <class T, int N>
static void lookup_units(const LookupCall &c) {
  // Four units per thread hide the loads' latency where there is work for all SMs; a few rows are spread as thin as they go.
  if (c.n * (c.dim / N) >= 1024ll * pbg_sm_count()) lookup_launch<T, N, 4>(c);
  else lookup_launch<T, N, 1>(c);
}
template <class T>
static void lookup_type(const LookupCall &c) {
  constexpr int V = Tok<T>::VEC, S = sizeof(T);
  auto fits = [&](int n) { return unit_fits(c.table, c.row_stride, c.dim, S, n) && unit_fits(c.out, c.dim, c.dim, S, n); };
  if (fits(V)) lookup_units<T, V>(c);
  else if (fits(V / 2)) lookup_units<T, V / 2>(c);
  else if (V == 8 && fits(2)) lookup_units<T, 2>(c);
  else lookup_units<T, 1>(c);
}

extern "C" int pbg_embedding_lookup(const void *table, int64_t row_stride, int64_t num_rows, int32_t dim, int32_t dtype, const int64_t *ids,
                                    int64_t n, float scale, void *out, int32_t *errors, void *stream) {
  if (n < 0 || num_rows < 0 || dim <= 0 || !tok_type(dtype) || row_stride < 0 || scale != scale) return PBG_ERR_BAD_ARGUMENT;
  if (n == 0) return PBG_OK;
  if (!table || !ids || !out || num_rows == 0) return PBG_ERR_BAD_ARGUMENT;
  if (n > 0x7fffffffll || num_rows > 0x7fffffffll || dim > 65536) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  const LookupCall c{table, row_stride, num_rows, dim, (const long long *)ids, n, scale, out, errors, (cudaStream_t)stream};
  TOK_DISPATCH(dtype, lookup_type, c);
  return tok_status();
}

static int grad_part_ld(int dim) { return (dim + 3) / 4 * 4; }
struct GradPlace { int64_t keys, vals, named, hist, part, bytes; };          // two of keys and of vals
static GradPlace grad_place(int64_t n, int64_t num_rows, int dim) {
  GradPlace p = {};
  if (n <= LS_SMALL) return p;                                           // nothing is sorted
  p.keys = 0;
  p.vals = p.keys + 2 * tok_up(n * 8, 256);
  p.named = p.vals + 2 * tok_up(n * 4, 256);
  p.hist = p.named + tok_up((num_rows + 31) / 32 * 4, 256);
  p.part = p.hist + (n <= LS_MAX ? 0 : tok_up((int64_t)pbg_sort_hist_entries((int)n) * 4, 256));
  p.bytes = p.part + (n + LG_TILE - 1) / LG_TILE * 2 * grad_part_ld(dim) * 4;
  return p;
}
extern "C" int64_t pbg_embedding_lookup_grad_workspace(int64_t n, int64_t num_rows, int32_t dim) {
  if (n <= 0 || num_rows <= 0 || dim <= 0 || n > (1ll << 30)) return 0;
  return grad_place(n, num_rows, dim).bytes;
}

struct LookupGradCall { const void *grad; const long long *ids; void *out; GradArgs a; int *errors; cudaStream_t st; };
template <class T, int N>
static void lookup_grad_launch(const LookupGradCall &c) {
  const long long tiles = (c.a.n + LG_TILE - 1) / LG_TILE, units = c.a.dim / N, blocks = (units + 31) / 32;
  GradArgs a = c.a;
  a.sum_ctas = (int)((tiles * blocks + 7) / 8);
  a.by_units = FastDiv((int)units);
  const long long words = 65536 / (32ll * c.a.dim * (long long)sizeof(T));                   // some 64 KB to a CTA
  a.zero_words = (int)(words < 1 ? 1 : words < LS_SMALL_WORDS ? words : LS_SMALL_WORDS);
  const long long zero_ctas = a.accumulate ? 0 : ((a.num_rows + 31) / 32 + a.zero_words - 1) / a.zero_words;
  if (a.n <= LS_SMALL) {
    auto kernel = a.n <= 512 ? lookup_grad_small_kernel<T, N, 2> : lookup_grad_small_kernel<T, N, LS_SMALL / 256>;
    pbg_launch(kernel, dim3((unsigned)(a.n + zero_ctas)), 256, 0, c.st, (const T *)c.grad, c.ids, (T *)c.out, a, c.errors);
    return;
  }
  pbg_launch(lookup_grad_kernel<T, N>, dim3((unsigned)(a.sum_ctas + zero_ctas)), 256, 0, c.st, (const T *)c.grad, (T *)c.out, a);
  pbg_launch(lookup_grad_join_kernel<T, N>, dim3((unsigned)((tiles + LG_JOIN_TILES - 1) / LG_JOIN_TILES * blocks)), 32 * LG_JOIN_WARPS, 0, c.st, (T *)c.out, a);
}
template <class T>
static void lookup_grad_type(const LookupGradCall &c) {
  constexpr int V = Tok<T>::VEC, S = sizeof(T);
  auto fits = [&](int n) { return unit_fits(c.grad, c.a.grad_stride, c.a.dim, S, n) && unit_fits(c.out, c.a.out_stride, c.a.dim, S, n); };
  if (fits(V)) lookup_grad_launch<T, V>(c);
  else if (fits(V / 2)) lookup_grad_launch<T, V / 2>(c);
  else if (V == 8 && fits(2)) lookup_grad_launch<T, 2>(c);
  else lookup_grad_launch<T, 1>(c);
}
template <int IPT>
static void sort_launch(const SortIds &a, cudaStream_t st) {
  pbg_opt_in_smem((const void *)lookup_sort_kernel<IPT>, (int)ls_smem<IPT>());
  pbg_launch(lookup_sort_kernel<IPT>, dim3(LS_CTAS), LS_THREADS, ls_smem<IPT>(), st, a);
}

extern "C" int pbg_embedding_lookup_grad(const void *grad, int64_t grad_stride, const int64_t *ids, int64_t n, int64_t num_rows, int32_t dim,
                                         int32_t dtype, float scale, void *out, int64_t out_stride, int32_t accumulate, void *workspace,
                                         int64_t workspace_bytes, int32_t *errors, void *stream) {
  if (n < 0 || num_rows < 0 || dim <= 0 || !tok_type(dtype) || grad_stride < 0 || out_stride < dim || scale != scale) return PBG_ERR_BAD_ARGUMENT;
  if (num_rows == 0) return n == 0 ? PBG_OK : PBG_ERR_BAD_ARGUMENT;
  if (!out || (n > 0 && (!grad || !ids))) return PBG_ERR_BAD_ARGUMENT;
  if (n > (1ll << 30) || num_rows > 0x7fffffffll - 1 || dim > 65536) return PBG_ERR_TOO_LARGE;
  const GradPlace p = n > 0 ? grad_place(n, num_rows, dim) : GradPlace{};
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255))) return PBG_ERR_BAD_ARGUMENT;
  if ((n + LG_TILE - 1) / LG_TILE * (((long long)dim + 31) / 32) > 0x7fffffffll) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  unsigned char *ws = (unsigned char *)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  LookupGradCall c{grad, (const long long *)ids, out, {}, errors, st};
  c.a.grad_stride = grad_stride; c.a.out_stride = out_stride; c.a.num_rows = num_rows;
  c.a.n = (int)n; c.a.dim = dim; c.a.part_ld = grad_part_ld(dim); c.a.accumulate = accumulate != 0; c.a.scale = scale;
  if (n <= LS_SMALL) {
    if (n > 0 || !accumulate) TOK_DISPATCH(dtype, lookup_grad_type, c);
  } else {
    SortPlan sp;
    for (int i = 0; i < 2; ++i) {
      sp.keys[i] = (unsigned long long *)(ws + p.keys + i * tok_up(n * 8, 256));
      sp.vals[i] = (unsigned int *)(ws + p.vals + i * tok_up(n * 4, 256));
    }
    sp.hist = (unsigned int *)(ws + p.hist);
    sp.max_n = (int)n;
    sp.result = 0;
    unsigned int *named = accumulate ? nullptr : (unsigned int *)(ws + p.named);
    int bits = 1;
    while ((unsigned long long)num_rows >> bits) ++bits;
    if (n <= LS_MAX) {
      const SortIds a{(const long long *)ids, num_rows, (int)n, bits, sp.keys[0], sp.vals[0], errors, named};
      if (n <= LS_MAX / 8) sort_launch<1>(a, st);
      else if (n <= LS_MAX / 4) sort_launch<2>(a, st);
      else if (n <= LS_MAX / 2) sort_launch<4>(a, st);
      else sort_launch<8>(a, st);
    } else {
      if (named && cudaMemsetAsync(named, 0, (size_t)(num_rows + 31) / 32 * 4, st) != cudaSuccess) pbg_note_launch();
      pbg_launch_in_order(id_keys_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, (const long long *)ids, (long long)num_rows, (int)n, sp.keys[0], sp.vals[0], errors, named);
      pbg_sort(sp, (int)n, bits, st);
    }
    c.a.named = named;
    c.a.keys = sp.keys[sp.result];
    c.a.vals = sp.vals[sp.result];
    c.a.part = (float *)(ws + p.part);
    TOK_DISPATCH(dtype, lookup_grad_type, c);
  }
  return tok_status();
}
