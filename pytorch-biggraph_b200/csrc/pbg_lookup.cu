// Rows of a table by id (scaled), and the gradient of that: the rows' gradients summed by id.
//
//   lookup  out[i] = s W[id_i]                         n rows read, n written: HBM
//   grad    dW[v]  = s sum_{i : id_i = v} g_i          n rows read, num_rows written: HBM, and the sort's latency
//
// The gradient sorts (id, i) first, so that the occurrences of an id lie next to each other in the order of i, and no sum
// depends on the order in which anything arrives.  Sums are fp32, rounded to the output's type once.
#include "pbg_tokens.cuh"

// N elements of T as one access of N * sizeof(T) bytes
template <class T, int N> struct __align__(sizeof(T) * N) Unit { T e[N]; };

// A group of G threads moves a row, U units per thread in flight.
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
// The sorted list is cut into tiles of LG_TILE occurrences; a warp sums one tile over 32 units of columns.  A run of one id that
// lies inside a tile is written out at once.  A run that reaches into the next tile is left as fp32 partial sums -- the tile's
// first run in slot 0, its last one in slot 1 -- and the join adds a run's partials in the order of the tiles.
#define LG_TILE 16
#define LG_JOIN_WARPS 8

struct GradArgs {
  const unsigned long long *keys;      // sorted ids, those outside of the table behind all others
  const unsigned int *vals;
  float *part;                         // [tiles][2][dim rounded up to 4]
  long long grad_stride, out_stride, num_rows;
  int n, dim, part_ld, accumulate;
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

template <class T, int N>
__global__ void __launch_bounds__(256) lookup_grad_kernel(const T *__restrict__ grad, T *__restrict__ out, GradArgs a) {
  pdl_begin();
  const int lane = threadIdx.x & 31, units = a.dim / N, blocks = (units + 31) / 32;
  const long long job = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int tile = (int)(job / blocks), unit = (int)(job - (long long)tile * blocks) * 32 + lane;
  const int i0 = tile * LG_TILE;
  if (i0 >= a.n) return;
  const int count = a.n - i0 < LG_TILE ? a.n - i0 : LG_TILE;
  // lane j holds occurrence j of the tile; lanes 16 and 17 the neighbours on either side
  unsigned long long key = ~0ull;
  unsigned int val = 0u;
  if (lane < count) { key = a.keys[i0 + lane]; val = a.vals[i0 + lane]; }
  const unsigned long long before = i0 > 0 ? a.keys[i0 - 1] : ~0ull, after = i0 + count < a.n ? a.keys[i0 + count] : ~0ull;
  const bool live = unit < units;
  Unit<T, N> g[LG_TILE];
#pragma unroll
  for (int j = 0; j < LG_TILE; ++j) {
    const unsigned long long k = __shfl_sync(0xffffffffu, key, j);
    const unsigned int v = __shfl_sync(0xffffffffu, val, j);
    if (live && k < (unsigned long long)a.num_rows) g[j] = reinterpret_cast<const Unit<T, N> *>(grad + (long long)v * a.grad_stride)[unit];
  }
  float acc[N];
  bool opened = false;                               // the run at hand began in this tile
#pragma unroll
  for (int j = 0; j < LG_TILE; ++j) {
    const unsigned long long k = __shfl_sync(0xffffffffu, key, j);
    const unsigned long long prev = j == 0 ? before : __shfl_sync(0xffffffffu, key, j > 0 ? j - 1 : 0);
    unsigned long long next = __shfl_sync(0xffffffffu, key, j + 1);
    if (j >= count || k >= (unsigned long long)a.num_rows) continue;                // (warp-uniform)
    if (j == count - 1) next = after;
    const bool head = k != prev;
    if (head || j == 0) {
      opened = head;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += Tok<T>::up(g[j].e[i]);
    }
    if (k == next && j < count - 1) continue;
    if (!live) continue;
    if (opened && k != next) grad_store<T, N>(out, a, k, unit, acc);
    else {
      float *p = a.part + ((long long)tile * 2 + (opened ? 1 : 0)) * a.part_ld + unit * N;
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = acc[i];
    }
  }
}

// One CTA per (tile, 32 units): where the tile's last run begins in it and goes on, its partials are added up.  The run's further
// tiles are dealt to the warps in blocks and the warps' sums added in their order.
template <class T, int N>
__global__ void __launch_bounds__(32 * LG_JOIN_WARPS) lookup_grad_join_kernel(T *__restrict__ out, GradArgs a) {
  __shared__ float sums[LG_JOIN_WARPS][32 * N];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, units = a.dim / N, blocks = (units + 31) / 32;
  const int tile = (int)(blockIdx.x / blocks), unit = (int)(blockIdx.x % blocks) * 32 + lane;
  const int last = tile * LG_TILE + LG_TILE - 1;
  if (last + 1 >= a.n) return;
  const unsigned long long k = a.keys[last];
  if (k >= (unsigned long long)a.num_rows || a.keys[last + 1] != k) return;
  if (a.keys[last - LG_TILE + 1] == k && tile > 0 && a.keys[last - LG_TILE] == k) return;      // began before this tile
  int lo = last + 1, hi = a.n;                                                                // the run's end: first key behind it
  while (lo < hi) { const int mid = lo + (hi - lo) / 2; if (a.keys[mid] == k) lo = mid + 1; else hi = mid; }
  const int tiles = (lo - 1) / LG_TILE - tile;                                                // further tiles of the run
  const int per = (tiles + LG_JOIN_WARPS - 1) / LG_JOIN_WARPS, t0 = w * per, t1 = t0 + per < tiles ? t0 + per : tiles;
  const bool live = unit < units;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  if (live) {
    if (w == 0) {
      const float *p = a.part + ((long long)tile * 2 + 1) * a.part_ld + unit * N;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = p[i];
    }
#pragma unroll 4
    for (int t = t0; t < t1; ++t) {
      const float *p = a.part + (long long)(tile + 1 + t) * 2 * a.part_ld + unit * N;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += p[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sums[w][lane * N + i] = acc[i];
  __syncthreads();
  if (w != 0 || !live) return;
  for (int o = 1; o < LG_JOIN_WARPS; ++o) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += sums[o][lane * N + i];
  }
  grad_store<T, N>(out, a, k, unit, acc);
}

// Zeros, row by row; rows that lie one behind the other come as one row of all.
template <class T, int N>
__global__ void __launch_bounds__(256) lookup_zero_kernel(T *__restrict__ out, long long stride, long long rows, long long units) {
  Unit<T, N> z;
#pragma unroll
  for (int i = 0; i < N; ++i) z.e[i] = Tok<T>::down(0.f);
  for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
    Unit<T, N> *dst = reinterpret_cast<Unit<T, N> *>(out + r * stride);
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) dst[u] = z;
  }
}

// What is sorted: (id, occurrence), ids outside of the table as num_rows.
__global__ void __launch_bounds__(256) id_keys_kernel(const long long *__restrict__ ids, long long num_rows, int n, unsigned long long *__restrict__ keys,
                                                      unsigned int *__restrict__ vals, int *errors) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long id = ids[i];
  const bool bad = id < 0 || id >= num_rows;
  if (bad && errors) atomicOr(errors, TOK_ERR_ID);
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
  if (c.n * (c.dim / N) >= 148ll * 1024) lookup_launch<T, N, 4>(c);
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
struct GradPlace { int64_t keys, vals, hist, part, bytes; };          // two of keys and of vals
static GradPlace grad_place(int64_t n, int dim) {
  GradPlace p;
  p.keys = 0;
  p.vals = p.keys + 2 * tok_up(n * 8, 256);
  p.hist = p.vals + 2 * tok_up(n * 4, 256);
  p.part = p.hist + tok_up((int64_t)pbg_sort_hist_entries((int)n) * 4, 256);
  p.bytes = p.part + (n + LG_TILE - 1) / LG_TILE * 2 * grad_part_ld(dim) * 4;
  return p;
}
extern "C" int64_t pbg_embedding_lookup_grad_workspace(int64_t n, int64_t num_rows, int32_t dim) {
  if (n <= 0 || num_rows <= 0 || dim <= 0 || n > (1ll << 30)) return 0;
  return grad_place(n, dim).bytes;
}

struct LookupGradCall { const void *grad; void *out; GradArgs a; cudaStream_t st; };
template <class T, int N>
static void lookup_grad_launch(const LookupGradCall &c) {
  const long long tiles = (c.a.n + LG_TILE - 1) / LG_TILE, blocks = (c.a.dim / N + 31) / 32;
  pbg_launch(lookup_grad_kernel<T, N>, dim3((unsigned)((tiles * blocks + 7) / 8)), 256, 0, c.st, (const T *)c.grad, (T *)c.out, c.a);
  pbg_launch(lookup_grad_join_kernel<T, N>, dim3((unsigned)(tiles * blocks)), 32 * LG_JOIN_WARPS, 0, c.st, (T *)c.out, c.a);
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
template <class T, int N>
static void zero_launch(const LookupGradCall &c, long long rows, long long width) {
  const long long units = width / N;
  const long long gx = (units + 255) / 256, want = 148 * 8;
  const dim3 grid((unsigned)(gx < want ? gx : want), (unsigned)(rows < 65535 ? rows : 65535));
  pbg_launch_in_order(lookup_zero_kernel<T, N>, grid, 256, 0, c.st, (T *)c.out, c.a.out_stride, rows, units);
}
template <class T>
static void zero_type(const LookupGradCall &c) {
  constexpr int V = Tok<T>::VEC;
  const bool flat = c.a.out_stride == c.a.dim;
  const long long rows = flat ? 1 : c.a.num_rows, width = flat ? c.a.num_rows * c.a.dim : c.a.dim;
  if (aligned16(c.out) && width % V == 0 && (flat || c.a.out_stride % V == 0)) zero_launch<T, V>(c, rows, width);
  else zero_launch<T, 1>(c, rows, width);
}

extern "C" int pbg_embedding_lookup_grad(const void *grad, int64_t grad_stride, const int64_t *ids, int64_t n, int64_t num_rows, int32_t dim,
                                         int32_t dtype, float scale, void *out, int64_t out_stride, int32_t accumulate, void *workspace,
                                         int64_t workspace_bytes, int32_t *errors, void *stream) {
  if (n < 0 || num_rows < 0 || dim <= 0 || !tok_type(dtype) || grad_stride < 0 || out_stride < dim || scale != scale) return PBG_ERR_BAD_ARGUMENT;
  if (num_rows == 0) return n == 0 ? PBG_OK : PBG_ERR_BAD_ARGUMENT;
  if (!out || (n > 0 && (!grad || !ids || !workspace))) return PBG_ERR_BAD_ARGUMENT;
  if (n > (1ll << 30) || num_rows > 0x7fffffffll - 1 || dim > 65536) return PBG_ERR_TOO_LARGE;
  const GradPlace p = n > 0 ? grad_place(n, dim) : GradPlace{};
  if (workspace_bytes < p.bytes || ((uintptr_t)workspace & 255)) return PBG_ERR_BAD_ARGUMENT;
  if ((n + LG_TILE - 1) / LG_TILE * (((long long)dim + 31) / 32) > 0x7fffffffll) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  unsigned char *ws = (unsigned char *)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  LookupGradCall c{grad, out, {}, st};
  c.a.grad_stride = grad_stride; c.a.out_stride = out_stride; c.a.num_rows = num_rows;
  c.a.n = (int)n; c.a.dim = dim; c.a.part_ld = grad_part_ld(dim); c.a.accumulate = accumulate != 0; c.a.scale = scale;
  if (!accumulate) TOK_DISPATCH(dtype, zero_type, c);
  if (n > 0) {
    SortPlan sp;
    for (int i = 0; i < 2; ++i) {
      sp.keys[i] = (unsigned long long *)(ws + p.keys + i * tok_up(n * 8, 256));
      sp.vals[i] = (unsigned int *)(ws + p.vals + i * tok_up(n * 4, 256));
    }
    sp.hist = (unsigned int *)(ws + p.hist);
    sp.max_n = (int)n;
    sp.result = 0;
    int bits = 1;
    while ((unsigned long long)num_rows >> bits) ++bits;
    pbg_launch_in_order(id_keys_kernel, dim3((unsigned)((n + 255) / 256)), 256, 0, st, (const long long *)ids, (long long)num_rows, (int)n, sp.keys[0], sp.vals[0], errors);
    pbg_sort(sp, (int)n, bits, st);
    c.a.keys = sp.keys[sp.result];
    c.a.vals = sp.vals[sp.result];
    c.a.part = (float *)(ws + p.part);
    TOK_DISPATCH(dtype, lookup_grad_type, c);
  }
  return tok_status();
}
