// Log probabilities over rows of scores in memory, and their gradient.
//
// With z = s x:  m = max z,  S = sum e^(z - m),  T = sum (z - m) e^(z - m):
//   lse = m + log S     log p_t = (z_t - m) - log S     H = log S - T / S
// T is never positive, so H is a sum of two numbers of one sign: no cancellation where the distribution is sharp.  The
// exponentials run in base 2, against the largest element so far (each thread its own; the sums are rebased where they join).
//
// Forward: a row is read once.  Gradient: one read, one write.  Both are bound by HBM.
#include <cooperative_groups.h>

#include "pbg_tokens.cuh"

namespace cg = cooperative_groups;

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_TOP_MAX 32
#define LP_VECS 4                        // 16-byte vectors per thread and step
#define LP_NO_ID 0x7fffffff

struct LogprobArgs {
  long long row_stride, vocab;
  const long long *targets;
  long long ignore_index;
  float scale;
  int top;
  float *logprob, *entropy, *lse;
  long long *rank;
  float *top_logprobs;
  long long *top_ids;
  int *errors;
};

// A warp's best scores so far: lane l holds the l-th, larger ones first, equal ones by id.
struct Best { float v; int id; };
__device__ __forceinline__ bool best_before(float v, int id, float w, int jd) { return v > w || (v == w && id < jd); }
// v, id: the same in every lane
__device__ __forceinline__ void best_insert(Best &b, float v, int id, int top, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, best_before(b.v, b.id, v, id)));
  if (at >= top) return;
  const float pv = __shfl_up_sync(0xffffffffu, b.v, 1);
  const int pi = __shfl_up_sync(0xffffffffu, b.id, 1);
  if (lane > at) { b.v = pv; b.id = pi; }
  if (lane == at) { b.v = v; b.id = id; }
}

struct RowScan {
  Soft s;
  Best best;
  unsigned rank;                         // scores in front of the target's so far
  int top, lane, target;
  float c, mine, above;                  // scale in base 2; the target's score; the next larger number

  __device__ __forceinline__ void start(float scale, float target_score, int target_id, int top_, int lane_) {
    s = Soft{-INFINITY, 0.f, 0.f, 0.f};
    best = Best{-INFINITY, LP_NO_ID};
    rank = 0u; top = top_; lane = lane_; target = target_id; c = scale * TOK_LOG2E; mine = target_score;
    above = mine == INFINITY ? __int_as_float(0x7fc00000) : nextafterf(mine, INFINITY);
  }

  // V vectors of N elements, `live` of them there (the others hold -inf); element i of vector u has the id first + u * step + i.
  // later: every id is larger than those of the steps before.
  template <bool TOP, int V, int N>
  __device__ __forceinline__ void step(const float (&x)[V * N], int first, int stride, int live, bool later) {
    float cm = x[0];
#pragma unroll
    for (int q = 1; q < V * N; ++q) cm = fmaxf(cm, x[q]);
    if (cm > s.m) { s.m = cm; soft_rebase(s, soft_reference(cm), c); }
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int id0 = first + u * stride;
      // score in front of the target: larger, or equal with a smaller id
      const float limit = id0 + N <= target ? mine : above;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float v = x[u * N + i];
        const float y = tok_max_nan((v - s.r) * c, -1000.f);             // 2^-1000 is 0 in fp32 too; -inf has no place in T
        const float e = tok_ex2(y);
        s.S += e;
        s.T = fmaf(y, e, s.T);
        rank += v >= limit ? 1u : 0u;
      }
      if (N > 1 && u < live && id0 <= target && target < id0 + N) {
#pragma unroll
        for (int i = 0; i < N; ++i) rank += x[u * N + i] == mine && id0 + i < target ? 1u : 0u;
      }
    }
    if (TOP) keep<V, N>(x, first, stride, live, cm, later);
  }

  template <int V, int N>
  __device__ __forceinline__ void keep(const float (&x)[V * N], int first, int stride, int live, float cm, bool later) {
    const float worst = __shfl_sync(0xffffffffu, best.v, top - 1);
    const bool full = __shfl_sync(0xffffffffu, best.id, top - 1) != LP_NO_ID;
    // where all ids are larger than the kept ones, a score equal to the worst does not enter
    const bool strict = full && later;
    if (full && !__any_sync(0xffffffffu, later ? cm > worst : cm >= worst)) return;
    float floor_v = worst;
    if (!full) {
      // the top-th largest of the lanes' maxima: at least `top` scores are not below it
      const float mx = live > 0 && cm == cm ? cm : -INFINITY;
      int at = 0;
      for (int l = 0; l < 32; ++l) {
        const float o = __shfl_sync(0xffffffffu, mx, l);
        at += o > mx || (o == mx && l < lane);
      }
      floor_v = __shfl_sync(0xffffffffu, mx, __ffs(__ballot_sync(0xffffffffu, at == top - 1)) - 1);
    }
    unsigned mask = 0u;
#pragma unroll
    for (int q = 0; q < V * N; ++q) {
      const float v = x[q] == x[q] ? x[q] : -INFINITY;
      if (q / N < live && (strict ? v > floor_v : v >= floor_v)) mask |= 1u << q;
    }
    for (unsigned have; (have = __ballot_sync(0xffffffffu, mask != 0u)) != 0u;) {
      const int src = __ffs(have) - 1, q = __ffs(mask) - 1;
      float pick[V * N];
#pragma unroll
      for (int i = 0; i < V * N; ++i) pick[i] = x[i];
#pragma unroll
      for (int half = V * N / 2; half >= 1; half /= 2)
#pragma unroll
        for (int i = 0; i < half; ++i) pick[i] = (q & half) ? pick[i + half] : pick[i];
      const float v = __shfl_sync(0xffffffffu, pick[0] == pick[0] ? pick[0] : -INFINITY, src);
      const int id = __shfl_sync(0xffffffffu, first + q / N * stride + q % N, src);
      if (lane == src) mask &= mask - 1u;
      best_insert(best, v, id, top, lane);
    }
  }
};

// A cluster of CTAs per row (a single CTA where there are rows for all SMs); the warps take steps of 32 x LP_VECS vectors in turn.
template <class T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const T *__restrict__ logits, LogprobArgs a) {
  constexpr int VEC = Tok<T>::VEC;
  struct Part { Soft s; unsigned rank; };
  __shared__ Part parts[LP_WARPS], cta_part;
  __shared__ Best bests[LP_WARPS][LP_TOP_MAX], cta_best[LP_TOP_MAX];
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const long long n = blockIdx.x / nct;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long target = a.targets[n];
  if (target == a.ignore_index) {                                      // (the whole cluster)
    if (cta == 0 && w == 0) {
      if (lane == 0) { a.logprob[n] = 0.f; a.entropy[n] = 0.f; a.lse[n] = 0.f; a.rank[n] = 0; }
      if (TOP && lane < a.top) { a.top_logprobs[n * a.top + lane] = 0.f; a.top_ids[n * a.top + lane] = -1; }
    }
    return;
  }
  const T *row = logits + n * a.row_stride;
  const bool known = target >= 0 && target < a.vocab;
  // the elements in front of the first 16-byte boundary and behind the last whole vector are the row's edges
  const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
  const int head = off == 0 ? 0 : VEC - off < a.vocab ? VEC - off : (int)a.vocab;
  const int vecs = (int)((a.vocab - head) / VEC), tail = (int)((a.vocab - head) % VEC);
  RowScan g;
  g.start(a.scale, known ? Tok<T>::up(row[target]) : __int_as_float(0x7fc00000), known ? (int)target : -1, a.top, lane);

  const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
  const int steps = (vecs + 32 * LP_VECS - 1) / (32 * LP_VECS);
  for (int b = cta * LP_WARPS + w; b < steps; b += nct * LP_WARPS) {
    const int v0 = b * 32 * LP_VECS + lane;
    const int live = v0 >= vecs ? 0 : (vecs - v0 + 31) / 32 < LP_VECS ? (vecs - v0 + 31) / 32 : LP_VECS;
    uint4 raw[LP_VECS];
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) if (u < live) raw[u] = __ldcs(vec + v0 + u * 32);
    float x[LP_VECS * VEC];
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) {
      float y[VEC];
      tok_unpack<T>(raw[u], y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[u * VEC + i] = u < live ? y[i] : -INFINITY;
    }
    g.step<TOP, LP_VECS, VEC>(x, head + v0 * VEC, 32 * VEC, live, true);
  }
  if (cta == nct - 1 && w == LP_WARPS - 1 && head + tail > 0) {           // the edges: an element per lane
    const int id = lane < 16 ? (lane < head ? lane : -1) : lane - 16 < tail ? (int)(a.vocab - tail) + lane - 16 : -1;
    const float x[1] = {id >= 0 ? Tok<T>::up(row[id]) : -INFINITY};
    g.step<TOP, 1, 1>(x, id >= 0 ? id : LP_NO_ID - 1, 0, id >= 0 ? 1 : 0, false);
  }

  // lanes, warps, CTAs
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    soft_join(g.s, soft_shfl(g.s, o), g.c);
    g.rank += __shfl_xor_sync(0xffffffffu, g.rank, o);
  }
  if (lane == 0) parts[w] = Part{g.s, g.rank};
  if (TOP) bests[w][lane] = g.best;
  __syncthreads();
  if (w == 0) {
    for (int o = 1; o < LP_WARPS; ++o) {
      soft_join(g.s, parts[o].s, g.c);
      g.rank += parts[o].rank;
      if (TOP) {
        for (int l = 0; l < a.top; ++l) {                                // (sorted: the first that does not enter ends it)
          const Best b = bests[o][l];
          const float wv = __shfl_sync(0xffffffffu, g.best.v, a.top - 1);
          const int wi = __shfl_sync(0xffffffffu, g.best.id, a.top - 1);
          if (!best_before(b.v, b.id, wv, wi)) break;
          best_insert(g.best, b.v, b.id, a.top, lane);
        }
      }
    }
    if (nct > 1) { if (lane == 0) cta_part = Part{g.s, g.rank}; if (TOP) cta_best[lane] = g.best; }
  }
  if (nct > 1) {
    cluster.sync();
    if (cta == 0 && w == 0) {
      for (int o = 1; o < nct; ++o) {
        const Part p = *cluster.map_shared_rank(&cta_part, o);
        soft_join(g.s, p.s, g.c);
        g.rank += p.rank;
        if (TOP) {
          const Best *list = cluster.map_shared_rank(cta_best, o);
          const Best mine = list[lane];
          for (int l = 0; l < a.top; ++l) {
            const float v = __shfl_sync(0xffffffffu, mine.v, l), wv = __shfl_sync(0xffffffffu, g.best.v, a.top - 1);
            const int id = __shfl_sync(0xffffffffu, mine.id, l), wi = __shfl_sync(0xffffffffu, g.best.id, a.top - 1);
            if (!best_before(v, id, wv, wi)) break;
            best_insert(g.best, v, id, a.top, lane);
          }
        }
      }
    }
    cluster.sync();                                                      // nobody leaves while its shared memory is read
  }
  if (cta != 0 || w != 0) return;
  const bool empty = g.s.m == -INFINITY && g.s.S == 0.f;                 // nothing but -inf
  const float log_s = logf(g.s.S), lse = empty ? -INFINITY : fmaf(g.s.r, a.scale, log_s);
  if (lane == 0) {
    if (!known && a.errors) atomicOr(a.errors, TOK_ERR_ID);
    a.lse[n] = lse;
    a.entropy[n] = empty ? 0.f : log_s - g.s.T * TOK_LN2 / g.s.S;
    a.logprob[n] = known && empty ? -INFINITY : (g.mine - g.s.r) * a.scale - log_s;
    a.rank[n] = known ? 1 + (long long)g.rank : 0;
  }
  if (TOP && lane < a.top) {
    const float x = Tok<T>::up(row[g.best.id < a.vocab ? g.best.id : 0]);                          // (as it is: NaN stands in the list as -inf)
    a.top_logprobs[n * a.top + lane] = empty ? -INFINITY : (x - g.s.r) * a.scale - log_s;
    a.top_ids[n * a.top + lane] = g.best.id;
  }
}

// ---- gradient -----------------------------------------------------------------------------------
//   dx = s (g ([v = t] - p) - h p (log p + H)),  log p = z - lse
struct LogprobGradArgs {
  long long row_stride, out_stride, vocab;
  const long long *targets;
  long long ignore_index;
  float scale;
  const float *lse, *entropy, *g, *h;
  int *errors;
};
struct RowGrad {
  float scale, lse, g, h, H;             // g, h times the scale
  __device__ __forceinline__ float at(float x) const {
    const float logp = fmaf(x, scale, -lse), p = tok_ex2(logp * TOK_LOG2E);
    return p > 0.f || p != p ? -p * fmaf(h, logp + H, g) : 0.f;         // (p = 0: log p may be -inf)
  }
};

// A CTA takes a piece of a row.  ALIKE: scores and gradients lie alike against 16 bytes; else the scores come one by one.
template <class T, bool ALIKE>
__global__ void __launch_bounds__(LP_THREADS) logprobs_grad_kernel(const T *logits, T *out, LogprobGradArgs a, int pieces) {
  constexpr int VEC = Tok<T>::VEC, STEP = LP_THREADS * LP_VECS;
  const long long n = blockIdx.x / pieces;
  const int piece = (int)(blockIdx.x % pieces);
  const T *row = logits + n * a.row_stride;
  T *to = out + n * a.out_stride;
  const int off = (int)(((uintptr_t)to & 15) / sizeof(T));
  const int head = off == 0 ? 0 : VEC - off < a.vocab ? VEC - off : (int)a.vocab;
  const int vecs = (int)((a.vocab - head) / VEC), tail = (int)((a.vocab - head) % VEC);
  const long long target = a.targets[n];
  const bool known = target >= 0 && target < a.vocab && target != a.ignore_index;
  if (!known && target != a.ignore_index && piece == 0 && threadIdx.x == 0 && a.errors) atomicOr(a.errors, TOK_ERR_ID);
  RowGrad r;
  r.scale = a.scale;
  r.lse = a.lse[n];
  r.g = a.g ? a.g[n] * a.scale : 0.f;
  r.h = a.h ? a.h[n] * a.scale : 0.f;
  r.H = a.h ? a.entropy[n] : 0.f;
  const bool none = !known || r.lse == -INFINITY;                        // padding, or a row of -inf alone: zeros
  const int t = none ? -1 : (int)target;
  uint4 *tv = reinterpret_cast<uint4 *>(to + head);
  const int v0 = piece * STEP + threadIdx.x;
  float x[LP_VECS][VEC];
  if (!none) {
    if (ALIKE) {
      const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
      uint4 raw[LP_VECS];
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u) if (v0 + u * LP_THREADS < vecs) raw[u] = __ldcs(vec + v0 + u * LP_THREADS);
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u) tok_unpack<T>(raw[u], x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u)
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[u][i] = v0 + u * LP_THREADS < vecs ? Tok<T>::up(row[head + (v0 + u * LP_THREADS) * VEC + i]) : 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < LP_VECS; ++u) {
    if (v0 + u * LP_THREADS >= vecs) continue;
    const int id0 = head + (v0 + u * LP_THREADS) * VEC;
    float d[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) d[i] = none ? 0.f : r.at(x[u][i]);
    if (id0 <= t && t < id0 + VEC) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) if (id0 + i == t) d[i] += r.g;
    }
    __stcs(tv + v0 + u * LP_THREADS, tok_pack<T>(d));
  }
  if (piece == pieces - 1 && threadIdx.x < 32) {                         // the edges: an element per lane
    const int lane = threadIdx.x;
    const int id = lane < 16 ? (lane < head ? lane : -1) : lane - 16 < tail ? (int)(a.vocab - tail) + lane - 16 : -1;
    if (id >= 0) to[id] = Tok<T>::down(none ? 0.f : r.at(Tok<T>::up(row[id])) + (id == t ? r.g : 0.f));
  }
}

// ---- host -----------------------------------------------------------------------------------------
struct LogprobCall { const void *logits; long long n; LogprobArgs a; cudaStream_t st; };
template <class T>
static void logprobs_type(const LogprobCall &c) {
  // A row is split over a cluster only as far as SMs would stand idle and every warp still has a step.
  const long long steps = c.a.vocab / (32 * LP_VECS * Tok<T>::VEC);
  int nct = 1;
  while (nct < 8 && c.n * nct < 2 * pbg_sm_count() && 2 * nct * LP_WARPS <= steps) nct *= 2;
  void (*kernel)(const T *, LogprobArgs) = c.a.top > 0 ? logprobs_kernel<T, true> : logprobs_kernel<T, false>;
  if (pbg_launch_failed()) return;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(c.n * nct)); cfg.blockDim = dim3(LP_THREADS); cfg.stream = c.st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = nct; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  pbg_note_launch(cudaLaunchKernelEx(&cfg, kernel, (const T *)c.logits, c.a));
}

extern "C" int pbg_token_logprobs(const void *logits, int64_t row_stride, int64_t n, int64_t vocab, int32_t dtype, const int64_t *targets,
                                  int64_t ignore_index, float scale, int32_t top, float *logprob, float *entropy, float *lse, int64_t *rank,
                                  float *top_logprobs, int64_t *top_ids, int32_t *errors, void *stream) {
  if (n < 0 || vocab <= 0 || row_stride < 0 || !tok_type(dtype) || !tok_scale(scale) || top < 0 || top > vocab) return PBG_ERR_BAD_ARGUMENT;
  if (n == 0) return PBG_OK;
  if (!logits || !targets || !logprob || !entropy || !lse || !rank || (top > 0 && (!top_logprobs || !top_ids))) return PBG_ERR_BAD_ARGUMENT;
  if (top > LP_TOP_MAX || n > 0x0fffffffll || vocab > 0x7fffffffll - 65536) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  const LogprobCall c{logits, n, LogprobArgs{row_stride, vocab, (const long long *)targets, ignore_index, scale, top, logprob, entropy, lse,
                                             (long long *)rank, top_logprobs, (long long *)top_ids, errors}, (cudaStream_t)stream};
  TOK_DISPATCH(dtype, logprobs_type, c);
  return tok_status();
}

struct LogprobGradCall { const void *logits; void *out; long long n; LogprobGradArgs a; cudaStream_t st; };
template <class T>
static void logprobs_grad_type(const LogprobGradCall &c) {
  const long long step = LP_THREADS * LP_VECS * Tok<T>::VEC;
  const long long pieces = (c.a.vocab + step - 1) / step;
  const long long lie = ((uintptr_t)c.logits ^ (uintptr_t)c.out) | (uintptr_t)((c.a.row_stride - c.a.out_stride) * (long long)sizeof(T));
  void (*kernel)(const T *, T *, LogprobGradArgs, int) = (lie & 15) == 0 ? logprobs_grad_kernel<T, true> : logprobs_grad_kernel<T, false>;
  pbg_launch_in_order(kernel, dim3((unsigned)(c.n * pieces)), LP_THREADS, 0, c.st, (const T *)c.logits, (T *)c.out, c.a, (int)pieces);
}

extern "C" int pbg_token_logprobs_grad(const void *logits, int64_t row_stride, int64_t n, int64_t vocab, int32_t dtype, const int64_t *targets,
                                       int64_t ignore_index, float scale, const float *lse, const float *entropy, const float *grad_logprob,
                                       const float *grad_entropy, void *out, int64_t out_stride, int32_t *errors, void *stream) {
  if (n < 0 || vocab <= 0 || row_stride < 0 || out_stride < vocab || !tok_type(dtype) || !tok_scale(scale)) return PBG_ERR_BAD_ARGUMENT;
  if (n == 0) return PBG_OK;
  if (!logits || !targets || !lse || !out || (grad_entropy && !entropy)) return PBG_ERR_BAD_ARGUMENT;
  if (vocab > 0x7fffffffll - 65536 || n > 0x7fffffffll || n * ((vocab + 4095) / 4096) > 0x7fffffffll) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  const LogprobGradCall c{logits, out, n, LogprobGradArgs{row_stride, out_stride, vocab, (const long long *)targets, ignore_index, scale, lse, entropy,
                                                          grad_logprob, grad_entropy, errors}, (cudaStream_t)stream};
  TOK_DISPATCH(dtype, logprobs_grad_type, c);
  return tok_status();
}
