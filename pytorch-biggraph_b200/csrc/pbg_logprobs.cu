// Log probabilities over rows of scores in memory, and their gradient.
//
// With z = s x:  m = max z,  S = sum e^(z - m),  T = sum (z - m) e^(z - m):
//   lse = m + log S     log p_t = (z_t - m) - log S     H = log S - T / S
// T is never positive, so H is a sum of two numbers of one sign: no cancellation where the distribution is sharp.  The
// exponentials run in base 2, against the largest element so far (each thread its own; the sums are rebased where they join).
// Far from zero an fp32 lse says little about p = e^(z - lse) (half a step of it is 0.03 at 1e6), so that what it leaves of m + log S is
// handed on beside it.
//
// Forward: a row is read once.  Gradient: one read, one write.  HBM bounds both; the forward pass comes near the issue slots too (16-bit
// scores at 6.5 TB/s are 11.6 to an SM and cycle, which issues 128 lanes of instructions: 11 for each score, of which the pass takes
// some seven).  4099 x 131,072 bf16 with the best 8, a call on other buffers each time: 227 to 240 us, 4.7 TB/s, 60 % of the issue slots; the gradient
// of 4096 336 to 349 us, 6.3 TB/s; four rows with the best 20, eight CTAs to a row: 14 us in a graph.
#include <cooperative_groups.h>

#include "pbg_tokens.cuh"

namespace cg = cooperative_groups;

#define LP_THREADS 256                   // of the gradient
#define LP_TOP_MAX 32
#define LP_VECS 4                        // 16-byte vectors per thread and step
#define LP_NO_ID 0x7fffffff

struct LogprobArgs {
  long long row_stride, vocab;
  const long long *targets;
  long long ignore_index;
  float scale;
  int top;
  float *logprob, *entropy, *lse, *lse_rest;      // lse_rest: null where it is not asked for
  long long *rank;
  float *top_logprobs;
  long long *top_ids;
  int *errors;
};

// The 16-byte vectors of a row.  16-bit scores are compared two at a time; the rest is fp32, two products or sums to an instruction.
template <class T> struct Row16;
template <> struct Row16<float> {
  static constexpr unsigned NEG_INF = 0xff800000u;
  float cm;
  __device__ __forceinline__ void start(unsigned w) { cm = __uint_as_float(w); }
  __device__ __forceinline__ void seen(unsigned w) { cm = fmaxf(cm, __uint_as_float(w)); }
  __device__ __forceinline__ float largest() const { return cm; }
};
template <class T, class T2> struct Row16Half {
  T2 m;
  __device__ __forceinline__ void start(unsigned w) { m = *reinterpret_cast<T2 *>(&w); }
  __device__ __forceinline__ void seen(unsigned w) { m = __hmax2(m, *reinterpret_cast<T2 *>(&w)); }
  __device__ __forceinline__ float largest() const { const float2 f = TokPair<T>::up(m); return fmaxf(f.x, f.y); }
};
template <> struct Row16<__nv_bfloat16> : Row16Half<__nv_bfloat16, __nv_bfloat162> { static constexpr unsigned NEG_INF = 0xff80ff80u; };
template <> struct Row16<__half> : Row16Half<__half, __half2> { static constexpr unsigned NEG_INF = 0xfc00fc00u; };

// one word of a vector: two 16-bit scores or one fp32 score
template <class T> __device__ __forceinline__ float2 word_up(unsigned w) { return TokPair<T>::up(*reinterpret_cast<typename TokPair<T>::type *>(&w)); }
template <> __device__ __forceinline__ float2 word_up<float>(unsigned w) { return make_float2(__uint_as_float(w), -INFINITY); }

// What a thread gathers over its part of a row: S and T of its even and odd scores against the reference s.r, and how many scores stand in
// front of the target's.
template <class T>
struct RowScan {
  static constexpr int WORDS = 4 * LP_VECS, VEC = Tok<T>::VEC;
  Soft s;                                // S and T: joined at the end
  unsigned long long S2, T2;
  unsigned rank;
  int target;
  float c, mine, above;                  // scale in base 2; the target's score; the next larger score
  unsigned mine2, above2;                // (the same, twice in a word)

  __device__ __forceinline__ void start(float scale, const T *row, bool known, int target_id) {
    s = Soft{-INFINITY, 0.f, 0.f, 0.f};
    S2 = T2 = f32x2(0.f, 0.f);
    rank = 0u; target = target_id; c = scale * TOK_LOG2E;
    const float nan = __int_as_float(0x7fc00000);
    mine = known ? Tok<T>::up(row[target]) : nan;
    above = mine == INFINITY ? nan : nextafterf(mine, INFINITY);
    if constexpr (sizeof(T) == 2) {
      // the next larger number of the type: the next pattern, towards zero for the negative ones
      const unsigned short b = known ? *reinterpret_cast<const unsigned short *>(row + target) : 0x7fff;
      const unsigned short n = mine != mine || mine == INFINITY ? 0x7fff : mine == 0.f ? 1 : mine > 0.f ? b + 1 : b - 1;
      mine2 = b * 0x10001u;
      above2 = n * 0x10001u;
    }
  }
  __device__ __forceinline__ void raise(float m) {                     // a new largest score
    s.m = m;
    const float r = soft_reference(m), d = fminf(fmaxf((s.r - r) * c, -1e30f), 0.f), f = tok_ex2(d);
    const unsigned long long d2 = f32x2(d, d), f2 = f32x2(f, f), zero = f32x2(0.f, 0.f);
    T2 = f32x2_fma(f32x2_fma(d2, S2, T2), f2, zero);
    S2 = f32x2_fma(S2, f2, zero);
    s.r = r;
  }
  __device__ __forceinline__ void finish() {
    const float2 a = f32x2_parts(S2), b = f32x2_parts(T2);
    s.S = a.x + a.y;
    s.T = b.x + b.y;
  }
  // LP_VECS vectors, `live` of them there (the others hold -inf); element i of vector u has the id first + u * 32 * VEC + i
  // their largest score
  __device__ __forceinline__ float step(const unsigned (&raw)[WORDS], int first, int live) {
    Row16<T> top;
    top.start(raw[0]);
#pragma unroll
    for (int q = 1; q < WORDS; ++q) top.seen(raw[q]);
    const float cm = top.largest();
    if (cm > s.m) raise(cm);
    // (x - r) c, not x c - r c: the rounding of r c would be a factor of all sums, 2^64 where every score is -1e9
    const unsigned long long c2 = f32x2(c, c), r2 = f32x2(-s.r, -s.r), zero = f32x2(0.f, 0.f);
    constexpr int PAIRS = sizeof(T) == 2 ? WORDS : WORDS / 2;
#pragma unroll
    for (int q = 0; q < PAIRS; ++q) {
      const float2 x = sizeof(T) == 2 ? word_up<T>(raw[q]) : make_float2(__uint_as_float(raw[2 * q % WORDS]), __uint_as_float(raw[(2 * q + 1) % WORDS]));
      float2 y = f32x2_parts(f32x2_fma(f32x2_add(f32x2(x.x, x.y), r2), c2, zero));
      y.x = tok_max_nan(y.x, -1000.f);                                   // 2^-1000 is 0 in fp32 too; -inf has no place in T
      y.y = tok_max_nan(y.y, -1000.f);
      const unsigned long long e2 = f32x2(tok_ex2(y.x), tok_ex2(y.y));
      S2 = f32x2_add(S2, e2);
      T2 = f32x2_fma(f32x2(y.x, y.y), e2, T2);
    }
    // scores in front of the target's: larger ones, and equal ones with a smaller id
    if constexpr (sizeof(T) == 2) {
      using P = typename TokPair<T>::type;
      unsigned zero = 0u;
      P count = *reinterpret_cast<P *>(&zero);
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u) {
        unsigned limit = first + u * 32 * VEC + VEC <= target ? mine2 : above2;
#pragma unroll
        for (int q = 0; q < 4; ++q) { unsigned w = raw[4 * u + q]; count = __hadd2(count, __hge2(*reinterpret_cast<P *>(&w), *reinterpret_cast<P *>(&limit))); }
      }
      const float2 f = TokPair<T>::up(count);                          // (at most 16 each)
      rank += (unsigned)(f.x + f.y);
    } else {
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u) {
        const float limit = first + u * 32 * VEC + VEC <= target ? mine : above;
#pragma unroll
        for (int q = 0; q < 4; ++q) rank += __uint_as_float(raw[4 * u + q]) >= limit ? 1u : 0u;
      }
    }
    const int at = target - first, u = at / (32 * VEC), in = at - u * 32 * VEC;
    if (at >= 0 && u < live && in < VEC) {                               // the vector that holds the target
#pragma unroll 1
      for (int i = 0; i < in; ++i) {
        const float2 x = word_up<T>(pick(raw, 4 * u + i * 4 / VEC));
        rank += ((sizeof(T) == 2 && (i & 1)) ? x.y : x.x) == mine ? 1u : 0u;
      }
    }
    return cm;
  }
  // raw[q] for a q that is not known to the compiler (rare paths)
  static __device__ __forceinline__ unsigned pick(const unsigned (&raw)[WORDS], int q) {
    unsigned w = raw[0];
#pragma unroll
    for (int i = 1; i < WORDS; ++i) w = i == q ? raw[i] : w;
    return w;
  }
  __device__ __forceinline__ void edge(float x, int id) {                // a single element
    if (x > s.m) raise(x);
    const float y = tok_max_nan((x - s.r) * c, -1000.f), e = tok_ex2(y);
    S2 = f32x2_add(S2, f32x2(e, 0.f));
    T2 = f32x2_fma(f32x2(y, 0.f), f32x2(e, 0.f), T2);
    rank += x > mine || (x == mine && id < target) ? 1u : 0u;
  }
};

// ---- the best scores ------------------------------------------------------------------------------------
// Order: larger scores first, equal ones by id, NaN as -inf.  The scan leaves the largest score of every thread, and of each sixteenth of
// its turns.  The top-th largest of 64 groups of threads is a threshold that at least `top` scores reach and hardly
// more than that pass.  The sixteenths that reach it are looked through again, all threads helping, and what reaches it is ranked by
// counting.  Where too much does (equal scores, mostly), those above it are taken and the first of those equal to it; where even
// that is too much, the best are found one after the other.  (A sorted list per warp, kept during the scan, took longer than the scan:
// 211 us for 1024 x 131,072 bf16 and the best 8, where the scan takes 59.)
#define LP_CANDIDATES 512
#define LP_SLOTS 16
struct Best { float v; int id; };
__device__ __forceinline__ bool best_before(Best a, Best b) { return a.v > b.v || (a.v == b.v && a.id < b.id); }

// A CTA's part of a row: the elements in front of the first 16-byte boundary and behind the last whole vector (the edges; the last CTA of
// a cluster has them, an element to a lane of its last warp), and every nct-th block of W steps (W: its warps).
template <class T, int W> struct RowPart {
  static constexpr int VEC = Tok<T>::VEC;
  const T *row;
  int vocab, head, vecs, tail, cta, nct;
  __device__ RowPart(const T *r, long long n, int cta_, int nct_) : row(r), vocab((int)n), cta(cta_), nct(nct_) {
    const int off = (int)(((uintptr_t)r & 15) / sizeof(T));
    head = off == 0 ? 0 : VEC - off < n ? VEC - off : (int)n;
    vecs = (int)((n - head) / VEC);
    tail = (int)((n - head) % VEC);
  }
  __device__ bool edges() const { return cta == nct - 1; }
  __device__ int steps() const { return (vecs + 32 * LP_VECS - 1) / (32 * LP_VECS); }                       // of all CTAs
  __device__ int vec(int warp, int turn, int u, int lane) const { return ((turn * nct + cta) * W + warp) * 32 * LP_VECS + u * 32 + lane; }
  __device__ int turns() const { return (steps() + nct * W - 1) / (nct * W); }
  __device__ int edge_id(int lane) const { return lane < 16 ? (lane < head ? lane : -1) : lane - 16 < tail ? vocab - tail + lane - 16 : -1; }
  __device__ float at(int id) const { const float x = Tok<T>::up(row[id]); return x != x ? -INFINITY : x; }
};

template <int W> struct TopShared {
  float group[64];
  float tau;
  int count, flagged;
  float slot[LP_SLOTS][32 * W];           // the largest score of a thread in its `per` turns of that slot
  unsigned short places[LP_CANDIDATES];  // slot x threads + thread
  Best cand[LP_CANDIDATES], list[LP_TOP_MAX], warp_best[W];
  int have;
};

// cand[0 .. count) to list[0 .. have), the first `top` in order
template <int W>
__device__ __forceinline__ void rank_candidates(TopShared<W> &sh, int top) {
  const int n = sh.count;
  for (int i = threadIdx.x; i < n; i += 32 * W) {
    const Best mine = sh.cand[i];
    int ahead = 0;
    for (int k = 0; k < n; ++k) ahead += best_before(sh.cand[k], mine) ? 1 : 0;
    if (ahead < top) sh.list[ahead] = mine;
  }
  if (threadIdx.x == 0) sh.have = n < top ? n : top;
  __syncthreads();
}

template <class T, int W>
__device__ void top_of_part(const RowPart<T, W> &p, float m, int top, TopShared<W> &sh) {
  constexpr int VEC = Tok<T>::VEC;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float g = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  if (W == 8) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
  if (lane % (W / 2) == 0) sh.group[threadIdx.x / (W / 2)] = g;
  if (threadIdx.x == 0) { sh.count = 0; sh.flagged = 0; sh.have = 0; }
  __syncthreads();
  if (threadIdx.x < 64) {
    const float mine = sh.group[threadIdx.x];
    int ahead = 0;
#pragma unroll 16
    for (int k = 0; k < 64; ++k) { const float o = sh.group[k]; ahead += o > mine || (o == mine && k < (int)threadIdx.x) ? 1 : 0; }
    if (ahead == top - 1) sh.tau = mine;
  }
  __syncthreads();
  const float tau = sh.tau;
  const int turns = p.turns(), per = (turns + LP_SLOTS - 1) / LP_SLOTS;
  auto gather = [&](bool strict) {
    for (int k = 0; k * per < turns; ++k) {
      const float x = sh.slot[k][threadIdx.x];
      if (strict ? x > tau : x >= tau) { const int at = atomicAdd(&sh.flagged, 1); if (at < LP_CANDIDATES) sh.places[at] = (unsigned short)(k * (32 * W) + threadIdx.x); }
    }
    __syncthreads();
    if (sh.flagged > LP_CANDIDATES) {                                    // too much already
      if (threadIdx.x == 0) sh.count = LP_CANDIDATES + 1;
      __syncthreads();
      return;
    }
    const int each = per * LP_VECS, items = sh.flagged * each;
    auto take = [&](float x, int id) {
      if (strict ? x > tau : x >= tau) { const int k = atomicAdd(&sh.count, 1); if (k < LP_CANDIDATES) sh.cand[k] = Best{x, id}; }
    };
    for (int i = threadIdx.x; i < items; i += 32 * W) {
      const int place = sh.places[i / each], r = i % each, who = place % (32 * W), turn = place / (32 * W) * per + r / LP_VECS;
      const int v = p.vec(who / 32, turn, r % LP_VECS, who % 32);
      if (turn >= turns || v >= p.vecs) continue;
      float x[VEC];
      tok_unpack<T>(reinterpret_cast<const uint4 *>(p.row + p.head)[v], x);
      float most = x[0];
#pragma unroll
      for (int k = 1; k < VEC; ++k) most = fmaxf(most, x[k]);
      if (!(strict ? most > tau : most >= tau)) continue;
#pragma unroll
      for (int k = 0; k < VEC; ++k) take(x[k], p.head + v * VEC + k);
    }
    if (p.edges() && w == W - 1 && p.edge_id(lane) >= 0) take(p.at(p.edge_id(lane)), p.edge_id(lane));
    __syncthreads();
  };
  bool strict = tau == -INFINITY;                                        // (fewer than `top` groups with a score at all)
  gather(strict);
  if (sh.count > LP_CANDIDATES && !strict) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = sh.flagged = 0;
    __syncthreads();
    strict = true;
    gather(true);
  }
  if (sh.count > LP_CANDIDATES) {
    // one after the other
    Best prev{INFINITY, -1};
    for (int k = 0; k < top; ++k) {
      Best best{-INFINITY, LP_NO_ID};
      auto see = [&](float x, int id) {
        const Best b{x != x ? -INFINITY : x, id};
        if (best_before(prev, b) && best_before(b, best)) best = b;
      };
      for (int turn = 0; turn < p.turns(); ++turn)
        for (int u = 0; u < LP_VECS; ++u) {
          const int v = p.vec(w, turn, u, lane);
          if (v >= p.vecs) break;
          float x[VEC];
          tok_unpack<T>(reinterpret_cast<const uint4 *>(p.row + p.head)[v], x);
#pragma unroll
          for (int e = 0; e < VEC; ++e) see(x[e], p.head + v * VEC + e);
        }
      if (p.edges() && w == W - 1 && p.edge_id(lane) >= 0) see(p.at(p.edge_id(lane)), p.edge_id(lane));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Best b{__shfl_xor_sync(0xffffffffu, best.v, o), __shfl_xor_sync(0xffffffffu, best.id, o)};
        if (best_before(b, best)) best = b;
      }
      __syncthreads();
      if (lane == 0) sh.warp_best[w] = best;
      __syncthreads();
      best = sh.warp_best[0];
      for (int o = 1; o < W; ++o) if (best_before(sh.warp_best[o], best)) best = sh.warp_best[o];
      if (best.id == LP_NO_ID) break;                                    // (the same in every thread)
      if (threadIdx.x == 0) { sh.list[k] = best; sh.have = k + 1; }
      prev = best;
    }
    __syncthreads();
    return;
  }
  rank_candidates(sh, top);
  if (!strict || sh.have >= top) return;
  // the first of those equal to the threshold
  if (w == 0) {
    int have = sh.have;
    auto more = [&](bool there, int id) {                                // a warp's look at 32 elements in the order of their ids
      const bool hit = there && p.at(id) == tau;
      const unsigned hits = __ballot_sync(0xffffffffu, hit);
      const int place = have + __popc(hits & ((1u << lane) - 1u));
      if (hit && place < top) sh.list[place] = Best{tau, id};
      have += __popc(hits);
    };
    if (p.edges()) more(lane < p.head, lane);
    const int span = W * 32 * LP_VECS * VEC;                             // elements of a turn
    for (int turn = 0; turn < p.turns() && have < top; ++turn) {
      const int first = p.head + p.vec(0, turn, 0, 0) * VEC, end = p.head + p.vecs * VEC;
      for (int i = 0; i < span && first + i < end && have < top; i += 32) more(i + lane < span && first + i + lane < end, first + i + lane);
    }
    if (p.edges() && have < top) more(lane < p.tail, p.vocab - p.tail + lane);
    if (lane == 0) sh.have = have < top ? have : top;
  }
  __syncthreads();
}

// A CTA of W warps per row, or a cluster of them where there are fewer rows than SMs could hold; the warps take steps of 32 x LP_VECS vectors in turn.
template <class T, bool TOP, int W>
__global__ void __launch_bounds__(32 * W, 32 / W) logprobs_kernel(const T *__restrict__ logits, LogprobArgs a) {
  constexpr int VEC = Tok<T>::VEC;
  struct Part { Soft s; unsigned rank; };
  __shared__ Part parts[W], cta_part;
  __shared__ TopShared<W> top_shared[1];
  cg::cluster_group cluster = cg::this_cluster();
  const int nct = W == 8 ? (int)cluster.num_blocks() : 1, cta = W == 8 ? (int)cluster.block_rank() : 0;
  const long long n = blockIdx.x / nct;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long target = a.targets[n];
  if (target == a.ignore_index) {                                      // (the whole cluster)
    if (cta == 0 && w == 0) {
      if (lane == 0) { a.logprob[n] = 0.f; a.entropy[n] = 0.f; a.lse[n] = 0.f; a.rank[n] = 0; if (a.lse_rest) a.lse_rest[n] = 0.f; }
      if (TOP && lane < a.top) { a.top_logprobs[n * a.top + lane] = 0.f; a.top_ids[n * a.top + lane] = -1; }
    }
    return;
  }
  const bool known = target >= 0 && target < a.vocab;
  const RowPart<T, W> p(logits + n * a.row_stride, a.vocab, cta, nct);
  RowScan<T> g;
  g.start(a.scale, p.row, known, known ? (int)target : -1);
  const uint4 *vec = reinterpret_cast<const uint4 *>(p.row + p.head);
  const int steps = p.steps();
  const int stride = nct * W, per = (p.turns() + LP_SLOTS - 1) / LP_SLOTS;
  int slot = 0, in_slot = 0;
  float slot_max = -INFINITY;
  if (TOP) for (int k = 0; k < LP_SLOTS; ++k) top_shared[0].slot[k][threadIdx.x] = -INFINITY;
  for (int b = cta * W + w; b < steps; b += stride) {
    const int v0 = b * 32 * LP_VECS + lane;
    unsigned raw[4 * LP_VECS];
    int live = LP_VECS;
    if ((b + 1) * 32 * LP_VECS <= p.vecs) {
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u) {
        const uint4 x = TOP ? vec[v0 + u * 32] : __ldcs(vec + v0 + u * 32);
        raw[4 * u] = x.x; raw[4 * u + 1] = x.y; raw[4 * u + 2] = x.z; raw[4 * u + 3] = x.w;
      }
    } else {
      live = v0 >= p.vecs ? 0 : (p.vecs - v0 + 31) / 32 < LP_VECS ? (p.vecs - v0 + 31) / 32 : LP_VECS;
#pragma unroll
      for (int u = 0; u < LP_VECS; ++u) {
        uint4 x = make_uint4(Row16<T>::NEG_INF, Row16<T>::NEG_INF, Row16<T>::NEG_INF, Row16<T>::NEG_INF);
        if (u < live) x = vec[v0 + u * 32];
        raw[4 * u] = x.x; raw[4 * u + 1] = x.y; raw[4 * u + 2] = x.z; raw[4 * u + 3] = x.w;
      }
    }
    const float cm = g.step(raw, p.head + v0 * VEC, live);
    if (TOP) {
      slot_max = fmaxf(slot_max, cm);
      if (++in_slot == per || b + stride >= steps) { top_shared[0].slot[slot++][threadIdx.x] = slot_max; slot_max = -INFINITY; in_slot = 0; }
    }
  }
  if (p.edges() && w == W - 1 && p.edge_id(lane) >= 0) g.edge(Tok<T>::up(p.row[p.edge_id(lane)]), p.edge_id(lane));
  g.finish();
  const float mine_m = g.s.m;

  // lanes, warps, CTAs
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    soft_join(g.s, soft_shfl(g.s, o), g.c);
    g.rank += __shfl_xor_sync(0xffffffffu, g.rank, o);
  }
  if (lane == 0) parts[w] = Part{g.s, g.rank};
  __syncthreads();
  if (w == 0) {
    g.s = parts[lane % W].s;
    g.rank = parts[lane % W].rank;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      soft_join(g.s, soft_shfl(g.s, o), g.c);
      g.rank += __shfl_xor_sync(0xffffffffu, g.rank, o);
    }
    if (nct > 1 && lane == 0) cta_part = Part{g.s, g.rank};
  }
  if (TOP) top_of_part<T, W>(p, mine_m, a.top, top_shared[0]);
  if (nct > 1) {
    cluster.sync();
    if (cta == 0) {
      if (w == 0)
        for (int o = 1; o < nct; ++o) {
          const Part q = *cluster.map_shared_rank(&cta_part, o);
          soft_join(g.s, q.s, g.c);
          g.rank += q.rank;
        }
      if (TOP) {
        static_assert(8 * LP_TOP_MAX <= LP_CANDIDATES, "the lists of a cluster");
        TopShared<W> &sh = top_shared[0];
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < nct * a.top; i += 32 * W) {
          const TopShared<W> *of = cluster.map_shared_rank(top_shared, i / a.top);
          if (i % a.top < of->have) sh.cand[atomicAdd(&sh.count, 1)] = of->list[i % a.top];
        }
        __syncthreads();
        rank_candidates(sh, a.top);
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
    if (a.lse_rest) a.lse_rest[n] = empty ? 0.f : fmaf(g.s.r, a.scale, -lse) + log_s;
    a.entropy[n] = empty ? 0.f : log_s - g.s.T * TOK_LN2 / g.s.S;
    a.logprob[n] = known && empty ? -INFINITY : (g.mine - g.s.r) * a.scale - log_s;
    a.rank[n] = known ? 1 + (long long)g.rank : 0;
  }
  if (TOP && lane < a.top) {
    const int id = top_shared[0].list[lane].id;
    const float x = Tok<T>::up(p.row[id >= 0 && id < a.vocab ? id : 0]);  // (as it is: NaN stands in the list as -inf)
    a.top_logprobs[n * a.top + lane] = empty ? -INFINITY : (x - g.s.r) * a.scale - log_s;
    a.top_ids[n * a.top + lane] = id;
  }
}

// ---- gradient -----------------------------------------------------------------------------------
//   dx = s (g ([v = t] - p) - h p (log p + H)),  log p = z - lse
struct LogprobGradArgs {
  long long row_stride, out_stride, vocab;
  const long long *targets;
  long long ignore_index;
  float scale;
  const float *lse, *lse_rest, *entropy, *g, *h;
  int *errors;
};
struct RowGrad {
  float scale, lse, rest, g, h, gh;      // rest, h in base 2; gh: g + h H; g, h, gh times the scale
  __device__ __forceinline__ float at(float x) const {
    const float logp = fmaf(fmaf(x, scale, -lse), TOK_LOG2E, -rest), p = tok_ex2(logp);       // (the difference first: it loses nothing)
    return p > 0.f || p != p ? -p * fmaf(h, logp, gh) : 0.f;            // (p = 0: log p may be -inf)
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
  uint4 *tv = reinterpret_cast<uint4 *>(to + head);
  const int v0 = piece * STEP + threadIdx.x;
  // the scores are asked for first: they wait for nothing that is read below
  uint4 raw[LP_VECS];
  float x[ALIKE ? 1 : LP_VECS][VEC];
  if (ALIKE) {
    const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u) if (v0 + u * LP_THREADS < vecs) raw[u] = __ldcs(vec + v0 + u * LP_THREADS);
  } else {
#pragma unroll
    for (int u = 0; u < LP_VECS; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[ALIKE ? 0 : u][i] = v0 + u * LP_THREADS < vecs ? Tok<T>::up(row[head + (v0 + u * LP_THREADS) * VEC + i]) : 0.f;
  }
  const long long target = a.targets[n];
  const bool known = target >= 0 && target < a.vocab && target != a.ignore_index;
  RowGrad r;
  r.scale = a.scale;
  r.lse = a.lse[n];
  r.rest = a.lse_rest ? a.lse_rest[n] * TOK_LOG2E : 0.f;
  // beyond it an lse is too far from zero for p: infinite, or with nothing beside it
  const float most = a.lse_rest ? 3.4e38f : 1e6f;
  r.g = a.g ? a.g[n] * a.scale : 0.f;
  r.h = a.h ? a.h[n] * a.scale : 0.f;
  r.gh = a.h ? fmaf(r.h, a.entropy[n], r.g) : r.g;
  r.h *= TOK_LN2;
  auto report = [&]() {
    if (piece != 0 || threadIdx.x != 0 || !a.errors || target == a.ignore_index) return;
    const float lse = a.lse[n];
    const int bad = !known ? TOK_ERR_ID : fabsf(lse) > most && lse != -INFINITY ? TOK_ERR_LSE : 0;
    if (bad) atomicOr(a.errors, bad);
  };
  // (where it stands decides the compiler's order of the loop: 4096 x 131,072 bf16 take 336 us ALIKE with it in front and 320 behind, else
  // 490 and 780)
  if (!ALIKE) report();
  // zeros for padding and where a mask left nothing: -inf alone, or -1e9 and the like below an lse that has nothing beside it (masks push
  // down; too far above zero nothing explains the row, and it becomes NaN)
  const bool none = !known || r.lse < -most;
  if (r.lse > most) r.lse = __int_as_float(0x7fc00000);
  const int t = none ? -1 : (int)target;
#pragma unroll
  for (int u = 0; u < LP_VECS; ++u) {
    if (v0 + u * LP_THREADS >= vecs) continue;
    const int id0 = head + (v0 + u * LP_THREADS) * VEC;
    if (ALIKE) tok_unpack<T>(raw[u], x[0]);
    float d[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) d[i] = none ? 0.f : r.at(x[ALIKE ? 0 : u][i]);
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
  if (ALIKE) report();
}

// ---- host -----------------------------------------------------------------------------------------
struct LogprobCall { const void *logits; long long n; LogprobArgs a; cudaStream_t st; };
template <class T>
static void logprobs_type(const LogprobCall &c) {
  // A row is split over a cluster only as far as SMs would stand idle and every warp still has a step.
  const long long steps = c.a.vocab / (32 * LP_VECS * Tok<T>::VEC);
  int nct = 1;
  const int sms = pbg_sm_count();
  while (nct < 8 && c.n * nct < 2 * sms && 2 * nct * 8 <= steps) nct *= 2;
  // Four warps to a CTA once there are more rows than CTAs of eight warps at a time: twice as many rows are under way, and one row's joins
  // and best scores, all waiting, are hidden behind others' scans (bf16, eight warps and four: 2368 x 14,951 with the best 8 36 and 28 us,
  // 131,072 140 and 136; two warps gain nothing on 300 scores and lose on 4096).  Not for long rows where a second turn of four-warp CTAs,
  // eight to an SM, would be half empty: 1500 rows of 131,072 fp32 126 and 143, of 131,072 bf16 84 and 86, of 50,257 fp32 56 and 61;
  // of 50,257 bf16 39.7 and 38.8, of 14,951 16.5 and 14.5.  128 KB is the size between these.
  const bool half_empty = c.n > 8ll * sms && c.n <= 12ll * sms && c.a.vocab * (long long)sizeof(T) > 128 * 1024;
  const bool eight = c.n <= 4ll * sms || half_empty;
  void (*kernel)(const T *, LogprobArgs) = eight ? (c.a.top > 0 ? logprobs_kernel<T, true, 8> : logprobs_kernel<T, false, 8>)
                                                 : (c.a.top > 0 ? logprobs_kernel<T, true, 4> : logprobs_kernel<T, false, 4>);
  if (pbg_launch_failed()) return;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(c.n * nct)); cfg.blockDim = dim3(eight ? 256 : 128); cfg.stream = c.st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = nct; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  pbg_note_launch(cudaLaunchKernelEx(&cfg, kernel, (const T *)c.logits, c.a));
}

extern "C" int pbg_token_logprobs_wide(const void *logits, int64_t row_stride, int64_t n, int64_t vocab, int32_t dtype, const int64_t *targets,
                                       int64_t ignore_index, float scale, int32_t top, float *logprob, float *entropy, float *lse, float *lse_rest,
                                       int64_t *rank, float *top_logprobs, int64_t *top_ids, int32_t *errors, void *stream) {
  if (n < 0 || vocab <= 0 || row_stride < 0 || !tok_type(dtype) || !tok_scale(scale) || top < 0 || top > vocab) return PBG_ERR_BAD_ARGUMENT;
  if (n == 0) return PBG_OK;
  if (!logits || !targets || !logprob || !entropy || !lse || !rank || (top > 0 && (!top_logprobs || !top_ids))) return PBG_ERR_BAD_ARGUMENT;
  if (top > LP_TOP_MAX || n > 0x7fffffffll || vocab > 0x7fffffffll - 65536) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  const LogprobCall c{logits, n, LogprobArgs{row_stride, vocab, (const long long *)targets, ignore_index, scale, top, logprob, entropy, lse, lse_rest,
                                             (long long *)rank, top_logprobs, (long long *)top_ids, errors}, (cudaStream_t)stream};
  TOK_DISPATCH(dtype, logprobs_type, c);
  return tok_status();
}
extern "C" int pbg_token_logprobs(const void *logits, int64_t row_stride, int64_t n, int64_t vocab, int32_t dtype, const int64_t *targets,
                                  int64_t ignore_index, float scale, int32_t top, float *logprob, float *entropy, float *lse, int64_t *rank,
                                  float *top_logprobs, int64_t *top_ids, int32_t *errors, void *stream) {
  return pbg_token_logprobs_wide(logits, row_stride, n, vocab, dtype, targets, ignore_index, scale, top, logprob, entropy, lse, nullptr, rank, top_logprobs, top_ids,
                                 errors, stream);
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

extern "C" int pbg_token_logprobs_grad_wide(const void *logits, int64_t row_stride, int64_t n, int64_t vocab, int32_t dtype, const int64_t *targets,
                                            int64_t ignore_index, float scale, const float *lse, const float *lse_rest, const float *entropy,
                                            const float *grad_logprob, const float *grad_entropy, void *out, int64_t out_stride, int32_t *errors, void *stream) {
  if (n < 0 || vocab <= 0 || row_stride < 0 || out_stride < vocab || !tok_type(dtype) || !tok_scale(scale)) return PBG_ERR_BAD_ARGUMENT;
  if (n == 0) return PBG_OK;
  if (!logits || !targets || !lse || !out || (grad_entropy && !entropy)) return PBG_ERR_BAD_ARGUMENT;
  if (vocab > 0x7fffffffll - 65536 || n > 0x7fffffffll || n * ((vocab + 4095) / 4096) > 0x7fffffffll) return PBG_ERR_TOO_LARGE;
  pbg_launch_error() = cudaSuccess;
  const LogprobGradCall c{logits, out, n, LogprobGradArgs{row_stride, out_stride, vocab, (const long long *)targets, ignore_index, scale, lse, lse_rest, entropy,
                                                          grad_logprob, grad_entropy, errors}, (cudaStream_t)stream};
  TOK_DISPATCH(dtype, logprobs_grad_type, c);
  return tok_status();
}
extern "C" int pbg_token_logprobs_grad(const void *logits, int64_t row_stride, int64_t n, int64_t vocab, int32_t dtype, const int64_t *targets,
                                       int64_t ignore_index, float scale, const float *lse, const float *entropy, const float *grad_logprob,
                                       const float *grad_entropy, void *out, int64_t out_stride, int32_t *errors, void *stream) {
  return pbg_token_logprobs_grad_wide(logits, row_stride, n, vocab, dtype, targets, ignore_index, scale, lse, nullptr, entropy, grad_logprob, grad_entropy, out,
                                      out_stride, errors, stream);
}
