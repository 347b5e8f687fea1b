// Log probabilities over all rows of a table, and their gradients: z = s Q W^T is never stored.
//
//   forward   per query: lse, entropy and log probability of the target          2 N V D operations, Q and W read
//   gradient  dz = s (g ([v = t] - p) - h p (log p + H));  dQ = dz W,  dW = dz^T Q   6 N V D operations (the scores once more)
//
// All products run on the tensor cores (tcgen05, kind::f16) with fp32 accumulators in tensor memory:
//   bf16, fp16   the tensors themselves are the operands, read by TMA where they lie; dz is rounded to the operands' type (that of
//                fp16 scaled by a power of two so that it cannot leave the type's range: its bound is known from g and h)
//   fp32         every operand as two fp16 planes, x 2^k = b0 + b1 (22 bits; k from the largest finite element, so that the
//                planes of everything down to 2^-17 of it are whole), and the three products b1 b0 + b0 b1 + b0 b0: the
//                dropped b1 b1 is 2^-22 of a product, the size of fp32 rounding.  Half the work of three bf16 planes.
//
// One persistent kernel per product, one CTA per SM, tiles of 128 x BN (BN <= 256):
//   warp 0     TMA: stages of 48 KB (64 k-values of one plane, or 32 of two) in a ring of four
//   warp 1     issues tcgen05.mma into one of two accumulators of 256 columns
//   warps 2-9  read the other accumulator and, two warps to every 32 rows: reduce it to (maximum, S, T) per row; or turn it into dz and
//              write that; or write the product
// Every wait is bounded: one that runs out sets bit 2 of the error word, and the CTA stops, frees its tensor memory and returns.
#include "pbg_tc.cuh"
#include "pbg_tokens.cuh"

enum { TAB_BF16 = 0, TAB_F16 = 1, TAB_F32 = 2 };            // operands: bf16, fp16, two fp16 planes
enum { EPI_STATS = 0, EPI_DZ = 1, EPI_OUT = 2 };

#define TAB_STAGES 4
#define TAB_STAGE_BYTES 49152
#define TAB_EPI_WARPS 8
#define TAB_THREADS (64 + 32 * TAB_EPI_WARPS)
#define TAB_SMEM (1024 + TAB_STAGES * TAB_STAGE_BYTES + TAB_EPI_WARPS * 4096)
#define TAB_DZ_BYTES (2ll << 30)                            // most memory for dz: beyond it the table goes in pieces
#define TAB_PARTS_BYTES (512ll << 20)                       // and for the tiles' partial sums: beyond it the queries do

template <int KIND> struct TabType;
template <> struct TabType<TAB_BF16> { using out = __nv_bfloat16; using elem = __nv_bfloat16; static constexpr int NPL = 1; static constexpr uint32_t FMT = 1; };
template <> struct TabType<TAB_F16> { using out = __half; using elem = __half; static constexpr int NPL = 1; static constexpr uint32_t FMT = 0; };
template <> struct TabType<TAB_F32> { using out = float; using elem = __half; static constexpr int NPL = 2; static constexpr uint32_t FMT = 0; };

// Powers of two that the operands were multiplied by, and their inverses; filled by tab_exponents_kernel.
struct TabScales { float q, w, dz, iq, iw, idz; unsigned max_q, max_w, max_g, unused; };

struct TabMaps { CUtensorMap a, b; };
struct TabArgs {
  long long M, N;                     // rows and columns of the product
  long long kblocks;                  // blocks of KB k-values
  int BN, splits, m_first;            // tile columns; parts of the contraction; the tiles of one column go to neighbouring CTAs
  float scale;
  const TabScales *sc;
  int *err;
  float4 *parts; int nparts;          // EPI_STATS: [M][nparts] (reference in base 2, S, T)
  const long long *targets; long long ignore_index, vocab, v0;         // EPI_DZ; v0: the table's row of column 0
  const float *lse, *entropy, *g, *h;
  void *dz; long long ldz, dz_plane;
  void *out; long long ldo;           // EPI_OUT: the result, or
  float *partial; int add;            //          [splits][M][N] fp32, stored or added
  float unscale_q, unscale_w, unscale_dz;                              // which inverses the product takes (1 or 0)
};

template <int EPI, int KIND, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(TAB_THREADS, 1) tab_kernel(const __grid_constant__ TabMaps maps, TabArgs g) {
  using Elem = typename TabType<KIND>::elem;
  using Out = typename TabType<KIND>::out;
  constexpr int NPL = TabType<KIND>::NPL, KB = NPL == 1 ? 64 : 32;
  constexpr uint32_t ROW_BYTES = KB * 2, ATOM_BYTES = KB * 128;          // a K-major row; 64 columns of an MN-major operand's plane
  constexpr uint32_t A_BYTES = NPL * 128 * ROW_BYTES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char *ostage = smem + TAB_STAGES * TAB_STAGE_BYTES;
  __shared__ __align__(8) unsigned long long bars[2 * TAB_STAGES + 4];
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(&bars[0]);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (TAB_STAGES + s); };
  auto accf_bar = [&](int a) { return bar0 + 8u * (2 * TAB_STAGES + a); };
  auto acce_bar = [&](int a) { return bar0 + 8u * (2 * TAB_STAGES + 2 + a); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * TAB_STAGES + 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar0 + 8u * i));
    for (int a = 0; a < 2; ++a) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(acce_bar(a)), "r"(32 * TAB_EPI_WARPS));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&tmem_base_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base_s;

  const long long tiles_m = (g.M + 127) / 128, tiles_n = (g.N + g.BN - 1) / g.BN, per_split = tiles_m * tiles_n, ntiles = per_split * g.splits;
  auto tile = [&](long long t, long long &m0, long long &n0, int &split, long long &kb0, long long &kb1) {
    split = (int)(t / per_split);
    t -= split * per_split;
    const long long m = g.m_first ? t % tiles_m : t / tiles_n, n = g.m_first ? t / tiles_m : t % tiles_n;
    m0 = m * 128;
    n0 = n * g.BN;
    kb0 = g.kblocks * split / g.splits;
    kb1 = g.kblocks * (split + 1) / g.splits;
  };
  const int b_atoms = g.BN / 64;
  const uint32_t b_plane = B_MN ? ATOM_BYTES : (uint32_t)g.BN * ROW_BYTES;
  const uint32_t stage_tx = A_BYTES + NPL * (uint32_t)g.BN * ROW_BYTES;

  if (warp == 0) {
    // ---------------- TMA: one box per K-major operand, one per 64 columns of an MN-major one, each from its own lane
    StageRing at;
    bool stop = false;
    constexpr int A_BOXES = A_MN ? 2 : 1;
    const int boxes = A_BOXES + (B_MN ? b_atoms : 1);
    for (long long t = blockIdx.x; t < ntiles && !stop; t += gridDim.x) {
      long long m0, n0, kb0, kb1;
      int split;
      tile(t, m0, n0, split, kb0, kb1);
      for (long long kb = kb0; kb < kb1; ++kb, at.next(TAB_STAGES)) {
        bool ok = failed == 0;
        if (ok && lane == 0) ok = mbar_wait(empty_bar(at.s), at.parity ^ 1u, g.err);
        if (!__all_sync(0xffffffffu, ok)) { failed = 1; stop = true; break; }
        const uint32_t fb = full_bar(at.s), a = smem_u32(smem) + (uint32_t)at.s * TAB_STAGE_BYTES, b = a + A_BYTES;
        if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(fb), "r"(stage_tx) : "memory");
        __syncwarp();
        const int k = (int)(kb * KB);
        if (lane < A_BOXES) {
          if (A_MN) tma_load_3d(a + lane * NPL * ATOM_BYTES, &maps.a, (int)m0 + 64 * lane, k, 0, fb);
          else tma_load_3d(a, &maps.a, k, (int)m0, 0, fb);
        } else if (lane < boxes) {
          const int j = lane - A_BOXES;
          if (B_MN) tma_load_3d(b + j * NPL * ATOM_BYTES, &maps.b, (int)n0 + 64 * j, k, 0, fb);
          else tma_load_3d(b, &maps.b, k, (int)n0, 0, fb);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- products.  D fp32; both operands of one type; planes (a, b): b1 b0, b0 b1, b0 b0
    const uint32_t idesc = (1u << 4) | (TabType<KIND>::FMT << 7) | (TabType<KIND>::FMT << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                           ((uint32_t)(g.BN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    // K-major: 128-byte rows in the 128-byte swizzle (layout 2) or 64-byte rows in the 64-byte one (layout 4), 32 bytes per 16 k-values;
    // MN-major: 64 columns x KB rows in the 128-byte swizzle, 2048 bytes per 16 k-values
    constexpr uint32_t K_SBO = KB == 64 ? 1024 : 512, K_LAYOUT = KB == 64 ? 2 : 4;
    constexpr uint32_t a_step = A_MN ? 2048 : 32, b_step = B_MN ? 2048 : 32, a_plane = A_MN ? ATOM_BYTES : 128 * ROW_BYTES;
    const bool leader = elect_one();
    StageRing at;
    int j = 0;
    for (long long t = blockIdx.x; t < ntiles; t += gridDim.x, ++j) {
      long long m0, n0, kb0, kb1;
      int split;
      tile(t, m0, n0, split, kb0, kb1);
      const int ab = j & 1;
      if (!__all_sync(0xffffffffu, failed == 0 && mbar_wait(acce_bar(ab), (uint32_t)((j >> 1) & 1) ^ 1u, g.err))) { failed = 1; break; }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + (uint32_t)ab * 256u;
      bool ok = true;
      for (long long kb = kb0; kb < kb1; ++kb, at.next(TAB_STAGES)) {
        if (!__all_sync(0xffffffffu, mbar_wait(full_bar(at.s), at.parity, g.err))) { failed = 1; ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t a = smem_u32(smem) + (uint32_t)at.s * TAB_STAGE_BYTES, b = a + A_BYTES;
        const uint64_t da = A_MN ? smem_desc(a, NPL * ATOM_BYTES, 1024, 2) : smem_desc(a, 0, K_SBO, K_LAYOUT);
        const uint64_t db = B_MN ? smem_desc(b, NPL * ATOM_BYTES, 1024, 2) : smem_desc(b, 0, K_SBO, K_LAYOUT);
#pragma unroll
        for (int k = 0; k < KB / 16; ++k) {
          if (NPL == 2 && leader) {
            mma_f16(acc, desc_at(da, a_plane + k * a_step), desc_at(db, k * b_step), idesc, kb > kb0 || k > 0);
            mma_f16(acc, desc_at(da, k * a_step), desc_at(db, b_plane + k * b_step), idesc, true);
          }
          if (leader) mma_f16(acc, desc_at(da, k * a_step), desc_at(db, k * b_step), idesc, NPL == 2 || kb > kb0 || k > 0);
        }
        if (leader) mma_commit(empty_bar(at.s));
      }
      if (!ok) break;
      if (leader) mma_commit(accf_bar(ab));
    }
  } else {
    // ---------------- epilogue
    const int q = warp & 3, half = (warp - 2) >> 2, hc = g.BN / 2;       // 32 rows of the tile; half of its columns
    unsigned char *buf = ostage + (size_t)(warp - 2) * 4096;
    const float unscale = (g.unscale_q != 0.f ? g.sc->iq : 1.f) * (g.unscale_w != 0.f ? g.sc->iw : 1.f) * (g.unscale_dz != 0.f ? g.sc->idz : 1.f);
    int j = 0;
    for (long long t = blockIdx.x; t < ntiles; t += gridDim.x, ++j) {
      long long m0, n0, kb0, kb1;
      int split;
      tile(t, m0, n0, split, kb0, kb1);
      const int ab = j & 1;
      const long long m = m0 + q * 32 + lane;
      // what a row of dz takes, read while the products run
      float lse = 0.f, H = 0.f, gg = 0.f, hh = 0.f;
      long long hot = -1;
      bool live = false;                                                 // neither padding nor without a target
      if (EPI == EPI_DZ && m < g.M) {
        const long long target = g.targets[m];
        if (target >= 0 && target < g.vocab && target != g.ignore_index) {
          const float up = g.scale * g.sc->dz;
          lse = g.lse[m];
          if (g.g) gg = g.g[m] * up;
          if (g.h) { hh = g.h[m] * up; H = g.entropy[m]; }
          hot = target - g.v0;
          live = true;
        } else if (target != g.ignore_index && n0 == 0 && half == 0 && g.v0 == 0) atomicOr(g.err, TOK_ERR_ID);
      }
      bool ok = failed == 0;
      if (ok && lane == 0) ok = mbar_wait(accf_bar(ab), (uint32_t)(j >> 1) & 1, g.err);
      if (!__all_sync(0xffffffffu, ok)) { failed = 1; break; }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + (uint32_t)ab * 256u + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * hc);
      const long long c0 = n0 + half * hc;                               // first column of this warp
      const int cols = c0 >= g.N ? 0 : g.N - c0 < hc ? (int)(g.N - c0) : hc;

      if (EPI == EPI_STATS) {
        const float c = g.scale * unscale * TOK_LOG2E;
        float mx = -INFINITY, r = 0.f, S = 0.f, T = 0.f;
        for (int x = 0; x < cols; x += 32) {
          uint32_t v[32];
          tmem_ld32(acc + x, v);
          if (cols - x < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) if (i >= cols - x) v[i] = __float_as_uint(-INFINITY);     // (columns that do not exist)
          }
          float cm = __uint_as_float(v[0]);
#pragma unroll
          for (int i = 1; i < 32; ++i) cm = fmaxf(cm, __uint_as_float(v[i]));
          if (cm > mx) {
            mx = cm;
            const float d = fminf(fmaxf(r - cm * c, -1e30f), 0.f), f = tok_ex2(d);
            T = (T + d * S) * f;
            S *= f;
            r = cm * c;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float y = tok_max_nan(fmaf(__uint_as_float(v[i]), c, -r), -1000.f), e = tok_ex2(y);
            S += e;
            T = fmaf(y, e, T);
          }
        }
        if (m < g.M) g.parts[m * g.nparts + n0 / g.BN * 2 + half] = make_float4(S == 0.f ? -1e30f : r, S, T, 0.f);
      } else if (EPI == EPI_DZ) {
        const float zs = g.scale * unscale;
        // the padding of the last columns is written too, as zeros: the contraction over the table's rows reads whole blocks
        const int span = c0 >= g.ldz ? 0 : g.ldz - c0 < hc ? (int)(g.ldz - c0) : hc;
        for (int x = 0; x < span; x += 64) {
          uint32_t pk[NPL][32];
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            uint32_t v[32];
            tmem_ld32(acc + x + part * 32, v);
            const long long col = c0 + x + part * 32;
            float d[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float logp = fmaf(__uint_as_float(v[i]), zs, -lse), p = tok_ex2(logp * TOK_LOG2E);
              d[i] = live && (p > 0.f || p != p) ? -p * fmaf(hh, logp + H, gg) : 0.f;
            }
            if (__any_sync(0xffffffffu, hot >= col && hot < col + 32)) {
#pragma unroll
              for (int i = 0; i < 32; ++i) if (hot == col + i) d[i] += gg;
            }
            if (col + 32 > g.N) {
#pragma unroll
              for (int i = 0; i < 32; ++i) if (col + i >= g.N) d[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              Elem e[2] = {Tok<Elem>::down(d[i]), Tok<Elem>::down(d[i + 1])};
              pk[0][part * 16 + i / 2] = *reinterpret_cast<uint32_t *>(e);
              if (NPL == 2) {
                Elem f[2] = {Tok<Elem>::down(d[i] - Tok<Elem>::up(e[0])), Tok<Elem>::down(d[i + 1] - Tok<Elem>::up(e[1]))};
                pk[NPL - 1][part * 16 + i / 2] = *reinterpret_cast<uint32_t *>(f);
              }
            }
          }
          // through shared memory: a row's 64 values leave as one line
#pragma unroll
          for (int pl = 0; pl < NPL; ++pl) {
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 8; ++u)
              *reinterpret_cast<uint4 *>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_uint4(pk[pl][4 * u], pk[pl][4 * u + 1], pk[pl][4 * u + 2], pk[pl][4 * u + 3]);
            __syncwarp();
            Elem *to = (Elem *)g.dz + pl * g.dz_plane + (m0 + q * 32) * g.ldz + c0 + x;
            const int rows = g.M - (m0 + q * 32) < 32 ? (int)(g.M - (m0 + q * 32)) : 32;
#pragma unroll 8
            for (int r = 0; r < rows; ++r)
              reinterpret_cast<uint32_t *>(to + r * g.ldz)[lane] = *reinterpret_cast<uint32_t *>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + ((lane & 3) << 2));
          }
        }
      } else {
        const int rows = g.M - (m0 + q * 32) < 32 ? (int)(g.M - (m0 + q * 32)) : 32;
        for (int x = 0; x < cols; x += 32) {
          uint32_t v[32];
          tmem_ld32(acc + x, v);
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4 *>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
          __syncwarp();
          const long long col = c0 + x + lane;
          if (x + lane < cols) {
#pragma unroll 8
            for (int r = 0; r < rows; ++r) {
              float val = *reinterpret_cast<float *>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + ((lane & 3) << 2)) * unscale;
              if (kb0 == kb1) val = 0.f;                                 // (a part without k-values: nothing was multiplied)
              const long long row = m0 + q * 32 + r;
              if (g.partial) {
                float *to = g.partial + ((long long)split * g.M + row) * g.N + col;
                *to = g.add ? *to + val : val;
              } else ((Out *)g.out)[row * g.ldo + col] = Tok<Out>::down(val);
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(acce_bar(ab)) : "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    // after a wait that ran out copies and products may still be in flight: a bounded grace before the tensor memory goes back
    if (failed) for (int i = 0; i < 200000; ++i) __nanosleep(20);
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
  }
}

// A query's partial sums to its statistics; the target's score is a dot product of its own, in fp32.
template <class T>
__global__ void __launch_bounds__(128) tab_stats_kernel(const T *__restrict__ queries, long long q_stride, const T *__restrict__ table, long long t_stride, long long vocab,
                                                        int dim, const long long *__restrict__ targets, long long ignore_index, float scale,
                                                        const float4 *__restrict__ parts, int nparts, float *logprob, float *entropy, float *lse, int *errors) {
  __shared__ float4 sums[4];
  const long long n = blockIdx.x, target = targets[n];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (target == ignore_index) {
    if (threadIdx.x == 0) { logprob[n] = 0.f; entropy[n] = 0.f; lse[n] = 0.f; }
    return;
  }
  const bool known = target >= 0 && target < vocab;
  float r = -1e30f, S = 0.f, A = 0.f, dot = 0.f;
  auto join = [&](float r2, float S2, float A2) {
    const float top = fmaxf(r, r2), d1 = r - top, d2 = r2 - top, f1 = tok_ex2(d1), f2 = tok_ex2(d2);
    A = (A + d1 * S) * f1 + (A2 + d2 * S2) * f2;
    S = S * f1 + S2 * f2;
    r = top;
  };
  for (int i = threadIdx.x; i < nparts; i += 128) { const float4 p = parts[n * nparts + i]; join(p.x, p.y, p.z); }
  if (known) {
    const T *a = queries + n * q_stride, *b = table + target * t_stride;
    for (int i = threadIdx.x; i < dim; i += 128) dot = fmaf(Tok<T>::up(a[i]), Tok<T>::up(b[i]), dot);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float r2 = __shfl_xor_sync(0xffffffffu, r, o), S2 = __shfl_xor_sync(0xffffffffu, S, o), A2 = __shfl_xor_sync(0xffffffffu, A, o);
    join(r2, S2, A2);
    dot += __shfl_xor_sync(0xffffffffu, dot, o);
  }
  if (lane == 0) sums[w] = make_float4(r, S, A, dot);
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 4; ++i) { join(sums[i].x, sums[i].y, sums[i].z); dot += sums[i].w; }
  const float log_s = logf(S), l = fmaf(r, TOK_LN2, log_s);
  lse[n] = l;
  entropy[n] = log_s - A * TOK_LN2 / S;
  logprob[n] = known ? dot * scale - l : __int_as_float(0x7fc00000);
  if (!known && errors) atomicOr(errors, TOK_ERR_ID);
}

// ---- preparation ---------------------------------------------------------------------------------------------
// Which rows count: those whose target is not ignore_index (any: nor outside of the table); without targets all.
struct TabRows {
  const long long *targets; long long ignore_index, vocab; int any;
  __device__ __forceinline__ bool operator()(long long r) const {
    if (!targets) return true;
    const long long t = targets[r];
    return t != ignore_index && (any || (t >= 0 && t < vocab));
  }
};
// Largest finite |x| of a matrix, as its bits.
__global__ void __launch_bounds__(256) tab_absmax_kernel(const float *__restrict__ x, long long stride, long long rows, int dim, TabRows counts, unsigned *out) {
  unsigned top = 0u;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x)
    if (counts(r)) for (int i = threadIdx.x; i < dim; i += 256) {
      const unsigned b = __float_as_uint(x[r * stride + i]) & 0x7fffffffu;
      if (b < 0x7f800000u && b > top) top = b;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0 && top) atomicMax(out, top);
}
// Bound of |dz| / scale: |g| + |h| (p |log p| + p H), p |log p| <= 1 / e, H <= log vocab < 22.
__global__ void __launch_bounds__(256) tab_gradmax_kernel(const float *__restrict__ g, const float *__restrict__ h, long long n, TabRows counts, unsigned *out) {
  unsigned top = 0u;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    if (!counts(i)) continue;
    const float v = (g ? fabsf(g[i]) : 0.f) + (h ? 23.f * fabsf(h[i]) : 0.f);
    const unsigned b = __float_as_uint(v);
    if (b < 0x7f800000u && b > top) top = b;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0 && top) atomicMax(out, top);
}
// 2^k that brings a number below 2^top, -100 <= k <= 100
__device__ __forceinline__ float tab_power(unsigned bits, int top, float &inverse) {
  int k = bits ? top - ((int)(bits >> 23) - 126) : 0;
  k = k < -100 ? -100 : k > 100 ? 100 : k;
  inverse = __uint_as_float((unsigned)(127 - k) << 23);
  return __uint_as_float((unsigned)(127 + k) << 23);
}
__global__ void tab_exponents_kernel(TabScales *sc, float scale, int planes, int dz) {
  sc->q = sc->w = sc->dz = sc->iq = sc->iw = sc->idz = 1.f;
  if (planes) { sc->q = tab_power(sc->max_q, 14, sc->iq); sc->w = tab_power(sc->max_w, 14, sc->iw); }
  if (dz) sc->dz = tab_power(__float_as_uint(fminf(__uint_as_float(sc->max_g) * scale, 1e38f)), 14, sc->idz);
}
// fp32 to two fp16 planes; 16-bit elements as they are.  Rows that do not count become zeros: whatever stands in padding, a
// product with its zero gradient is zero.
template <class T>
__global__ void __launch_bounds__(256) tab_pack_kernel(const T *__restrict__ x, long long stride, long long rows, int dim, TabRows counts, void *to, long long ld, long long plane,
                                                       const float *power) {
  const float up = sizeof(T) == 4 ? *power : 1.f;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const bool keep = counts(r);
    for (int i = threadIdx.x; i < dim; i += 256) {
      const T e = keep ? x[r * stride + i] : Tok<T>::down(0.f);
      if (sizeof(T) == 4) {
        const float v = Tok<T>::up(e) * up;
        const __half b0 = __float2half_rn(v), b1 = __float2half_rn(v - __half2float(b0));
        ((__half *)to)[r * ld + i] = b0;
        ((__half *)to)[plane + r * ld + i] = __hisinf(b0) || __hisnan(b0) ? __float2half_rn(0.f) : b1;
      } else ((T *)to)[r * ld + i] = e;
    }
  }
}
// The parts of a split contraction, added in their order.
template <class T>
__global__ void __launch_bounds__(256) tab_join_kernel(const float *__restrict__ partial, int splits, long long count, T *__restrict__ out) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) {
    float s = partial[i];
    for (int k = 1; k < splits; ++k) s += partial[k * count + i];
    out[i] = Tok<T>::down(s);
  }
}

// ---- host --------------------------------------------------------------------------------------------------
struct TabOperand { const void *base; long long rows, inner, ld, plane; };   // [planes][rows][ld], 16-bit elements

static bool tab_encode(CUtensorMap *tm, int kind, const TabOperand &o, int box_inner, int box_rows) {
  const int npl = kind == TAB_F32 ? 2 : 1;
  const cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.rows, (cuuint64_t)npl};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(npl > 1 ? o.plane : o.ld * 8) * 2};
  const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, (cuuint32_t)npl};
  return encode_map(tm, kind == TAB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, o.base, 3, dims, strides, box,
                    box_inner == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int EPI, int KIND, bool A_MN, bool B_MN>
static bool tab_launch(const TabOperand &a, const TabOperand &b, const TabArgs &g, cudaStream_t st) {
  constexpr int KB = KIND == TAB_F32 ? 32 : 64;
  if (pbg_launch_failed()) return true;
  TabMaps maps;
  if (!tab_encode(&maps.a, KIND, a, A_MN ? 64 : KB, A_MN ? KB : 128) || !tab_encode(&maps.b, KIND, b, B_MN ? 64 : KB, B_MN ? KB : g.BN)) return false;
  void (*kernel)(TabMaps, TabArgs) = tab_kernel<EPI, KIND, A_MN, B_MN>;
  pbg_opt_in_smem((const void *)kernel, TAB_SMEM);
  const long long tiles = (g.M + 127) / 128 * ((g.N + g.BN - 1) / g.BN) * g.splits, sms = pbg_sm_count();
  pbg_launch_in_order(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), TAB_THREADS, TAB_SMEM, st, maps, g);
  return true;
}

// Tile columns: the fewest columns for the SM with the most of them, with what a tile costs beside them.
static int tab_columns(long long tiles_m, long long N, int step) {
  const long long sms = pbg_sm_count();
  int best = 256;
  long long cost = -1;
  for (int bn = 256; bn >= step; bn -= step) {
    const long long tiles = tiles_m * ((N + bn - 1) / bn), c = (tiles + sms - 1) / sms * (bn + 16);
    if (cost < 0 || c < cost) { cost = c; best = bn; }
  }
  return best;
}

static int tab_kind(int dtype) { return dtype == PBG_F32 ? TAB_F32 : dtype == PBG_BF16 ? TAB_BF16 : TAB_F16; }
// TMA reads rows where they lie if they start on 16-byte boundaries
static bool tab_packed(const void *p, long long stride, int dim, int dtype) { return dtype == PBG_F32 || !aligned16(p) || stride % 8 != 0 || stride < dim; }

// What the workspace holds.  Its size is asked for without addresses, so it has room for packed operands wherever they may be needed.
struct TabPlace {
  int64_t scales, q, w, parts, dz, partial, bytes;
  long long ld, columns, ldz;         // packed rows' length; table rows per piece of dz, and its rows' length
  long long piece;                    // queries per pass of the forward
  int npl, bn, nparts, splits;
};
static TabPlace tab_place(long long n, long long rows, int dim, int dtype, bool grad) {
  TabPlace p;
  p.npl = dtype == PBG_F32 ? 2 : 1;
  p.ld = tok_up(dim, 8);
  p.scales = 0;
  p.q = 256;
  p.w = p.q + tok_up(n * p.ld * 2 * p.npl, 256);
  int64_t at = p.w + tok_up(rows * p.ld * 2 * p.npl, 256);
  p.parts = p.dz = p.partial = at;
  p.columns = p.ldz = 0;
  p.piece = n;
  p.bn = p.nparts = p.splits = 0;
  if (!grad) {
    p.bn = tab_columns((n + 127) / 128, rows, 64);
    p.nparts = (int)((rows + p.bn - 1) / p.bn * 2);
    long long most = TAB_PARTS_BYTES / (16ll * p.nparts) / 128 * 128;
    if (most < 128) most = 128;
    if (p.piece > most) p.piece = most;
    at += p.piece * p.nparts * 16;
  } else {
    long long most = TAB_DZ_BYTES / (2 * p.npl * n) / 256 * 256;
    if (most < 256) most = 256;
    p.columns = rows < most ? rows : most;
    p.ldz = tok_up(p.columns, 64);
    at += tok_up(n * p.ldz * 2 * p.npl, 256);
    p.partial = at;
    const long long tiles = (n + 127) / 128 * ((dim + 255) / 256), blocks = (p.columns + 63) / 64;
    long long s = pbg_sm_count() / tiles;
    if (s > blocks / 8) s = blocks / 8;
    p.splits = (int)(s < 1 ? 1 : s);
    if (p.splits > 1 || p.columns < rows) at += tok_up((int64_t)p.splits * n * dim * 4, 256);
  }
  p.bytes = at;
  return p;
}

struct TabCall {
  const void *queries; int64_t q_stride, n; const void *table; int64_t t_stride, rows; int dim, dtype;
  const long long *targets; int64_t ignore_index; float scale; unsigned char *ws; int *errors; cudaStream_t st;
  TabScales *sc; int *err;
  TabOperand q, w;
};

static unsigned tab_grid(long long rows) { return (unsigned)(rows < 4096 ? rows : 4096); }
template <class T>
static void tab_pack(const TabCall &c, const void *x, long long stride, long long rows, bool always, const TabRows &counts, unsigned char *to, const TabPlace &p, const float *power,
                     TabOperand &o) {
  o = TabOperand{x, rows, c.dim, stride, 0};
  if (!always && !tab_packed(x, stride, c.dim, c.dtype)) return;
  o = TabOperand{to, rows, c.dim, p.ld, rows * p.ld};
  pbg_launch_in_order(tab_pack_kernel<T>, dim3(tab_grid(rows)), 256, 0, c.st, (const T *)x, (long long)stride, rows, c.dim, counts, (void *)to, p.ld, o.plane, power);
}
// Scales and operands.  For the gradient the queries are always copied: the rows that do not count have to be zeros.
template <class T>
static void tab_prepare(TabCall &c, const TabPlace &p, bool grad, const float *g, const float *h) {
  c.sc = (TabScales *)(c.ws + p.scales);
  c.err = c.errors ? c.errors : (int *)(c.ws + p.scales + 128);
  if (cudaMemsetAsync(c.ws, 0, 256, c.st) != cudaSuccess) pbg_note_launch();
  const TabRows counts{c.targets, c.ignore_index, c.rows, grad ? 0 : 1}, all{nullptr, 0, 0, 1};
  const bool planes = c.dtype == PBG_F32, dz = grad && c.dtype != PBG_BF16;
  if (planes) {
    pbg_launch_in_order(tab_absmax_kernel, dim3(tab_grid(c.n)), 256, 0, c.st, (const float *)c.queries, (long long)c.q_stride, (long long)c.n, c.dim, counts, &c.sc->max_q);
    pbg_launch_in_order(tab_absmax_kernel, dim3(tab_grid(c.rows)), 256, 0, c.st, (const float *)c.table, (long long)c.t_stride, (long long)c.rows, c.dim, all, &c.sc->max_w);
  }
  if (dz) pbg_launch_in_order(tab_gradmax_kernel, dim3(tab_grid((c.n + 255) / 256)), 256, 0, c.st, g, h, (long long)c.n, counts, &c.sc->max_g);
  pbg_launch_in_order(tab_exponents_kernel, dim3(1), 1, 0, c.st, c.sc, c.scale, (int)planes, (int)dz);
  tab_pack<T>(c, c.queries, c.q_stride, c.n, grad, counts, c.ws + p.q, p, &c.sc->q, c.q);
  tab_pack<T>(c, c.table, c.t_stride, c.rows, false, all, c.ws + p.w, p, &c.sc->w, c.w);
}

struct TabForward { TabCall c; TabPlace p; float *logprob, *entropy, *lse; bool ok; };
template <class T, int KIND>
static void tab_forward(TabForward &f) {
  TabCall &c = f.c;
  tab_prepare<T>(c, f.p, false, nullptr, nullptr);
  for (long long n0 = 0; n0 < c.n && f.ok; n0 += f.p.piece) {
    const long long n = c.n - n0 < f.p.piece ? c.n - n0 : f.p.piece;
    TabOperand q = c.q;
    q.base = (const char *)q.base + n0 * q.ld * 2;
    q.rows = n;
    TabArgs g = {};
    g.M = n; g.N = c.rows; g.kblocks = (c.dim + (KIND == TAB_F32 ? 31 : 63)) / (KIND == TAB_F32 ? 32 : 64);
    g.BN = f.p.bn;
    g.splits = 1; g.m_first = 1; g.scale = c.scale; g.sc = c.sc; g.err = c.err;
    g.unscale_q = g.unscale_w = 1.f;
    g.parts = (float4 *)(c.ws + f.p.parts); g.nparts = f.p.nparts;
    f.ok = tab_launch<EPI_STATS, KIND, false, false>(q, c.w, g, c.st);
    pbg_launch_in_order(tab_stats_kernel<T>, dim3((unsigned)n), 128, 0, c.st, (const T *)c.queries + n0 * c.q_stride, (long long)c.q_stride, (const T *)c.table, (long long)c.t_stride,
                        (long long)c.rows, c.dim, c.targets + n0, (long long)c.ignore_index, c.scale, (const float4 *)g.parts, g.nparts, f.logprob + n0, f.entropy + n0, f.lse + n0, c.errors);
  }
}

struct TabBackward { TabCall c; TabPlace p; const float *lse, *entropy, *g, *h; void *dq, *dt; bool ok; };
template <class T, int KIND>
static void tab_backward(TabBackward &f) {
  TabCall &c = f.c;
  constexpr int KB = KIND == TAB_F32 ? 32 : 64;
  tab_prepare<T>(c, f.p, true, f.g, f.h);
  const long long tiles_m = (c.n + 127) / 128;
  const bool partial = f.p.splits > 1 || f.p.columns < c.rows;
  for (long long v0 = 0; v0 < c.rows && f.ok; v0 += f.p.columns) {
    const long long cols = c.rows - v0 < f.p.columns ? c.rows - v0 : f.p.columns;
    TabOperand w = c.w;
    w.base = (const char *)w.base + v0 * w.ld * 2;
    w.rows = cols;
    TabArgs g = {};
    g.M = c.n; g.N = cols; g.kblocks = (c.dim + KB - 1) / KB; g.BN = tab_columns(tiles_m, cols, 128);
    g.splits = 1; g.m_first = 1; g.scale = c.scale; g.sc = c.sc; g.err = c.err;
    g.unscale_q = g.unscale_w = 1.f;
    g.targets = c.targets; g.ignore_index = c.ignore_index; g.vocab = c.rows; g.v0 = v0;
    g.lse = f.lse; g.entropy = f.entropy; g.g = f.g; g.h = f.h;
    g.dz = c.ws + f.p.dz; g.ldz = f.p.ldz; g.dz_plane = c.n * f.p.ldz;
    f.ok = tab_launch<EPI_DZ, KIND, false, false>(c.q, w, g, c.st);
    const TabOperand dz{g.dz, c.n, cols, f.p.ldz, g.dz_plane};
    if (f.dq && f.ok) {
      TabArgs d = {};
      d.M = c.n; d.N = c.dim; d.kblocks = (cols + KB - 1) / KB; d.BN = tab_columns(tiles_m * f.p.splits, c.dim, 64);
      d.splits = f.p.splits; d.scale = 1.f; d.sc = c.sc; d.err = c.err;
      d.unscale_dz = d.unscale_w = 1.f;
      d.out = f.dq; d.ldo = c.dim;
      if (partial) { d.partial = (float *)(c.ws + f.p.partial); d.add = v0 > 0; }
      f.ok = tab_launch<EPI_OUT, KIND, false, true>(dz, w, d, c.st);
    }
    if (f.dt && f.ok) {
      TabArgs d = {};
      d.M = cols; d.N = c.dim; d.kblocks = (c.n + KB - 1) / KB; d.BN = tab_columns((cols + 127) / 128, c.dim, 64);
      d.splits = 1; d.scale = 1.f; d.sc = c.sc; d.err = c.err;
      d.unscale_dz = d.unscale_q = 1.f;
      d.out = (T *)f.dt + v0 * c.dim; d.ldo = c.dim;
      f.ok = tab_launch<EPI_OUT, KIND, true, true>(dz, c.q, d, c.st);
    }
  }
  if (f.dq && partial && f.ok) {
    const long long count = c.n * c.dim, blocks = (count + 255) / 256;
    pbg_launch_in_order(tab_join_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), 256, 0, c.st, (const float *)(c.ws + f.p.partial), f.p.splits, count, (T *)f.dq);
  }
}

static int tab_check(const TabCall &c, int64_t bytes, bool grad) {
  if (c.n < 0 || c.rows <= 0 || c.dim <= 0 || c.q_stride < 0 || c.t_stride < 0 || !tok_type(c.dtype) || !tok_scale(c.scale)) return PBG_ERR_BAD_ARGUMENT;
  if (c.dim > 65536 || c.n > (1ll << 30) || c.rows > 0x7fffffffll - 65536) return PBG_ERR_TOO_LARGE;
  if (c.n == 0) return PBG_OK;
  if (!c.queries || !c.table || !c.targets || !c.ws || ((uintptr_t)c.ws & 255) || bytes < tab_place(c.n, c.rows, c.dim, c.dtype, grad).bytes) return PBG_ERR_BAD_ARGUMENT;
  // rows that TMA reads where they lie are less than 2^40 bytes apart
  if (c.q_stride >= (1ll << 38) || c.t_stride >= (1ll << 38)) return PBG_ERR_TOO_LARGE;
  return PBG_OK;
}

extern "C" int64_t pbg_table_logprobs_workspace(int64_t n, int64_t rows, int32_t dim, int32_t dtype, int32_t grad) {
  if (n <= 0 || rows <= 0 || dim <= 0 || !tok_type(dtype) || n > (1ll << 30) || rows > 0x7fffffffll) return 0;
  return tab_place(n, rows, dim, dtype, grad != 0).bytes;
}

extern "C" int pbg_table_logprobs(const void *queries, int64_t q_stride, int64_t n, const void *table, int64_t t_stride, int64_t rows, int32_t dim, int32_t dtype,
                                  const int64_t *targets, int64_t ignore_index, float scale, float *logprob, float *entropy, float *lse, void *workspace,
                                  int64_t workspace_bytes, int32_t *errors, void *stream) {
  TabForward f{{queries, q_stride, n, table, t_stride, rows, dim, dtype, (const long long *)targets, ignore_index, scale, (unsigned char *)workspace, errors, (cudaStream_t)stream},
               {}, logprob, entropy, lse, true};
  const int rc = tab_check(f.c, workspace_bytes, false);
  if (rc != PBG_OK || n == 0) return rc;
  if (!logprob || !entropy || !lse) return PBG_ERR_BAD_ARGUMENT;
  if (!get_encode()) return PBG_ERR_CUDA;
  pbg_launch_error() = cudaSuccess;
  f.p = tab_place(n, rows, dim, dtype, false);
  if (dtype == PBG_F32) tab_forward<float, TAB_F32>(f);
  else if (dtype == PBG_BF16) tab_forward<__nv_bfloat16, TAB_BF16>(f);
  else tab_forward<__half, TAB_F16>(f);
  const int status = tok_status();
  return f.ok ? status : PBG_ERR_CUDA;
}

extern "C" int pbg_table_logprobs_grad(const void *queries, int64_t q_stride, int64_t n, const void *table, int64_t t_stride, int64_t rows, int32_t dim, int32_t dtype,
                                       const int64_t *targets, int64_t ignore_index, float scale, const float *lse, const float *entropy, const float *grad_logprob,
                                       const float *grad_entropy, void *grad_queries, void *grad_table, void *workspace, int64_t workspace_bytes, int32_t *errors, void *stream) {
  TabBackward f{{queries, q_stride, n, table, t_stride, rows, dim, dtype, (const long long *)targets, ignore_index, scale, (unsigned char *)workspace, errors, (cudaStream_t)stream},
                {}, lse, entropy, grad_logprob, grad_entropy, grad_queries, grad_table, true};
  const int rc = tab_check(f.c, workspace_bytes, true);
  if (rc != PBG_OK) return rc;
  pbg_launch_error() = cudaSuccess;
  if (n == 0) {
    if (grad_table && cudaMemsetAsync(grad_table, 0, (size_t)rows * dim * tok_size(dtype), f.c.st) != cudaSuccess) pbg_note_launch();
    return tok_status();
  }
  if (!lse || (grad_entropy && !entropy) || (!grad_queries && !grad_table)) return PBG_ERR_BAD_ARGUMENT;
  if (!get_encode()) return PBG_ERR_CUDA;
  f.p = tab_place(n, rows, dim, dtype, true);
  if (dtype == PBG_F32) tab_backward<float, TAB_F32>(f);
  else if (dtype == PBG_BF16) tab_backward<__nv_bfloat16, TAB_BF16>(f);
  else tab_backward<__half, TAB_F16>(f);
  const int status = tok_status();
  return f.ok ? status : PBG_ERR_CUDA;
}
