// Log probabilities over all rows of a table, and their gradients: z = s Q W^T is never stored.
//
//   forward   per query: lse, entropy and log probability of the target          2 N V D operations, Q and W read
//   gradient  dz = s (g ([v = t] - p) - h p (log p + H));  dQ = dz W,  dW = dz^T Q   6 N V D operations (the scores once more)
//
// All products run on the tensor cores (tcgen05, kind::f16) with fp32 accumulators in tensor memory:
//   bf16, fp16   the tensors themselves are the operands, read by TMA where they lie; dz is kept in two planes of the operands' type, or
//                rounded to it (tab_place).  That of fp16 is scaled by a power of two so that its bound, known from g and h, lies below 2^14:
//                what is cut off below fp16's smallest step is 2^-39 of the bound, and results in fp16 end at 2^-25
//   fp32         scores: every operand as two fp16 planes, x 2^k = b0 + b1 (22 bits; k from the largest finite element of its row, so
//                that the planes of everything down to 2^-17 of it are whole), and the three products b1 b0 + b0 b1 + b0 b0: the dropped
//                b1 b1 is 2^-22 of a product, the size of fp32 rounding.  The powers leave the scores as factors of a row and of a column;
//                one k for a whole matrix would let one large row take the bits of all others.
//                Products with dz: three bf16 planes (24 bits) and six products.  Their sums run over the table's rows or over the
//                queries, whose powers are no factors of them, and dz spans more binades than fp16 has: bf16 has fp32's range, so that
//                elements, rows of dz with a small g and columns that no query comes near keep their bits down to 2^-150 of the largest.
//
// One persistent kernel per product, one CTA per SM, tiles of 128 x BN (BN <= 256) or, by a pair of CTAs, 256 x BN:
//   warp 0     TMA into a ring of stages (64 k-values of one plane, or 32 of two or three)
//   warp 1     issues tcgen05.mma into one of two accumulators of 256 columns
//   warps 2-9  read the other accumulator, two warps to every 32 rows: reduce it to (maximum, S, T) per row; or turn it into
//              dz and write that; or write the product
// A pair (cta_group::2): each CTA holds 128 rows of A and half of B's columns, the first one issues for both, and an operand byte
// in shared memory feeds twice as many products.  Alone, a tile of 128 x 256 writes and reads 192 bytes of shared memory per cycle of
// its products where the SM moves 128; a pair 128.
//
// What the loop waits for was found by leaving out the loads, then the products: a stage of four products (512 cycles) took 890 with loads
// alone, whatever its bytes, because of a cluster-wide acquire in front of every stage and of loads issued from several lanes.
// 4096 x 16,384 x 2048 bf16 (ncu): dz 227 us, dQ 354 and dW 330 with the tensor pipe active 61, 81 (the last round of tiles is half empty)
// and 90 % of the time; 4099 x 65,536 x 2048, a call: 4.3 ms, 1.28 PFLOP/s with both planes of dz counted, as the power allows.  fp32, 5000 x
// 14,951 x 400: dz 199 us, dQ 304, dW 331 (six products, 512 columns for 400).  7 queries x 131,072 x 2048 bf16: 98 us, 68 % of DRAM's peak.
//
// Up to sixteen fp32 queries take no tensor cores: making planes of the table reads and writes it three times over, where fp32 products
// on the CUDA cores keep up with one reading of it (tab_few_kernel).
//
// Every wait is bounded: one that runs out sets 2 in the error word, the CTA's products stop, and whatever it had still to
// write is NaN -- partial sums, dz or results, so that all results that depend on them are NaN too; then it frees its tensor memory
// and returns.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "pbg_tc.cuh"
#include "pbg_tokens.cuh"

enum { EPI_STATS = 0, EPI_DZ = 1, EPI_OUT = 2 };

#define TAB_STAGES_MAX 6
#define TAB_DZ_BYTES (2ll << 30)                            // most memory for dz: beyond it the table goes in pieces
#define TAB_PARTS_BYTES (512ll << 20)                       // and for the tiles' partial sums: beyond it the queries do
#define TAB_SPLIT_BYTES (512ll << 20)                       // and for the parts of dQ
// The tensor cores cut off what they add up instead of rounding it, a bias of half a step (2^-25 of the sum) per instruction and, of
// products that reach below the sum's last bit, for each of its 16.  Scores and fp32 results are therefore added up in parts, which
// are added in registers: blocks of k-values per part, 18 instructions for scores of fp32 operands, 32 for those of 16-bit operands, 24 for
// the products with fp32 dz.  Scores of 2048 terms of one sign are 3e-7 off (fp32), 5e-7 (bf16) and 1.6e-6 (fp16, whose products are the
// longest), in one piece 7e-7 with 36 instructions a part, 3e-6 and 7e-6; of both signs 1 to 2e-7.  The forward pass and the gradient cut the
// scores alike, so that what is cut off is the same in z and in lse, and the p of a row add up to 1.  Both sides: with 36
// instructions a part 4096 x 65,536 x 1024 fp32 take 7 % less time; in one piece 7 x 131,072 x 2048 bf16 take 91 us instead of 99,
// 4099 x 65,536 x 2048 700 instead of 780.  Products of 5000 fp32 terms with dz were 3.9e-5 off in one piece.
// 16-bit gradients are cut up too where half a step per addition comes near the result's own: 2^21 terms of one sign in one piece
// were 1 % off; a part of TAB_PART_LONG blocks is 2^-13 off at most.
#define TAB_PART_F32 3
#define TAB_PART_F32_OUT 2
#define TAB_PART_16 8
#define TAB_PART_LONG 512

// Eight warps share a tile's columns (two to every 32 rows), each with 4 KB of shared memory to write from; the ring of stages has the
// rest.  (Sixteen warps with half the columns each had registers for half of what they need and were slower.)
#define TAB_EPI_WARPS 8
#define TAB_THREADS (64 + 32 * TAB_EPI_WARPS)
#define TAB_SMEM 230400
// (planes of dz take 4 KB each, and the factors of each warp's 128 columns stand behind them all)
template <int EPI, class MATH> struct TabSmem {
  static constexpr bool DZ3 = EPI == EPI_DZ && MATH::NPB == 2;
  static constexpr int OUT = DZ3 ? 12288 : EPI == EPI_DZ ? 8192 : 4096, RING = TAB_SMEM - 1024 - TAB_EPI_WARPS * (OUT + (DZ3 ? 512 : 0));
};

// Operands: their elements, the planes of A and B, the type of results
template <class E, class O, int PA, int PB, class DZ = E> struct TabMath { using elem = E; using out = O; using dz = DZ; static constexpr int NPA = PA, NPB = PB; };
using TabBf16 = TabMath<__nv_bfloat16, __nv_bfloat16, 1, 1>;
using TabF16 = TabMath<__half, __half, 1, 1>;
using TabF32 = TabMath<__half, float, 2, 2, __nv_bfloat16>;               // scores, whose dz has three bf16 planes
using TabF32Out = TabMath<__nv_bfloat16, float, 3, 3>;
using TabBf16Fine = TabMath<__nv_bfloat16, __nv_bfloat16, 2, 1>;          // dz in two planes
using TabF16Fine = TabMath<__half, __half, 2, 1>;

// Powers of two that the operands were multiplied by, and their inverses: fp32 operands and their dz, to below 2^40 (products of two and
// sums of 2^31 of them stay in fp32); dz of fp16 operands, to below 2^14
struct TabScales { float q, w, dz, iq, iw, idz; };

struct TabMaps { CUtensorMap a, b, c; };                              // operands; what is written by bulk stores
struct TabArgs {
  long long M, N;                     // rows and columns of the product
  int kblocks;                        // blocks of KB k-values
  int BN, splits, m_first;            // tile columns; parts of the contraction; the tiles of one column go to neighbouring CTAs
  int stages, part;                   // stages of the ring; k-blocks added up in tensor memory at a time
  float scale;
  const float *row_f, *col_f;         // scores of fp32 operands: what takes a product to a score in base 2, by row and by column
  const TabScales *sc;                // null: all 1
  int *err;
  float4 *parts; int nparts;          // EPI_STATS: [M][nparts] (the members of Soft)
  float *at_target;                   //            [M] the target's product, as it stands in S
  const long long *targets; long long ignore_index, vocab, v0;         // v0: the table's row of column 0
  const float *lse, *entropy, *g, *h;
  long long ldz; int dz_planes;
  void *out; long long ldo;           // EPI_DZ: dz; EPI_OUT: the result, or
  float *partial; int add;            //          [splits][M][N] fp32, stored or added
  int bulk;                           //          either way by bulk stores
  int by_q;                           // EPI_OUT: the other operand is the queries
  int a_rows;                         // rows of A that are loaded: 128, or fewer where there is one row tile and nothing to fill it with
  int b_whole;                        // MN-major B: its rows are whole blocks of 64 columns, read as one box
  int wait_limit;                     // how often a wait asks before it gives up
};

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
// the address of the pair's first CTA that corresponds to an address of this one
__device__ __forceinline__ uint32_t in_first_cta(uint32_t a) { uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a)); return r; }
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
template <int CG>
__device__ __forceinline__ void tab_load(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
  if (CG == 1) tma_load_3d(dst, map, c0, c1, 0, bar);
  else asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                    :: "r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(0), "r"(bar) : "memory");
}
// blocks of 64 columns: (0, k row, 0, block)
template <int CG>
__device__ __forceinline__ void tab_load_blocks(uint32_t dst, const CUtensorMap *map, int k, int block, uint32_t bar) {
  if (CG == 1) tma_load_4d(dst, map, 0, k, 0, block, bar);
  else asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                    :: "r"(dst), "l"(map), "r"(0), "r"(k), "r"(0), "r"(block), "r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tab_mma(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if (CG == 1) mma_f16(acc, a, b, idesc, add);
  else asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" :: "r"(acc), "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u) : "memory");
}
// arrives on the barrier (the pair's two) when the products issued so far are done
template <int CG>
__device__ __forceinline__ void tab_commit(uint32_t bar) {
  if (CG == 1) mma_commit(bar);
  else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" :: "r"(bar), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ bool tab_wait(uint32_t bar, uint32_t parity, const TabArgs &g) {
  for (int it = 0; it < g.wait_limit; ++it) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
  }
  atomicOr(g.err, TOK_ERR_TIMEOUT);
  return false;
}
template <int EPI, class MATH, bool A_MN, bool B_MN, int CG, bool PARTS>        // PARTS: the contraction is added up in registers
__global__ void __launch_bounds__(TAB_THREADS, 1) tab_kernel(const __grid_constant__ TabMaps maps, TabArgs g) {
  using Elem = typename MATH::elem;
  using Out = typename MATH::out;
  using Dz = typename MATH::dz;
  constexpr int NPA = MATH::NPA, NPB = MATH::NPB, KB = NPA == 1 ? 64 : 32;
  constexpr uint32_t FMT = std::is_same<Elem, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t ROW_BYTES = KB * 2, ATOM_BYTES = KB * 128;          // a K-major row; 64 columns of an MN-major operand's plane
  constexpr uint32_t A_BYTES = NPA * 128 * ROW_BYTES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = (unsigned char *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char *ostage = smem + TabSmem<EPI, MATH>::RING;
  __shared__ __align__(8) unsigned long long bars[2 * TAB_STAGES_MAX + 4];
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cta_rank() : 0u;
  const uint32_t bar0 = smem_u32(&bars[0]);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (TAB_STAGES_MAX + s); };
  auto accf_bar = [&](int a) { return bar0 + 8u * (2 * TAB_STAGES_MAX + a); };
  auto acce_bar = [&](int a) { return bar0 + 8u * (2 * TAB_STAGES_MAX + 2 + a); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * TAB_STAGES_MAX + 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar0 + 8u * i));
    for (int a = 0; a < 2; ++a) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(acce_bar(a)), "r"(TAB_EPI_WARPS * CG));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
  }
  if (warp == 1) {
    if (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&tmem_base_s)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_u32(&tmem_base_s)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG == 2) pair_sync();                                              // the other CTA's barriers are set up too
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base_s;
  pdl_begin();

  const long long tiles_m = (g.M + 128 * CG - 1) / (128 * CG), tiles_n = (g.N + g.BN - 1) / g.BN, per_split = tiles_m * tiles_n, ntiles = per_split * g.splits;
  const long long first = blockIdx.x / CG, step = gridDim.x / CG;
  // m0: this CTA's rows; n0: the tile's columns
  auto tile = [&](long long t, long long &m0, long long &n0, int &split, int &kb0, int &kb1) {
    split = (int)(t / per_split);
    t -= split * per_split;
    const long long m = g.m_first ? t % tiles_m : t / tiles_n, n = g.m_first ? t / tiles_m : t % tiles_n;
    m0 = m * 128 * CG + 128 * rank;
    n0 = n * g.BN;
    kb0 = (int)((long long)g.kblocks * split / g.splits);
    kb1 = (int)((long long)g.kblocks * (split + 1) / g.splits);
  };
  const int b_cols = g.BN / CG;                                          // columns of B in this CTA
  const uint32_t b_plane = B_MN ? ATOM_BYTES : (uint32_t)b_cols * ROW_BYTES;
  const uint32_t stage_bytes = A_BYTES + NPB * (uint32_t)b_cols * ROW_BYTES;
  const uint32_t a_plane = A_MN ? ATOM_BYTES : (uint32_t)g.a_rows * ROW_BYTES;

  if (warp == 0) {
    // ---------------- TMA: one box per operand, or one per 64 columns of an MN-major one.  One thread does it all: a stage takes
    // it 294 cycles with two boxes.  One lane that waits, a vote, and a box from each of two lanes took 560, which is more than the
    // stage's products (512).
    if (lane == 0) {
      StageRing at;
      bool ok = true;
      for (long long t = first; t < ntiles && ok; t += step) {
        long long m0, n0;
        int split, kb0, kb1;
        tile(t, m0, n0, split, kb0, kb1);
        n0 += rank * b_cols;
        ok = failed == 0;
        for (int kb = kb0; kb < kb1 && ok; ++kb, at.next(g.stages)) {
          ok = tab_wait(empty_bar(at.s), at.parity ^ 1u, g);
          if (!ok) { failed = 1; break; }
          const uint32_t a = smem_u32(smem) + (uint32_t)at.s * stage_bytes, b = a + A_BYTES;
          // a pair's loads are all counted by the first CTA, which issues the products
          const uint32_t fb = CG == 1 ? full_bar(at.s) : in_first_cta(full_bar(at.s));
          if (rank == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(full_bar(at.s)), "r"(CG * (stage_bytes - NPA * (128 - (uint32_t)g.a_rows) * ROW_BYTES)) : "memory");
          const int k = kb * KB;
          if (A_MN) tab_load_blocks<CG>(a, &maps.a, k, (int)(m0 / 64), fb);
          else tab_load<CG>(a, &maps.a, k, (int)m0, fb);
          if (!B_MN) tab_load<CG>(b, &maps.b, k, (int)n0, fb);
          else if (g.b_whole) tab_load_blocks<CG>(b, &maps.b, k, (int)(n0 / 64), fb);
          else for (int j = 0; j < b_cols / 64; ++j) tab_load<CG>(b + j * NPB * ATOM_BYTES, &maps.b, (int)n0 + 64 * j, k, fb);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- products.  D fp32; both operands of one type; the smallest planes' products first, (0, 0) last
    const uint32_t idesc = (1u << 4) | (FMT << 7) | (FMT << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                           ((uint32_t)(g.BN >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
    // K-major: 128-byte rows in the 128-byte swizzle (layout 2) or 64-byte rows in the 64-byte one (layout 4), 32 bytes per 16 k-values;
    // MN-major: 64 columns x KB rows in the 128-byte swizzle, 2048 bytes per 16 k-values
    constexpr uint32_t K_SBO = KB == 64 ? 1024 : 512, K_LAYOUT = KB == 64 ? 2 : 4;
    constexpr uint32_t a_step = A_MN ? 2048 : 32, b_step = B_MN ? 2048 : 32;
    const bool leader = elect_one();
    StageRing at;
    int j = 0;
    bool ok = rank == 0;
    for (long long t = first; t < ntiles && ok; t += step) {
      long long m0, n0;
      int split, kb0, kb1;
      tile(t, m0, n0, split, kb0, kb1);
      for (int p0 = kb0, p1; p0 < kb1 && ok; p0 = p1, ++j) {
        const int ab = j & 1;
        p1 = kb1 - p0 < g.part ? kb1 : p0 + g.part;
        ok = failed == 0 && tab_wait(acce_bar(ab), (uint32_t)((j >> 1) & 1) ^ 1u, g);
        if (!__all_sync(0xffffffffu, ok)) { failed = 1; ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem + (uint32_t)ab * 256u;
        for (int kb = p0; kb < p1; ++kb, at.next(g.stages)) {
          ok = tab_wait(full_bar(at.s), at.parity, g);
          if (!__all_sync(0xffffffffu, ok)) { failed = 1; ok = false; break; }
          const uint32_t a = smem_u32(smem) + (uint32_t)at.s * stage_bytes, b = a + A_BYTES;
          const uint64_t da = A_MN ? smem_desc(a, NPA * ATOM_BYTES, 1024, 2) : smem_desc(a, 0, K_SBO, K_LAYOUT);
          const uint64_t db = B_MN ? smem_desc(b, NPB * ATOM_BYTES, 1024, 2) : smem_desc(b, 0, K_SBO, K_LAYOUT);
          // (one branch for all of a stage: each of its own costs the issuing warp more than a product takes)
          if (leader) {
#pragma unroll
            for (int k = 0; k < KB / 16; ++k) {
              bool more = k > 0 || kb > p0;
#pragma unroll
              for (int sum = (NPA > NPB ? NPA : NPB) - 1; sum >= 0; --sum)
#pragma unroll
                for (int pa = sum; pa >= 0; --pa) {
                  if (pa >= NPA || sum - pa >= NPB) continue;
                  tab_mma<CG>(acc, desc_at(da, pa * a_plane + k * a_step), desc_at(db, (sum - pa) * b_plane + k * b_step), idesc, more);
                  more = true;
                }
            }
            tab_commit<CG>(empty_bar(at.s));
          }
          __syncwarp();
        }
        if (ok && leader) tab_commit<CG>(accf_bar(ab));
      }
    }
  } else {
    // ---------------- epilogue
    const int q = warp & 3, half = (warp - 2) >> 2, hc = g.BN / 2;       // 32 rows of the tile; half of its columns
    unsigned char *buf = ostage + (size_t)(warp - 2) * TabSmem<EPI, MATH>::OUT;
    const uint32_t drained = CG == 1 ? 0u : in_first_cta(acce_bar(0));
    // what a result is multiplied by (two factors where one could leave fp32), and a score's way to base 2
    float unscale = 1.f, unscale2 = 1.f, up = 1.f;
    const float to2 = g.scale * TOK_LOG2E;
    if (g.sc) {
      up = g.sc->dz;
      const float iop = g.by_q ? g.sc->iq : g.sc->iw;
      unscale = NPB == 3 ? fminf(iop, g.sc->idz) : iop * g.sc->idz;      // (the smaller one first)
      unscale2 = fmaxf(iop, g.sc->idz);
    }
    auto result = [&](float v) { return NPB == 3 ? v * unscale * unscale2 : v * unscale; };
    constexpr int MOST_PLANES = NPB == 2 ? 3 : 2;
    const int planes = NPB == 2 ? 3 : g.dz_planes;
    int j = 0;
    bool ok = true;
    long long t = first;
    for (; t < ntiles; t += step) {
      long long m0, n0;
      int split, kb0, kb1;
      tile(t, m0, n0, split, kb0, kb1);
      const long long m = m0 + q * 32 + lane;
      // what a row of dz takes, read while the products run: dz = -p (gg + hh log2 p) (+ g0 at the target)
      float lse = 0.f, g0 = 0.f, gg = 0.f, hh = 0.f;
      long long hot = -1;
      if (EPI != EPI_OUT && m < g.M) {
        const long long target = g.targets[m];
        if (target >= 0 && target < g.vocab && target != g.ignore_index) {
          if (EPI == EPI_DZ) {
            lse = g.lse[m] * TOK_LOG2E;
            if (g.g) g0 = gg = g.g[m] * g.scale * up;
            if (g.h) { const float h = g.h[m] * g.scale * up; hh = h * TOK_LN2; gg = fmaf(h, g.entropy[m], gg); }
          }
          hot = target - g.v0;
        } else if (EPI == EPI_DZ && target != g.ignore_index && n0 == 0 && half == 0 && g.v0 == 0) atomicOr(g.err, TOK_ERR_ID);
      }
      const long long c0 = n0 + half * hc;                               // first column of this warp
      const int cols = c0 >= g.N ? 0 : g.N - c0 < hc ? (int)(g.N - c0) : hc;
      const bool idle = m0 + q * 32 >= g.M;                              // none of these rows exists
      const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * hc);
      // the columns' factors, for all rows of the warp
      constexpr bool SCALED = EPI != EPI_OUT && NPB == 2;
      float4 *cols_f = reinterpret_cast<float4 *>(EPI == EPI_DZ ? ostage + TAB_EPI_WARPS * TabSmem<EPI, MATH>::OUT + (warp - 2) * 512 : buf);
      float row_f = 0.f;
      if (SCALED) {
        __syncwarp();
        if (4 * lane < hc) cols_f[lane] = reinterpret_cast<const float4 *>(g.col_f + c0)[lane];
        if (m < g.M) row_f = g.row_f[m];
        __syncwarp();
      }
      // The tile's values.  PARTS: all of them, added up in registers as the accumulators fill; else read by 32 columns below.
      float sum[PARTS ? 128 : 1];
      // (the whole warp waits: one lane that does and a vote behind it take 200 cycles longer)
      auto wait_full = [&]() {
        const bool w = tab_wait(accf_bar(j & 1), (uint32_t)(j >> 1) & 1, g);
        if (!__all_sync(0xffffffffu, w)) { failed = 1; return false; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        return true;
      };
      // (one arrival per warp, and no release beyond the tensor memory's: a release to the cluster waits for every store made so far)
      auto give_back = [&]() {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (CG == 1) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(acce_bar(j & 1)) : "memory");
          else asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" :: "r"(drained + 8u * (j & 1)) : "memory");
        }
        ++j;
      };
      if (PARTS) {
#pragma unroll
        for (int i = 0; i < 128; ++i) sum[PARTS ? i : 0] = 0.f;
        for (int p0 = kb0; p0 < kb1; p0 = kb1 - p0 < g.part ? kb1 : p0 + g.part) {
          ok = wait_full();
          if (!ok) break;
#pragma unroll
          for (int x = 0; x < 128; x += 32) {
            if (x >= hc || idle) continue;
            uint32_t v[32];
            tmem_ld32(lanes + (uint32_t)(j & 1) * 256u + x, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[PARTS ? x + i : 0] += __uint_as_float(v[i]);
          }
          give_back();
        }
        if (!ok) break;
      } else if (kb0 < kb1) {
        ok = wait_full();
        if (!ok) break;
      }
      // 32 columns of the tile (a split without k-values holds zeros)
      auto values = [&](int x, float (&v)[32]) {
        if (PARTS) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = sum[PARTS ? x + i : 0];
        } else if (kb0 < kb1) {
          uint32_t r[32];
          tmem_ld32(lanes + (uint32_t)(j & 1) * 256u + x, r);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
      };

      float mx = -INFINITY, r = 0.f;                                     // EPI_STATS: largest product, reference; sums of even and odd columns
      unsigned long long S2 = f32x2(0.f, 0.f), T2 = S2;
      // the padding of dz's last columns is written too, as zeros: the contraction over the table's rows reads whole blocks
      const int span = EPI == EPI_DZ ? (c0 >= g.ldz ? 0 : g.ldz - c0 < hc ? (int)(g.ldz - c0) : hc) : cols;
      const int rows = g.M - (m0 + q * 32) < 32 ? (int)(g.M - (m0 + q * 32)) : 32;
      // before the buffer is written again, what was stored from it has been read; then it goes
      auto store_ready = [&]() {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
      };
      auto store_go = [&](int col, int row, int part, bool any) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && any) {
          asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" :: "l"(&maps.c), "r"(col), "r"(row), "r"(part), "r"(smem_u32(buf)) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      };
#pragma unroll(PARTS ? 4 : 1)
      for (int x = 0; x < 128; x += 32) {
        if (x >= span || idle) break;
        float v[32];
        values(x, v);
        const float c = SCALED ? 1.f : to2;                              // from here to a score in base 2
        if (SCALED) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 f = cols_f[(x + i) / 4];
            v[i] *= row_f * f.x; v[i + 1] *= row_f * f.y; v[i + 2] *= row_f * f.z; v[i + 3] *= row_f * f.w;
          }
        }
        if (EPI == EPI_STATS) {
          if (__any_sync(0xffffffffu, hot >= c0 + x && hot < c0 + x + 32)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) if (hot == c0 + x + i) g.at_target[m] = v[i];
          }
          if (cols - x < 32) {                                             // columns that do not exist
#pragma unroll
            for (int i = 0; i < 32; ++i) if (i >= cols - x) v[i] = -INFINITY;
          }
          float cm = v[0];
#pragma unroll
          for (int i = 1; i < 32; ++i) cm = fmaxf(cm, v[i]);
          if (cm > mx) {
            mx = cm;
            const float d = fminf(fmaxf((r - cm) * c, -1e30f), 0.f), f = tok_ex2(d);
            const unsigned long long f2 = f32x2(f, f), zero = f32x2(0.f, 0.f);
            T2 = f32x2_fma(f32x2_fma(f32x2(d, d), S2, T2), f2, zero);
            S2 = f32x2_fma(S2, f2, zero);
            r = cm;
          }
          // (the difference to the largest is formed first: nothing of it is lost, however large the two are)
          const unsigned long long r2 = f32x2(-r, -r), c2 = f32x2(c, c);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            unsigned long long d2 = f32x2_add(f32x2(v[i], v[i + 1]), r2);
            if (!SCALED) d2 = f32x2_fma(d2, c2, f32x2(0.f, 0.f));
            const float2 d = f32x2_parts(d2);
            const float y0 = tok_max_nan(d.x, -1000.f), y1 = tok_max_nan(d.y, -1000.f);      // (2^-1000 is 0 too, and 0 times -inf no number)
            const unsigned long long e2 = f32x2(tok_ex2(y0), tok_ex2(y1));
            S2 = f32x2_add(S2, e2);
            T2 = f32x2_fma(f32x2(y0, y1), e2, T2);
          }
        } else if (EPI == EPI_DZ) {
          const long long col = c0 + x;
          // a row that does not count is a query of zeros: its score is 0, and with lse = gg = hh = 0 so is its dz
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            // log p and p, in base 2.  p is 0 for a score of -inf, and never above 1, however little the score and lse share where both are large
            // (a query of 1e12 with a gradient of 0 adds 0 to the table's)
            const float y = tok_min_nan(tok_max_nan(fmaf(v[i], c, -lse), -1000.f), 0.f), p = tok_ex2(y);
            v[i] = -p * fmaf(hh, y, gg);
          }
          if (__any_sync(0xffffffffu, hot >= col && hot < col + 32)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) if (hot == col + i) v[i] += g0;
          }
          if (col + 32 > g.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i) if (col + i >= g.N) v[i] = 0.f;
          }
          // planes of 32 rows through shared memory; 64 columns of each leave as one bulk store, clipped at the last row (columns come in 64s).  (Of 32
          // columns: 225 us instead of 199 for the dz of 5000 x 14,951 x 400 fp32.)
          if ((x & 32) == 0) store_ready();
#pragma unroll
          for (int pl = 0; pl < MOST_PLANES; ++pl) {
            if (pl >= planes) break;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float &a = v[8 * u + 2 * i], &b = v[8 * u + 2 * i + 1];
                const typename TokPair<Dz>::type e = TokPair<Dz>::down(a, b);
                if (pl < MOST_PLANES - 1) { const float2 f = TokPair<Dz>::up(e); a -= f.x; b -= f.y; }      // what the next plane holds
                w[i] = *reinterpret_cast<const uint32_t *>(&e);
              }
              unsigned char *at = buf + pl * 4096 + lane * 128 + (((u + (x & 32) / 8) ^ (lane & 7)) << 4);
              *reinterpret_cast<uint4 *>(at) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && rows > 0 && (x & 32)) {
            for (int pl = 0; pl < planes; ++pl)
              asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                           :: "l"(&maps.c), "r"((int)(col - 32)), "r"((int)(m0 + q * 32)), "r"(pl), "r"(smem_u32(buf + pl * 4096)) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else if (!g.bulk) {
          // row by row, whatever the rows' alignment
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4 *>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
          __syncwarp();
          const long long col = c0 + x + lane;
          if (x + lane < cols) {
            for (int r0 = 0; r0 < rows; ++r0) {
              const float val = result(*reinterpret_cast<float *>(buf + r0 * 128 + (((lane >> 2) ^ (r0 & 7)) << 4) + ((lane & 3) << 2)));
              const long long row = m0 + q * 32 + r0;
              if (g.partial) {
                float *to = g.partial + ((long long)split * g.M + row) * g.N + col;
                *to = g.add ? *to + val : val;
              } else ((Out *)g.out)[row * g.ldo + col] = Tok<Out>::down(val);
            }
          }
        } else if (sizeof(Out) == 4 || g.partial) {
          // 32 x 32 values as one bulk store, clipped at the matrix' edges
          store_ready();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4 *>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_float4(result(v[4 * u]), result(v[4 * u + 1]), result(v[4 * u + 2]), result(v[4 * u + 3]));
          store_go((int)(c0 + x), (int)(m0 + q * 32), split, rows > 0);
        } else {
          // 16-bit results: 64 columns to a row of 128 bytes
          if ((x & 32) == 0) store_ready();
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const auto e = TokPair<Elem>::down(result(v[8 * u + 2 * i]), result(v[8 * u + 2 * i + 1]));
              w[i] = *reinterpret_cast<const uint32_t *>(&e);
            }
            *reinterpret_cast<uint4 *>(buf + lane * 128 + (((u + (x & 32) / 8) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if ((x & 32) || x + 32 >= span) store_go((int)(c0 + (x & ~32)), (int)(m0 + q * 32), 0, rows > 0);
        }
      }
      if (EPI == EPI_STATS && m < g.M) g.parts[m * g.nparts + n0 / g.BN * 2 + half] = make_float4(mx, r, f32x2_parts(S2).x + f32x2_parts(S2).y, f32x2_parts(T2).x + f32x2_parts(T2).y);
      if (!PARTS && kb0 < kb1) give_back();
    }
    // a wait has run out: what this warp had still to write
    if (!ok) for (; t < ntiles; t += step) {
      long long m0, n0;
      int split, kb0, kb1;
      tile(t, m0, n0, split, kb0, kb1);
      const long long m = m0 + q * 32 + lane, c0 = n0 + half * hc, c1 = c0 + hc < g.N ? c0 + hc : g.N;
      const float nan = __int_as_float(0x7fc00000);
      if (m >= g.M) continue;
      if (EPI == EPI_STATS) g.parts[m * g.nparts + n0 / g.BN * 2 + half] = make_float4(0.f, 0.f, nan, nan);
      else for (long long c = c0; c < c1; ++c) {
        if (EPI == EPI_DZ) for (int pl = 0; pl < planes; ++pl) ((Dz *)g.out)[(pl * g.M + m) * g.ldz + c] = Tok<Dz>::down(nan);
        else if (g.partial) g.partial[((long long)split * g.M + m) * g.N + c] = nan;
        else ((Out *)g.out)[m * g.ldo + c] = Tok<Out>::down(nan);
      }
    }
    if (EPI != EPI_STATS && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");         // the stores are performed
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CG == 2) pair_sync();                                              // the other CTA's products read this one's shared memory
  if (warp == 1) {
    // after a wait that ran out copies and products may still be in flight: a bounded grace before the tensor memory goes back
    if (failed) for (int i = 0; i < 200000; ++i) __nanosleep(20);
    if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
  }
}

// A query's partial sums to its statistics; c and natural take a product to a score in base 2 and to one.  The target's score is the
// product that S was made of: another one, as exact as it may be, could come out above lse.
__global__ void __launch_bounds__(128) tab_stats_kernel(const long long *__restrict__ targets, long long ignore_index, long long vocab, float c, float natural,
                                                        const float4 *__restrict__ parts, int nparts, const float *__restrict__ at_target, float *logprob, float *entropy,
                                                        float *lse, int *errors) {
  __shared__ Soft sums[4];
  pdl_begin();
  const long long n = blockIdx.x, target = targets[n];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (target == ignore_index) {
    if (threadIdx.x == 0) { logprob[n] = 0.f; entropy[n] = 0.f; lse[n] = 0.f; }
    return;
  }
  const bool known = target >= 0 && target < vocab;
  Soft s{-INFINITY, 0.f, 0.f, 0.f};
  for (int i = threadIdx.x; i < nparts; i += 128) { const float4 p = parts[n * nparts + i]; soft_join(s, Soft{p.x, p.y, p.z, p.w}, c); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) soft_join(s, soft_shfl(s, o), c);
  if (lane == 0) sums[w] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 4; ++i) soft_join(s, sums[i], c);
  const bool empty = s.m == -INFINITY && s.S == 0.f;                     // nothing but -inf
  const float log_s = logf(s.S);
  lse[n] = empty ? -INFINITY : fmaf(s.r, natural, log_s);
  // (S holds the largest score's term, which is 1, and the target's)
  entropy[n] = empty ? 0.f : tok_max_nan(log_s - s.T * TOK_LN2 / s.S, 0.f);
  logprob[n] = !known ? __int_as_float(0x7fc00000) : empty ? -INFINITY : tok_min_nan(fmaf(at_target[n] - s.r, natural, -log_s), 0.f);
  if (!known && errors) atomicOr(errors, TOK_ERR_ID);
}

// ---- a few fp32 queries ----------------------------------------------------------------------------------------
// The queries lie in shared memory; a warp takes R rows of the table at a time, its lanes along the rows, so that a query's
// 512 bytes serve R rows.  HBM bounds it up to 8 queries (65,536 x 2048: one 85 us, seven 107; planes take 300 for 17), then the reads
// of the queries (sixteen 161 us).
#define TAB_FEW 16
#define TAB_FEW_WARPS 16
#define TAB_FEW_BYTES 196608
static __host__ __device__ constexpr int few_rows(int nq) { return nq <= 8 ? 4 : 2; }

template <int NQ, bool WIDE>
__global__ void __launch_bounds__(32 * TAB_FEW_WARPS, 1)
tab_few_kernel(const float *__restrict__ queries, long long q_stride, int n, const float *__restrict__ table, long long t_stride, long long vocab, int dim, float scale,
               const long long *__restrict__ targets, float4 *parts, float *at_target) {
  constexpr int R = few_rows(NQ), C = R * NQ, V = WIDE ? 4 : 1;
  extern __shared__ __align__(16) float few_q[];                         // [NQ][dim rounded up to 4]
  __shared__ Soft sums[TAB_FEW_WARPS][C];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, ld = (dim + 3) / 4 * 4;
  for (int q = w; q < NQ; q += TAB_FEW_WARPS)
    for (int i = lane; i < ld; i += 32) few_q[q * ld + i] = q < n && i < dim ? queries[q * q_stride + i] : 0.f;
  __syncthreads();
  const float c = scale * TOK_LOG2E;
  Soft s{-INFINITY, 0.f, 0.f, 0.f};
  constexpr int SHIFT = C == 32 ? 0 : C == 16 ? 1 : C == 8 ? 2 : 3;
  const int mine = lane >> SHIFT, my_row = mine / NQ;   // the product that ends in this lane
  const long long target = mine % NQ < n && (lane & ((1 << SHIFT) - 1)) == 0 ? targets[mine % NQ] : -1;
  for (long long v0 = ((long long)blockIdx.x * TAB_FEW_WARPS + w) * R; v0 < vocab; v0 += (long long)gridDim.x * TAB_FEW_WARPS * R) {
    float acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    const float *row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) row[r] = table + (v0 + r < vocab ? v0 + r : vocab - 1) * t_stride;
#pragma unroll 2
    for (int i = lane; i < dim / V; i += 32) {
      float x[R][V];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (WIDE) { const float4 f = __ldcs((const float4 *)row[r] + i); x[r][0] = f.x; x[r][1] = f.y; x[r][2] = f.z; x[r][3] = f.w; }
        else x[r][0] = row[r][i];
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float y[V];
        if constexpr (WIDE) { const float4 f = ((const float4 *)(few_q + q * ld))[i]; y[0] = f.x; y[1] = f.y; y[2] = f.z; y[3] = f.w; }
        else y[0] = few_q[q * ld + i];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int k = 0; k < V; ++k) acc[r * NQ + q] = fmaf(x[r][k], y[k], acc[r * NQ + q]);
      }
    }
    // the lanes' sums, halving what a lane still holds at every step
    int have = C;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (have > 1) {
        have /= 2;
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          if (i >= have) break;
          const float keep = lane & o ? acc[i + have] : acc[i], give = lane & o ? acc[i] : acc[i + have];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      } else acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
    }
    if (v0 + my_row < vocab) {
      const float z = acc[0];
      if (v0 + my_row == target) at_target[mine % NQ] = z;
      if (z > s.m) { s.m = z; soft_rebase(s, soft_reference(z), c); }
      const float y = tok_max_nan((z - s.r) * c, -1000.f), e = tok_ex2(y);
      s.S += e;
      s.T = fmaf(y, e, s.T);
    }
  }
  if ((lane & ((1 << SHIFT) - 1)) == 0) sums[w][mine] = s;
  __syncthreads();
  if (threadIdx.x < n) {
    Soft a{-INFINITY, 0.f, 0.f, 0.f};
    for (int i = 0; i < TAB_FEW_WARPS; ++i)
      for (int r = 0; r < R; ++r) soft_join(a, sums[i][r * NQ + threadIdx.x], c);
    parts[(long long)threadIdx.x * gridDim.x + blockIdx.x] = make_float4(a.m, a.r, a.S, a.T);
  }
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
// A matrix on its way to becoming an operand: `blocks` CTAs of a preparing kernel work on it.
struct TabSource { const void *x; long long stride, rows; TabRows counts; int blocks; void *to; long long ld, plane; };
struct TabPrep {
  TabSource q, w;                                          // blocks 0: not prepared
  const float *g, *h; long long n; int gblocks;            // gblocks 0: dz is not scaled
  float scale; int dim, planes, wide;                      // wide: rows of whole 16-byte vectors on 16-byte boundaries
  FastDiv by_units;                                        // units of a row: vectors, or elements
  unsigned *block_max; int max_q, max_w;                   // the largest elements of parts of the queries, of the table, and of dz's bound
  TabScales *sc;
};

// Hands the units of type U of a CTA's rows (those that do not count as zeros) to a function (row, unit, value), four in flight.
template <class U, class F>
__device__ __forceinline__ void tab_units(const TabPrep &a, const TabSource &s, int b, F &&f) {
  const int units = a.dim / (int)(sizeof(U) / (a.planes ? 4 : 2));
  const long long per = (s.rows + s.blocks - 1) / s.blocks, r0 = b * per, rows = s.rows - r0 < per ? s.rows - r0 : per;
  const int total = rows > 0 ? (int)(rows * units) : 0;
  for (int i0 = threadIdx.x; i0 < total; i0 += 4 * 256) {
    U v[4];
    long long row[4];
    int at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * 256 < total ? i0 + k * 256 : i0, r = a.by_units.div(i);
      row[k] = r0 + r;
      at[k] = i - r * units;
      v[k] = U{};
      if (s.counts(row[k])) v[k] = ((const U *)((const char *)s.x + row[k] * s.stride * (a.planes ? 4 : 2)))[at[k]];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) if (i0 + k * 256 < total) f(row[k], at[k], v[k]);
  }
}
// The bound of dz / scale: |g| + |h| (p |log p| + p H), p |log p| <= 1 / e, H <= log rows < 22.  The largest finite one of a CTA's queries,
// bit by bit (of a thread).
__device__ __forceinline__ unsigned tab_dz_bound(const float *g, const float *h, const TabRows &counts, long long n, int b, int blocks) {
  unsigned top = 0u;
  for (long long i = (long long)b * 256 + threadIdx.x; i < n; i += blocks * 256) {
    if (!counts(i)) continue;
    const unsigned bits = __float_as_uint((g ? fabsf(g[i]) : 0.f) + (h ? 23.f * fabsf(h[i]) : 0.f));
    if (bits < 0x7f800000u) top = max(top, bits);
  }
  return top;
}
// The largest of a CTA's threads' numbers to block_max[blockIdx.x].
__device__ __forceinline__ void tab_leave_max(unsigned top, unsigned *block_max) {
  __shared__ unsigned tops[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) top = max(top, tops[i]);
    block_max[blockIdx.x] = top;
  }
}
__global__ void __launch_bounds__(256) tab_max_kernel(TabPrep a) {
  pdl_begin();
  tab_leave_max(tab_dz_bound(a.g, a.h, a.q.counts, a.n, blockIdx.x, a.gblocks), a.block_max);
}
// 2^k that brings a number below 2^top, |k| <= 126: 2^-k is a normal number too, and the smallest normal one comes out at 1
__device__ __forceinline__ float tab_power(unsigned bits, int top, float &inverse) {
  int k = bits ? top - ((int)(bits >> 23) - 126) : 0;
  k = k < -126 ? -126 : k > 126 ? 126 : k;
  inverse = __uint_as_float((unsigned)(127 - k) << 23);
  return __uint_as_float((unsigned)(127 + k) << 23);
}
__device__ __forceinline__ void tab_split3(float v, __nv_bfloat16 &b0, __nv_bfloat16 &b1, __nv_bfloat16 &b2) {
  b0 = __float2bfloat16_rn(v);
  const float r = __hisinf(b0) || __hisnan(b0) ? 0.f : v - __bfloat162float(b0);
  b1 = __float2bfloat16_rn(r);
  b2 = __float2bfloat16_rn(r - __bfloat162float(b1));
}
__device__ __forceinline__ void tab_split(float v, __half &b0, __half &b1) {
  b0 = __float2half_rn(v);
  b1 = __hisinf(b0) || __hisnan(b0) ? __float2half_rn(0.f) : __float2half_rn(v - __half2float(b0));
}
// fp32 to three bf16 planes; 16-bit elements as they are (rows that TMA cannot read where they lie, and the gradient's queries).
// Rows that do not count become zeros: whatever stands in padding, a product with its zero gradient is zero.
template <class T>
__global__ void __launch_bounds__(256) tab_pack_kernel(TabPrep a) {
  __shared__ unsigned tops[3];
  pdl_begin();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float up_q = 1.f, up_w = 1.f;
  if (a.sc) {
    const int nq = a.max_q, nw = a.max_w;
    if (w < 3) {                                                          // a warp each: queries, table, gradients
      const int lo = w == 0 ? 0 : w == 1 ? nq : nq + nw, hi = w == 0 ? nq : w == 1 ? nq + nw : nq + nw + a.gblocks;
      unsigned top = 0u;
      for (int i = lo + lane; i < hi; i += 32) top = max(top, a.block_max[i]);
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) tops[w] = top;
    }
    __syncthreads();
    TabScales s = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (a.planes) { s.q = tab_power(tops[0], 40, s.iq); s.w = tab_power(tops[1], 40, s.iw); }
    if (a.gblocks) s.dz = tab_power(__float_as_uint(fminf(__uint_as_float(tops[2]) * a.scale, 1e38f)), a.planes ? 40 : 14, s.idz);
    up_q = s.q;
    up_w = s.w;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.sc = s;
  }
  const bool of_q = (int)blockIdx.x < a.q.blocks;
  const TabSource &s = of_q ? a.q : a.w;
  const int b = of_q ? blockIdx.x : blockIdx.x - a.q.blocks;
  const float up = of_q ? up_q : up_w;
  if constexpr (sizeof(T) == 4) {
    __nv_bfloat16 *p0 = (__nv_bfloat16 *)s.to, *p1 = p0 + s.plane, *p2 = p1 + s.plane;
    if (a.wide) tab_units<float4>(a, s, b, [&](long long r, int i, const float4 &v) {
      __align__(8) __nv_bfloat16 h0[4], h1[4], h2[4];
      tab_split3(v.x * up, h0[0], h1[0], h2[0]); tab_split3(v.y * up, h0[1], h1[1], h2[1]);
      tab_split3(v.z * up, h0[2], h1[2], h2[2]); tab_split3(v.w * up, h0[3], h1[3], h2[3]);
      ((uint2 *)(p0 + r * s.ld))[i] = *(uint2 *)h0;
      ((uint2 *)(p1 + r * s.ld))[i] = *(uint2 *)h1;
      ((uint2 *)(p2 + r * s.ld))[i] = *(uint2 *)h2;
    });
    else tab_units<float>(a, s, b, [&](long long r, int i, float v) { tab_split3(v * up, p0[r * s.ld + i], p1[r * s.ld + i], p2[r * s.ld + i]); });
  } else {
    if (a.wide) tab_units<uint4>(a, s, b, [&](long long r, int i, const uint4 &v) { ((uint4 *)((T *)s.to + r * s.ld))[i] = v; });
    else tab_units<unsigned short>(a, s, b, [&](long long r, int i, unsigned short v) { ((unsigned short *)s.to)[r * s.ld + i] = v; });
  }
}
// Rows of fp32 to two fp16 planes, each times the power of two that brings its own largest finite element below 2^14; the factors take
// what undoes it, times fq or fw.  `group` threads to a row (up to the whole CTA), which stays in registers up to 8 units to a thread and
// is read again from there on.  Rows that do not count become zeros.
struct TabRowsPrep {
  TabSource q, w;                                          // blocks 0: not prepared
  float fq, fw, *row_f, *col_f;
  int dim, group;
  const float *g, *h; long long n; int gblocks;
  unsigned *block_max;                                     // null, or for the largest element that each CTA has seen
};
template <class U>
__global__ void __launch_bounds__(256) tab_rows_kernel(TabRowsPrep a) {
  __shared__ unsigned tops[8];
  pdl_begin();
  constexpr int V = sizeof(U) / 4;
  const bool of_q = (int)blockIdx.x < a.q.blocks;
  const int b = of_q ? blockIdx.x : blockIdx.x - a.q.blocks, group = a.group;
  if (!of_q && b >= a.w.blocks) {
    tab_leave_max(tab_dz_bound(a.g, a.h, a.q.counts, a.n, b - a.w.blocks, a.gblocks), a.block_max);
    return;
  }
  const TabSource &s = of_q ? a.q : a.w;
  float *factors = of_q ? a.row_f : a.col_f;
  const float factor = of_q ? a.fq : a.fw;
  const int sub = threadIdx.x % group, units = a.dim / V;
  const long long per = 256 / group;
  unsigned most = 0u;
  __half *p0 = (__half *)s.to, *p1 = p0 + s.plane;
  for (long long r0 = b * per; r0 < s.rows; r0 += s.blocks * per) {
    const long long r = r0 + threadIdx.x / group;
    const bool there = r < s.rows, counts = there && s.counts(r);
    const U *row = (const U *)((const float *)s.x + r * s.stride);
    U v[8];
    auto load = [&](int i0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) { v[k] = U{}; if (counts && i0 + k * group < units) v[k] = row[i0 + k * group]; }
    };
    unsigned top = 0u;
    for (int i0 = sub; i0 < units; i0 += 8 * group) {
      load(i0);
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const unsigned bits = __float_as_uint(reinterpret_cast<const float *>(&v[k])[e]) & 0x7fffffffu;
          if (bits < 0x7f800000u) top = max(top, bits);
        }
    }
    for (int o = group < 32 ? group / 2 : 16; o > 0; o /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (group > 32) {
      const int w = threadIdx.x / 32, warps = group / 32;
      if (threadIdx.x % 32 == 0) tops[w] = top;
      __syncthreads();
      for (int k = w / warps * warps; k < (w / warps + 1) * warps; ++k) top = max(top, tops[k]);
      __syncthreads();
    }
    most = max(most, top);
    float inverse;
    const float up = tab_power(top, 14, inverse);
    if (there && sub == 0) factors[r] = inverse * factor;
    for (int i0 = sub; i0 < units; i0 += 8 * group) {
      if (units > 8 * group) load(i0);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (!there || i0 + k * group >= units) continue;
        __align__(8) __half h0[V], h1[V];
#pragma unroll
        for (int e = 0; e < V; ++e) tab_split(reinterpret_cast<const float *>(&v[k])[e] * up, h0[e], h1[e]);
        if (V == 4) {
          reinterpret_cast<uint2 *>(p0 + r * s.ld)[i0 + k * group] = *reinterpret_cast<uint2 *>(h0);
          reinterpret_cast<uint2 *>(p1 + r * s.ld)[i0 + k * group] = *reinterpret_cast<uint2 *>(h1);
        } else { p0[r * s.ld + i0 + k * group] = h0[0]; p1[r * s.ld + i0 + k * group] = h1[0]; }
      }
    }
  }
  if (a.block_max) tab_leave_max(most, a.block_max);
}
// The parts of a split contraction, added in their order.
template <class T>
__global__ void __launch_bounds__(256) tab_join_kernel(const float *__restrict__ partial, int splits, long long count, T *__restrict__ out) {
  pdl_begin();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) {
    float s = partial[i];
    for (int k = 1; k < splits; ++k) s += partial[k * count + i];
    out[i] = Tok<T>::down(s);
  }
}

// ---- host --------------------------------------------------------------------------------------------------
static std::atomic<int> tab_wait_limit{TC_WAIT_LIMIT};
extern "C" int32_t pbg_table_logprobs_wait_limit(int32_t limit) { return tab_wait_limit.exchange(limit < 0 ? TC_WAIT_LIMIT : limit); }

struct TabOperand { const void *base; long long rows, inner, ld, plane; int planes; bool room; };   // [planes][rows][ld], 16-bit elements; ours: room for whole blocks of 64

static bool tab_encode(CUtensorMap *tm, bool bf16, const TabOperand &o, int box_inner, int box_rows, int box_planes) {
  const cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane : o.ld * 8) * 2};
  const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, (cuuint32_t)box_planes};
  return encode_map(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, o.base, 3, dims, strides, box,
                    box_inner == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

// The same for an MN-major operand whose rows (with the room behind them) are whole blocks of 64 columns: the blocks are a dimension
// of their own, so that `blocks` of them are one box.  A box costs its issue; what lies beyond `inner` belongs to columns that are clipped.
// (The caller's rows have no such room, however far apart they lie: behind the last one the memory may end.)
static bool tab_encode_blocks(CUtensorMap *tm, bool bf16, const TabOperand &o, int box_rows, int blocks) {
  const cuuint64_t dims[4] = {64, (cuuint64_t)o.rows, (cuuint64_t)o.planes, (cuuint64_t)((o.inner + 63) / 64)};
  const cuuint64_t strides[3] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane : o.ld * 8) * 2, 128};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)o.planes, (cuuint32_t)blocks};
  return encode_map(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, o.base, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
static bool tab_whole(const TabOperand &o) { return o.inner % 64 == 0 || o.room; }

template <int EPI, class MATH, bool A_MN, bool B_MN, int CG, bool PARTS>
static bool tab_launch_as(const TabOperand &a, const TabOperand &b, const TabOperand *c, TabArgs &g, cudaStream_t st) {
  constexpr int KB = MATH::NPA == 1 ? 64 : 32;
  constexpr bool bf16 = std::is_same<typename MATH::elem, __nv_bfloat16>::value;
  if (pbg_launch_failed()) return true;
  TabMaps maps;
  g.wait_limit = tab_wait_limit.load();
  g.b_whole = B_MN && tab_whole(b);
  // Rows outside of the matrix are written as zeros, at a price: a box of 7 rows and 121 of zeros takes longer than one of 128 rows (7
  // queries, 131,072 x 2048 bf16: 127 us against 100).  A row of products depends on its own row of A alone, so what
  // stands in the rows that are not loaded is nobody's.
  g.a_rows = !A_MN && g.M < 128 ? (int)tok_up(g.M, 8) : 128;
  if (!(A_MN ? tab_encode_blocks(&maps.a, bf16, a, KB, 2) : tab_encode(&maps.a, bf16, a, KB, g.a_rows, a.planes))) return false;
  constexpr bool dz_bf16 = std::is_same<typename MATH::dz, __nv_bfloat16>::value;
  if (EPI == EPI_DZ && !tab_encode(&maps.c, dz_bf16, *c, 64, 32, 1)) return false;
  if (EPI == EPI_OUT) {
    // rows that begin on 16-byte boundaries; sums of several launches are added row by row
    const bool fp32 = g.partial || sizeof(typename MATH::out) == 4;
    const void *to = g.partial ? (const void *)g.partial : g.out;
    const long long row = (g.partial ? g.N : g.ldo) * (fp32 ? 4 : 2);
    g.bulk = aligned16(to) && row % 16 == 0 && !(g.partial && g.add);
    const cuuint64_t dims[3] = {(cuuint64_t)g.N, (cuuint64_t)g.M, (cuuint64_t)g.splits}, strides[2] = {(cuuint64_t)row, (cuuint64_t)row * g.M};
    const cuuint32_t box[3] = {fp32 ? 32u : 64u, 32, 1};
    if (g.bulk && !encode_map(&maps.c, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, to, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return false;
  }
  if (!(g.b_whole ? tab_encode_blocks(&maps.b, bf16, b, KB, g.BN / CG / 64) : tab_encode(&maps.b, bf16, b, B_MN ? 64 : KB, B_MN ? KB : g.BN / CG, b.planes))) return false;
  const int stage = MATH::NPA * 128 * KB * 2 + MATH::NPB * (g.BN / CG) * KB * 2;
  g.stages = std::min(int(TabSmem<EPI, MATH>::RING) / stage, TAB_STAGES_MAX);
  void (*kernel)(TabMaps, TabArgs) = tab_kernel<EPI, MATH, A_MN, B_MN, CG, PARTS>;
  pbg_opt_in_smem((const void *)kernel, TAB_SMEM);
  const long long tiles = (g.M + 128 * CG - 1) / (128 * CG) * ((g.N + g.BN - 1) / g.BN) * g.splits, most = pbg_sm_count() / CG;
  const unsigned groups = (unsigned)(tiles < most ? tiles : most);
  if (CG == 1) pbg_launch(kernel, dim3(groups), TAB_THREADS, TAB_SMEM, st, maps, g);
  else pbg_launch_clusters(kernel, (int)groups, CG, TAB_THREADS, TAB_SMEM, st, maps, g);
  return true;
}

// Tile columns, 128 or 256: the fewest columns for the SM with the most of them, with what a tile costs beside them -- a pair's, whose loads
// are no longer hidden behind its products when these are half as many, more than one of few queries, which waits for HBM either way.
static int tab_columns(long long tiles_m, long long N, int cg) {
  const long long groups = pbg_sm_count() / cg > 0 ? pbg_sm_count() / cg : 1;
  int best = 256;
  long long cost = -1;
  for (int bn = 256; bn >= 128; bn -= 128) {
    const long long tiles = tiles_m * ((N + bn - 1) / bn), c = (tiles + groups - 1) / groups * (bn + (cg == 2 ? 64 : 16));
    if (cost < 0 || c < cost) { cost = c; best = bn; }
  }
  return best;
}
// Parts of dQ's contraction over K table rows: the rounds of tiles that the SMs make, shortened by the parts, against writing and
// reading the parts' sums (in ns: 4096 products a cycle and SM at 1.7 GHz, 5 TB/s, 3 us for the launch that joins them).
static bool tab_pairs(long long M, long long N);
static int tab_splits(long long n, long long dim, long long K, int products) {
  const bool pairs = tab_pairs(n, dim);
  const long long groups = pbg_sm_count() / (pairs ? 2 : 1) > 0 ? pbg_sm_count() / (pairs ? 2 : 1) : 1;
  const long long tiles = (n + (pairs ? 255 : 127)) / (pairs ? 256 : 128) * ((dim + 255) / 256);
  int best = 1;
  double cost = 0.;
  for (int s = 1; s <= 64 && (s == 1 || (s * 512ll <= K && 4ll * s * n * dim <= TAB_SPLIT_BYTES)); ++s) {
    const double rounds = (double)((tiles * s + groups - 1) / groups) / s;
    const double c = rounds * ((double)K / 16 * products * 128 / 1.7) + (s > 1 ? 3000. + s * 8. * n * dim / 5000. : 0.);
    if (s == 1 || c < cost) { cost = c; best = s; }
  }
  return best;
}
// Pairs of CTAs where there are two row tiles for them and columns for whole halves.
static bool tab_pairs(long long M, long long N) { return M > 128 && N > 64; }

template <int EPI, class MATH, bool A_MN, bool B_MN>
static bool tab_launch(const TabOperand &a, const TabOperand &b, TabArgs &g, bool pairs, cudaStream_t st, const TabOperand *c = nullptr) {
  g.part = MATH::NPB == 1 ? TAB_PART_16 : EPI == EPI_OUT ? TAB_PART_F32_OUT : TAB_PART_F32;
  auto as = [&](auto parts) {
    return pairs ? tab_launch_as<EPI, MATH, A_MN, B_MN, 2, decltype(parts)::value>(a, b, c, g, st) : tab_launch_as<EPI, MATH, A_MN, B_MN, 1, decltype(parts)::value>(a, b, c, g, st);
  };
  if constexpr (MATH::NPB > 1) return as(std::true_type());
  else {
    if constexpr (EPI != EPI_OUT) if (g.kblocks > TAB_PART_16) return as(std::true_type());
    if constexpr (EPI == EPI_OUT)
      if (g.kblocks > TAB_PART_LONG) {
        g.part = TAB_PART_LONG;
        return as(std::true_type());
      }
    g.part = 0x7fffffff;
    return as(std::false_type());
  }
}

// TMA reads rows where they lie if they start on 16-byte boundaries
static bool tab_packed(const void *p, long long stride, int dim, int dtype) { return dtype == PBG_F32 || !aligned16(p) || stride % 8 != 0 || stride < dim; }

// What the workspace holds.  Its size is asked for without addresses, so it has room for packed operands wherever they may be needed.
#define TAB_MAX_BLOCKS 2048                                  // of a preparing kernel
struct TabPlace {
  int64_t scales, block_max, q, w, q3, w3, row_f, col_f, parts, at_target, dz, partial, bytes;                // q3, w3: bf16 planes of fp32 operands
  long long ld, columns, ldz;         // packed rows' length; table rows per piece of dz, and its rows' length
  long long piece;                    // queries per pass of the forward
  int npl, bn, nparts, splits, dz_planes;
  bool pairs, few;
};
static bool tab_few(long long n, int dim, int dtype);
static TabPlace tab_place(long long n, long long rows, int dim, int dtype, bool grad, bool rounded = false) {
  TabPlace p;
  p.npl = dtype == PBG_F32 ? 2 : 1;
  p.ld = tok_up(dim, 64);
  p.scales = 0;
  p.block_max = 256;
  p.q = p.block_max + TAB_MAX_BLOCKS * 4;
  p.w = p.q + tok_up(n * p.ld * 2 * p.npl, 256);
  int64_t at = p.w + tok_up(rows * p.ld * 2 * p.npl, 256);
  p.row_f = p.col_f = p.q3 = p.w3 = at;
  if (dtype == PBG_F32) {
    p.col_f = p.row_f + tok_up(n * 4, 256);
    p.q3 = p.col_f + tok_up(rows, 256) * 4;                                 // (whole tiles of columns are read)
    p.w3 = p.q3 + (grad ? tok_up(n * p.ld * 6, 256) : 0);
    at = p.w3 + (grad ? tok_up(rows * p.ld * 6, 256) : 0);
  }
  p.parts = p.at_target = p.dz = p.partial = at;
  p.columns = p.ldz = 0;
  p.piece = n;
  p.bn = p.nparts = p.splits = p.dz_planes = 0;
  p.pairs = tab_pairs(n, rows);
  p.few = !grad && tab_few(n, dim, dtype);
  if (p.few) {
    const long long groups = (rows + 4 * TAB_FEW_WARPS - 1) / (4 * TAB_FEW_WARPS);
    p.nparts = (int)(groups < pbg_sm_count() ? groups : pbg_sm_count());
    at = p.parts = p.q;                                      // no copies
    p.at_target = p.parts + n * p.nparts * 16;
    at = p.at_target + n * 4;
  } else if (!grad) {
    p.bn = tab_columns((n + (p.pairs ? 255 : 127)) / (p.pairs ? 256 : 128), rows, p.pairs ? 2 : 1);
    p.nparts = (int)((rows + p.bn - 1) / p.bn * 2);
    long long most = TAB_PARTS_BYTES / (16ll * p.nparts) / 256 * 256;
    if (most < 256) most = 256;
    if (p.piece > most) p.piece = most;
    p.at_target = at + p.piece * p.nparts * 16;
    at = p.at_target + p.piece * 4;
  } else {
    // dz of 16-bit operands keeps 16 bits or more in two planes of their type, and results are off by their own rounding (bf16 1.7e-3).  In one
    // plane it is rounded as they are: 2.3e-3, 3.8e-3 where the table's rows have much in common, for a third less time (4099 x 65,536 x 2048:
    // 4.2 and 2.7 ms; 1000 x 65,536 x 1024: 0.64 and 0.39).  Where the queries leave most of a tile's rows idle the reading of the
    // table covers the products, and one plane gains nothing.
    p.dz_planes = dtype == PBG_F32 ? 3 : rounded && n > 128 ? 1 : 2;
    long long most = TAB_DZ_BYTES / (2 * p.dz_planes * n) / 256 * 256;
    if (most < 256) most = 256;
    p.columns = rows < most ? rows : most;
    p.ldz = tok_up(p.columns, 64);
    at += tok_up(n * p.ldz * 2 * p.dz_planes, 256);
    p.partial = at;
    p.splits = tab_splits(n, dim, p.columns, dtype == PBG_F32 ? 6 : p.dz_planes);
    if (p.splits > 1 || p.columns < rows) at += tok_up((int64_t)p.splits * n * dim * 4, 256);
  }
  p.bytes = at;
  return p;
}

struct TabCall {
  const void *queries; int64_t q_stride, n; const void *table; int64_t t_stride, rows; int dim, dtype;
  const long long *targets; int64_t ignore_index; float scale; unsigned char *ws; int *errors; cudaStream_t st;
  TabScales *sc; int *err;
  TabOperand q, w, q3, w3;            // for the scores, and for the products with dz
};

static int tab_blocks(long long rows, int most) { const long long b = (rows + 7) / 8; return (int)(b < most ? b : most); }
static void tab_begin(TabCall &c, const TabPlace &p) {
  c.err = c.errors ? c.errors : (int *)(c.ws + p.scales + 128);          // (nobody reads the latter: the results say it)
  c.sc = nullptr;
  c.q = c.q3 = TabOperand{c.queries, c.n, c.dim, c.q_stride, 0, 1, false};
  c.w = c.w3 = TabOperand{c.table, c.rows, c.dim, c.t_stride, 0, 1, false};
}
static TabRows tab_counts(const TabCall &c, bool grad) { return TabRows{c.targets, c.ignore_index, c.rows, grad ? 0 : 1}; }
// Scales and operands, but for the scores of fp32.  For the gradient the queries are always copied: the rows that do not count have to be zeros.
template <class T>
static void tab_prepare(TabCall &c, const TabPlace &p, bool grad, const float *g, const float *h, int max_q, int max_w, int gblocks) {
  constexpr bool F32 = sizeof(T) == 4;
  const bool pack_q = grad || tab_packed(c.queries, c.q_stride, c.dim, c.dtype), pack_w = tab_packed(c.table, c.t_stride, c.dim, c.dtype);
  if (!pack_q && !pack_w) return;
  constexpr int V = F32 ? 4 : 8;
  TabPrep a = {};
  a.q.counts = tab_counts(c, grad);
  a.w.counts = TabRows{nullptr, 0, 0, 1};
  a.g = g; a.h = h; a.n = c.n; a.scale = c.scale; a.dim = c.dim; a.planes = F32; a.sc = c.sc;
  a.gblocks = gblocks; a.max_q = max_q; a.max_w = max_w;
  a.block_max = (unsigned *)(c.ws + p.block_max);
  a.wide = c.dim % V == 0;
  auto source = [&](TabSource &s, TabOperand &o, const void *x, long long stride, long long rows, int64_t at, int most) {
    s.x = x; s.stride = stride; s.rows = rows; s.to = c.ws + at; s.ld = p.ld; s.plane = rows * p.ld;
    s.blocks = tab_blocks(rows, most);
    if (!aligned16(x) || stride % V != 0) a.wide = 0;
    o = TabOperand{s.to, rows, c.dim, p.ld, s.plane, F32 ? 3 : 1, true};
  };
  if (pack_q) source(a.q, c.q3, c.queries, c.q_stride, c.n, F32 ? p.q3 : p.q, 296);
  if (pack_w) source(a.w, c.w3, c.table, c.t_stride, c.rows, F32 ? p.w3 : p.w, 1184);
  a.by_units = FastDiv(a.wide ? c.dim / V : c.dim);
  pbg_launch(tab_pack_kernel<T>, dim3(a.q.blocks + a.w.blocks), 256, 0, c.st, a);
  if (!F32) { c.q = c.q3; c.w = c.w3; }
}

// The operands of fp32 scores.  (The factors carry half of the scale's power each: their product is one of a score.)
static TabRowsPrep tab_rows_prep(TabCall &c, const TabPlace &p, bool grad) {
  TabRowsPrep a = {};
  const float to2 = c.scale * TOK_LOG2E;
  a.fq = ldexpf(1.f, ilogbf(to2) / 2);
  a.fw = to2 / a.fq;
  a.row_f = (float *)(c.ws + p.row_f);
  a.col_f = (float *)(c.ws + p.col_f);
  a.dim = c.dim;
  a.q = {c.queries, c.q_stride, c.n, tab_counts(c, grad), 0, c.ws + p.q, p.ld, c.n * p.ld};
  a.w = {c.table, c.t_stride, c.rows, TabRows{nullptr, 0, 0, 1}, 0, c.ws + p.w, p.ld, c.rows * p.ld};
  c.q = TabOperand{a.q.to, c.n, c.dim, p.ld, a.q.plane, 2, true};
  c.w = TabOperand{a.w.to, c.rows, c.dim, p.ld, a.w.plane, 2, true};
  return a;
}
static void tab_rows_launch(const TabCall &c, TabRowsPrep &a, bool q, bool w) {
  auto fits = [&](const TabSource &s) { return c.dim % 4 == 0 && s.stride % 4 == 0 && aligned16(s.x); };
  const bool wide = (!q || fits(a.q)) && (!w || fits(a.w));
  a.group = 1;
  while (a.group < 256 && a.group * 8 < (wide ? c.dim / 4 : c.dim)) a.group *= 2;
  const int per = 256 / a.group;
  auto blocks = [&](long long rows, int most) { const long long b = (rows + per - 1) / per; return (int)(b < most ? b : most); };
  a.q.blocks = q ? blocks(a.q.rows, w ? 296 : 1184) : 0;
  a.w.blocks = w ? blocks(a.w.rows, 1184) : 0;
  pbg_launch(wide ? tab_rows_kernel<float4> : tab_rows_kernel<float>, dim3(a.q.blocks + a.w.blocks + a.gblocks), 256, 0, c.st, a);
}

static bool tab_few(long long n, int dim, int dtype) {
  if (dtype != PBG_F32 || n > TAB_FEW) return false;
  long long nq = 1;
  while (nq < n) nq *= 2;
  return nq * tok_up(dim, 4) * 4 <= TAB_FEW_BYTES;
}
template <int NQ>
static void tab_few_launch(const TabCall &c, float4 *parts, int64_t at_target, int blocks) {
  const float *q = (const float *)c.queries, *t = (const float *)c.table;
  const bool wide = c.dim % 4 == 0 && aligned16(t) && c.t_stride % 4 == 0;
  auto kernel = wide ? tab_few_kernel<NQ, true> : tab_few_kernel<NQ, false>;
  const int smem = (int)(NQ * tok_up(c.dim, 4) * 4);
  pbg_opt_in_smem((const void *)kernel, TAB_FEW_BYTES);
  pbg_launch(kernel, dim3(blocks), 32 * TAB_FEW_WARPS, smem, c.st, q, (long long)c.q_stride, (int)c.n, t, (long long)c.t_stride, (long long)c.rows, c.dim, c.scale, c.targets, parts,
             (float *)(c.ws + at_target));
}

struct TabForward { TabCall c; TabPlace p; float *logprob, *entropy, *lse; bool ok; };
template <class T, class MATH>
static void tab_forward(TabForward &f) {
  TabCall &c = f.c;
  auto finish = [&](long long n0, long long n, float to2, float natural) {
    pbg_launch(tab_stats_kernel, dim3((unsigned)n), 128, 0, c.st, c.targets + n0, (long long)c.ignore_index, (long long)c.rows, to2, natural, (const float4 *)(c.ws + f.p.parts),
               f.p.nparts, (const float *)(c.ws + f.p.at_target), f.logprob + n0, f.entropy + n0, f.lse + n0, c.errors);
  };
  const float to2 = c.scale * TOK_LOG2E;
  if (f.p.few) {
    float4 *parts = (float4 *)(c.ws + f.p.parts);
    if (c.n == 1) tab_few_launch<1>(c, parts, f.p.at_target, f.p.nparts);
    else if (c.n == 2) tab_few_launch<2>(c, parts, f.p.at_target, f.p.nparts);
    else if (c.n <= 4) tab_few_launch<4>(c, parts, f.p.at_target, f.p.nparts);
    else if (c.n <= 8) tab_few_launch<8>(c, parts, f.p.at_target, f.p.nparts);
    else tab_few_launch<16>(c, parts, f.p.at_target, f.p.nparts);
    finish(0, c.n, to2, c.scale);
    return;
  }
  tab_begin(c, f.p);
  if (MATH::NPB == 2) {
    TabRowsPrep a = tab_rows_prep(c, f.p, false);
    tab_rows_launch(c, a, true, false);
    tab_rows_launch(c, a, false, true);
  } else tab_prepare<T>(c, f.p, false, nullptr, nullptr, 0, 0, 0);
  constexpr int KB = MATH::NPA == 1 ? 64 : 32;
  for (long long n0 = 0; n0 < c.n && f.ok; n0 += f.p.piece) {
    const long long n = c.n - n0 < f.p.piece ? c.n - n0 : f.p.piece;
    TabOperand q = c.q;
    q.base = (const char *)q.base + n0 * q.ld * 2;
    q.rows = n;
    TabArgs g = {};
    g.M = n; g.N = c.rows; g.kblocks = (int)((c.dim + KB - 1) / KB);
    g.BN = f.p.bn; g.splits = 1; g.m_first = 1; g.scale = c.scale; g.sc = c.sc; g.err = c.err;
    g.row_f = (const float *)(c.ws + f.p.row_f) + n0; g.col_f = (const float *)(c.ws + f.p.col_f);
    g.parts = (float4 *)(c.ws + f.p.parts); g.nparts = f.p.nparts; g.at_target = (float *)(c.ws + f.p.at_target);
    g.targets = c.targets + n0; g.ignore_index = c.ignore_index; g.vocab = c.rows;
    f.ok = tab_launch<EPI_STATS, MATH, false, false>(q, c.w, g, f.p.pairs, c.st);
    if (MATH::NPB == 2) finish(n0, n, 1.f, TOK_LN2);
    else finish(n0, n, to2, c.scale);
  }
}

struct TabBackward { TabCall c; TabPlace p; const float *lse, *entropy, *g, *h; void *dq, *dt; bool ok; };
// MATH: of the scores; DZMATH: of the products with dz
template <class T, class MATH, class DZMATH>
static void tab_backward(TabBackward &f) {
  TabCall &c = f.c;
  constexpr int KB = MATH::NPA == 1 ? 64 : 32, KB2 = DZMATH::NPA == 1 ? 64 : 32;
  tab_begin(c, f.p);
  const bool scaled = c.dtype != PBG_BF16;                               // dz is (and fp32 operands are)
  const int gblocks = scaled ? tab_blocks((c.n + 31) / 32, 64) : 0;
  int max_q = 0, max_w = 0;
  if (scaled) c.sc = (TabScales *)(c.ws + f.p.scales);
  if (MATH::NPB == 2) {
    TabRowsPrep a = tab_rows_prep(c, f.p, true);
    a.g = f.g; a.h = f.h; a.n = c.n; a.gblocks = gblocks; a.block_max = (unsigned *)(c.ws + f.p.block_max);
    tab_rows_launch(c, a, true, true);
    max_q = a.q.blocks; max_w = a.w.blocks;
  } else if (scaled) {
    TabPrep a = {};
    a.g = f.g; a.h = f.h; a.n = c.n; a.q.counts = tab_counts(c, true); a.gblocks = gblocks; a.block_max = (unsigned *)(c.ws + f.p.block_max);
    pbg_launch(tab_max_kernel, dim3(gblocks), 256, 0, c.st, a);
  }
  tab_prepare<T>(c, f.p, true, f.g, f.h, max_q, max_w, gblocks);
  const bool partial = f.p.splits > 1 || f.p.columns < c.rows;
  auto plan = [&](TabArgs &a, bool &pairs, long long M, long long N, int splits) {
    pairs = tab_pairs(M, N);
    a.M = M; a.N = N; a.splits = splits; a.sc = c.sc; a.err = c.err;
    a.BN = tab_columns((M + (pairs ? 255 : 127)) / (pairs ? 256 : 128) * splits, N, pairs ? 2 : 1);
  };
  for (long long v0 = 0; v0 < c.rows && f.ok; v0 += f.p.columns) {
    const long long cols = c.rows - v0 < f.p.columns ? c.rows - v0 : f.p.columns;
    TabOperand w = c.w, w3 = c.w3;
    for (TabOperand *o : {&w, &w3}) { o->base = (const char *)o->base + v0 * o->ld * 2; o->rows = cols; }
    TabArgs g = {};
    bool pairs;
    plan(g, pairs, c.n, cols, 1);
    g.kblocks = (int)((c.dim + KB - 1) / KB);
    g.m_first = 1; g.scale = c.scale;
    g.row_f = (const float *)(c.ws + f.p.row_f); g.col_f = (const float *)(c.ws + f.p.col_f) + v0;
    g.targets = c.targets; g.ignore_index = c.ignore_index; g.vocab = c.rows; g.v0 = v0;
    g.lse = f.lse; g.entropy = f.entropy; g.g = f.g; g.h = f.h;
    g.ldz = f.p.ldz; g.dz_planes = f.p.dz_planes; g.out = c.ws + f.p.dz;
    const TabOperand dz{c.ws + f.p.dz, c.n, cols, f.p.ldz, c.n * f.p.ldz, f.p.dz_planes, true};
    TabOperand written = dz;
    written.inner = f.p.ldz;
    f.ok = tab_launch<EPI_DZ, MATH, false, false>(c.q, w, g, pairs, c.st, &written);
    if (f.dq && f.ok) {
      TabArgs d = {};
      plan(d, pairs, c.n, c.dim, f.p.splits);
      d.kblocks = (int)((cols + KB2 - 1) / KB2);
      d.out = f.dq; d.ldo = c.dim;
      if (partial) { d.partial = (float *)(c.ws + f.p.partial); d.add = v0 > 0; }
      f.ok = tab_launch<EPI_OUT, DZMATH, false, true>(dz, w3, d, pairs, c.st);
    }
    if (f.dt && f.ok) {
      TabArgs d = {};
      plan(d, pairs, cols, c.dim, 1);
      d.kblocks = (int)((c.n + KB2 - 1) / KB2);
      d.by_q = 1;
      d.out = (T *)f.dt + v0 * c.dim; d.ldo = c.dim;
      f.ok = tab_launch<EPI_OUT, DZMATH, true, true>(dz, c.q3, d, pairs, c.st);
    }
  }
  if (f.dq && partial && f.ok) {
    const long long count = c.n * c.dim, blocks = (count + 255) / 256;
    pbg_launch(tab_join_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), 256, 0, c.st, (const float *)(c.ws + f.p.partial), f.p.splits, count, (T *)f.dq);
  }
}

static int tab_check(const TabCall &c, int64_t bytes, bool grad, bool rounded = false) {
  if (c.n < 0 || c.rows <= 0 || c.dim <= 0 || c.q_stride < 0 || c.t_stride < 0 || !tok_type(c.dtype) || !tok_scale(c.scale)) return PBG_ERR_BAD_ARGUMENT;
  if (c.dim > 65536 || c.n > (1ll << 30) || c.rows > 0x7fffffffll - 65536) return PBG_ERR_TOO_LARGE;
  if (c.n == 0) return PBG_OK;
  if (!c.queries || !c.table || !c.targets || !c.ws || ((uintptr_t)c.ws & 255) || bytes < tab_place(c.n, c.rows, c.dim, c.dtype, grad, rounded).bytes) return PBG_ERR_BAD_ARGUMENT;
  // rows that TMA reads where they lie: eight of them, a plane's stride, are less than 2^40 bytes
  if (c.q_stride >= (1ll << 36) || c.t_stride >= (1ll << 36)) return PBG_ERR_TOO_LARGE;
  return PBG_OK;
}

extern "C" int64_t pbg_table_logprobs_workspace(int64_t n, int64_t rows, int32_t dim, int32_t dtype, int32_t grad) {
  if (n <= 0 || rows <= 0 || dim <= 0 || !tok_type(dtype) || n > (1ll << 30) || rows > 0x7fffffffll) return 0;
  return tab_place(n, rows, dim, dtype, grad != 0, grad == 2).bytes;
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
  if (dtype == PBG_F32) tab_forward<float, TabF32>(f);
  else if (dtype == PBG_BF16) tab_forward<__nv_bfloat16, TabBf16>(f);
  else tab_forward<__half, TabF16>(f);
  const int status = tok_status();
  return f.ok ? status : PBG_ERR_CUDA;
}

static int tab_grad(const void *queries, int64_t q_stride, int64_t n, const void *table, int64_t t_stride, int64_t rows, int32_t dim, int32_t dtype,
                    const int64_t *targets, int64_t ignore_index, float scale, const float *lse, const float *entropy, const float *grad_logprob,
                    const float *grad_entropy, void *grad_queries, void *grad_table, void *workspace, int64_t workspace_bytes, int32_t *errors, void *stream, bool rounded) {
  TabBackward f{{queries, q_stride, n, table, t_stride, rows, dim, dtype, (const long long *)targets, ignore_index, scale, (unsigned char *)workspace, errors, (cudaStream_t)stream},
                {}, lse, entropy, grad_logprob, grad_entropy, grad_queries, grad_table, true};
  const int rc = tab_check(f.c, workspace_bytes, true, rounded);
  if (rc != PBG_OK) return rc;
  pbg_launch_error() = cudaSuccess;
  if (n == 0) {
    if (grad_table && cudaMemsetAsync(grad_table, 0, (size_t)rows * dim * tok_size(dtype), f.c.st) != cudaSuccess) pbg_note_launch();
    return tok_status();
  }
  if (!lse || (grad_entropy && !entropy) || (!grad_queries && !grad_table)) return PBG_ERR_BAD_ARGUMENT;
  if (!get_encode()) return PBG_ERR_CUDA;
  f.p = tab_place(n, rows, dim, dtype, true, rounded);
  if (dtype == PBG_F32) tab_backward<float, TabF32, TabF32Out>(f);
  else if (dtype == PBG_BF16) {
    if (f.p.dz_planes == 2) tab_backward<__nv_bfloat16, TabBf16, TabBf16Fine>(f);
    else tab_backward<__nv_bfloat16, TabBf16, TabBf16>(f);
  } else {
    if (f.p.dz_planes == 2) tab_backward<__half, TabF16, TabF16Fine>(f);
    else tab_backward<__half, TabF16, TabF16>(f);
  }
  const int status = tok_status();
  return f.ok ? status : PBG_ERR_CUDA;
}
extern "C" int pbg_table_logprobs_grad(const void *queries, int64_t q_stride, int64_t n, const void *table, int64_t t_stride, int64_t rows, int32_t dim, int32_t dtype,
                                       const int64_t *targets, int64_t ignore_index, float scale, const float *lse, const float *entropy, const float *grad_logprob,
                                       const float *grad_entropy, void *grad_queries, void *grad_table, void *workspace, int64_t workspace_bytes, int32_t *errors, void *stream) {
  return tab_grad(queries, q_stride, n, table, t_stride, rows, dim, dtype, targets, ignore_index, scale, lse, entropy, grad_logprob, grad_entropy, grad_queries, grad_table,
                  workspace, workspace_bytes, errors, stream, false);
}
extern "C" int pbg_table_logprobs_grad_rounded(const void *queries, int64_t q_stride, int64_t n, const void *table, int64_t t_stride, int64_t rows, int32_t dim, int32_t dtype,
                                            const int64_t *targets, int64_t ignore_index, float scale, const float *lse, const float *entropy, const float *grad_logprob,
                                            const float *grad_entropy, void *grad_queries, void *grad_table, void *workspace, int64_t workspace_bytes, int32_t *errors,
                                            void *stream) {
  return tab_grad(queries, q_stride, n, table, t_stride, rows, dim, dtype, targets, ignore_index, scale, lse, entropy, grad_logprob, grad_entropy, grad_queries, grad_table,
                  workspace, workspace_bytes, errors, stream, true);
}
