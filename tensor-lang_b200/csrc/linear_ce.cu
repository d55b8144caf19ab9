// Cross entropy of a linear layer over a large vocabulary, in pieces of the
// vocabulary, without keeping the logits, and its gradients:
//
//   z = x W (+ bias)   lse_r = log sum_v exp z_rv   row_loss_r = lse_r - z_r,t
//   g = (exp(z - lse) - onehot(t)) * upstream / divisor      (rows with a target)
//   dx = g W^T    dW = x^T g    dbias = sum_rows g
//
// It is linear (kernel_generator.py:1584-1661), softmax (:564-640) and
// cross_entropy (:1816-1885) with their VJPs as one operator: unfused, the
// logits and the probabilities, [rows, classes] each, are written and read
// several times, and kept until the backward.
//
// Forward: one matrix product whose epilogue reduces each row of a 256 x 256
// tile of logits, still in registers, to (maximum, sum of exponentials) of 128
// columns; a second kernel joins the columns of a row.  Backward, piece by
// piece of the vocabulary: the same product again, its epilogue turning logits
// into g (bf16 in scratch); then dx += g W^T (float32 in scratch) and dW = x^T g.
// That is 8 x rows x classes x width operations instead of the 6 of an
// unfused step; the two more buy not storing 4 bytes per logit.
//
// The tensor cores bound it: 2048 x 32768 x 4096 bf16, the product with the
// gradients' epilogue 371 us = 1.48 PFLOP/s (0.88 of the library's measured rate),
// tensor pipe active 80%; 8192 x 131072 x 4096 forward and backward 28.3 ms under
// the power cap.  Two CTAs load 64 KB per step of 512 cycles, near what L2 gives;
// the epilogues are hidden behind the next tile.  Few rows are bound by reading W:
// 1 row x 32768 x 4096 60 us, 4.5 TB/s with the launches and the joining counted.
//
// The product kernel computes 256 x 256 tiles by clusters of two CTAs
// (tcgen05.mma.cta_group::2, operands by TMA in the 128-byte swizzle, two
// accumulators of 256 columns in tensor memory), as gemm_tc.cu does for
// float32 operands, and 128 x 128 tiles by single CTAs where x has at most 128
// rows: warp 0 loads, warp 1 of the leading CTA issues the MMAs,
// eight warps drain finished chunks of K into registers and run the epilogue
// while the next chunk or tile is multiplied.  Operands are read in the major
// order they have in memory (K-major or MN-major boxes); nothing is transposed.
// Up to 16 rows of float32 take other kernels (linear_ce_few.cuh).
//
// float32 operands: each is split exactly into three bf16 terms, a = a0 + a1 +
// a2 (8 bits of the significand each), and six of the nine products are kept
// (a0 b0, a0 b1, a1 b0, a1 b1, a0 b2, a2 b0; the others are below 2^-24), each
// a bf16 product over the same K, exact up to its float32 sum.  Within a chunk
// of K the small products come first: the tensor core's accumulator rounds
// toward zero, and only a0 b0's additions meet a sum of full size.  The GEMM's
// two-term scheme (gemm_tc.cu) has half the products and an error of 4e-6;
// here that error would sit in gradients whose own size is a difference, p - 1.
// Against 64 bits the gradients of 2048 x 32000 x 1024 are off by 3.5e-7 (of the
// norm), those of float32 products and sums by 3.2e-6.
//
// g of bf16 operands is held in bf16, unscaled: each element is off by at most
// 2^-8 of itself, so dx and dW are off by at most 2^-8 of the magnitudes that they
// sum, beside their own rounding.  Where one term carries a sum that is as much
// again as the output's rounding; where terms cancel it is that much of the terms.
// Measured against 64 bits, of the norm: 1.7e-3 with g in bf16 and 1.7e-3 with g in
// float32 for 1537 rows and for 8192, 2.0e-3 and 1.7e-3 for few rows.  Two terms of
// g would double the products of dx and dW, half of a training pass.  A caller
// who needs more gives float32 operands.  The scale upstream / divisor is applied in
// float32 afterwards.
#include <math.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "lm_common.cuh"
#include "tc_ptx.cuh"

namespace tl {
namespace {

constexpr int BK = 64;                   // bf16 per stage row: 128 bytes
constexpr int TILE_BYTES = 128 * BK * 2; // 16 KB: 128 rows of A, or of B, per CTA
// The ring of operand stages: six of 32 KB, or more where tiles are narrow or A has
// few rows, so that as many bytes are on their way.
constexpr int RING_BYTES = 6 * 2 * TILE_BYTES;
constexpr int MAX_STAGES = 24;
constexpr int EPI_WARPS = 8;             // two per quarter of the rows
constexpr int CW = 128;                  // columns of an epilogue warp
// Three warpgroups: loads and MMAs (and two idle warps), then the epilogue's two.
// A launch of 384 threads gives each 168 registers; the first group keeps 72 and
// the others take 216 (128 * 72 + 256 * 216 = 384 * 168): an epilogue thread holds
// 128 sums, and with 168 registers it spilled more (2 to 4% slower).  12 to 28 bytes
// a thread still go to local memory in the kGrad and kSum kernels of a K-major A.
constexpr int THREADS = 128 + 32 * EPI_WARPS;
constexpr int kFewRegs = 72, kManyRegs = 216;
constexpr int STG_TILE = 4096;           // per epilogue warp: 32 rows x 128 bytes
constexpr int SMEM_BYTES = RING_BYTES + EPI_WARPS * STG_TILE + 1024 + 512;
constexpr int TMEM_COLS = 512;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

// The six products of two three-term operands, smallest first; one product of
// plain bf16 operands.
constexpr int kTerms = 6;
__device__ __constant__ const signed char kTermA[kTerms] = {2, 1, 0, 1, 0, 0};
__device__ __constant__ const signed char kTermB[kTerms] = {0, 1, 2, 0, 1, 0};

enum Epi { kStats, kGrad, kSum, kOut };

struct TileParams {
  int M, N, K;
  int terms;      // 1, or kTerms
  int kc;         // k-blocks per accumulation chunk
  int splits;     // K split this many ways (kSum)
  int nt;         // columns of a tile: 256, or fewer where that fills the GPU better
  int a_rows;     // rows of A that a CTA loads (K-major A): 128, or all that exist
  int stages;     // of the ring, stage_bytes apart, B's half of a stage at b_at
  int stage_bytes, b_at;
  // kStats, kGrad
  const float* bias;      // of this piece's columns, or null
  const void* target;     // [M], of the whole vocabulary
  int index_type;
  int64_t classes;
  int col0;               // first class of this piece
  float2* part;           // kStats: [slot][part_ld] (maximum, sum of exp)
  int64_t part_ld;
  float* zt;              // kStats: [M] logit of the target
  const float* lse;       // kGrad
  float* colsum;          // kGrad: [M / 32 rounded up][N] sums of g, or null
  int planes;             // kGrad: terms of g (1 or 3)
  float divisor;          // kGrad: an idle warp writes upstream / divisor (0: rows with
  const float* upstream;  // a target) to *scale_out, where that is not null
  float* scale_out;
  // kSum
  int add;                // add to the sums there
  // kOut
  const float* scale;     // one float on the device
  void* out;
  int64_t ldo;
  int out_bf16, accumulate, tma_out;
};

// CG 2: a cluster of two CTAs works on a 256-row tile; CG 1: one CTA on a 128-row
// tile (products of at most 128 rows).  TMA load of a box at (c0, c1, plane),
// completing on `bar` (CG 2: the leader's).
template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                         int c2) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                    uint32_t accumulate) {
  if constexpr (CG == 2)
    mma2_bf16(d_tmem, a_desc, b_desc, idesc, accumulate);
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrive on `bar` (CG 2: in both CTAs) once the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 2)
    mma2_commit_both(bar);
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void sync_ctas() {
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
}

// float32 sums in memory += a staged tile (one addition per element)
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1,
                                           int c2) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];"
      ::"l"((uint64_t)map), "r"(src), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Shared-memory matrix descriptors (128-byte swizzle) of a tile's first 16-deep
// k-step; kStep is what a further one adds.
//   K-major tile: rows of 128 bytes, 8-row groups 1 KB apart; a k-step is 32
//   bytes into the row.
//   MN-major tile: chunks of 64 (M or N) x 64 k, 8 KB apart, a k a row of 128
//   bytes; a k-step is 16 rows = 2 KB.
// The address field counts 16 bytes and stays below its 14 bits (232 KB), so
// stages and k-steps are additions: the issuing thread's loop is short, which
// matters where a step's MMAs are (128 columns: 256 cycles).
template <int MN>
__device__ __forceinline__ uint64_t tile_desc(uint32_t tile) {
  uint64_t d = 0;
  d |= (uint64_t)((tile >> 4) & 0x3FFF);
  d |= (uint64_t)(((MN ? 8192 : 16) >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((1024 >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version for tcgen05
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}
template <int MN>
constexpr uint64_t kStep = (MN ? 2048 : 32) >> 4;
// kind::f16, bf16 operands, float32 accumulator, 128 CG x nt
template <int CG, int A_MN, int B_MN>
__device__ __forceinline__ uint32_t idesc(int nt) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
         ((uint32_t)(nt >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
}

struct Tile {
  int split, m0, n0, kb0, nk;
};
// Tile g: bands of eight M tiles, within a band M fastest (a wave of clusters
// shares a few row blocks of A and of B in L2); splits of K outermost.
template <int TM>
__device__ __forceinline__ Tile tile_of(const TileParams& p, int g) {
  constexpr int kBand = 8;
  const int mt = (p.M + TM - 1) / TM, nt = (p.N + p.nt - 1) / p.nt, nk = (p.K + BK - 1) / BK;
  Tile t;
  t.split = g / (mt * nt);
  const int r = g - t.split * mt * nt;
  const int band = r / (kBand * nt), in = r - band * kBand * nt;
  const int rows = min(kBand, mt - band * kBand);
  t.m0 = (band * kBand + in % rows) * TM;
  t.n0 = in / rows * p.nt;
  t.kb0 = (int)((int64_t)t.split * nk / p.splits);
  t.nk = (int)((int64_t)(t.split + 1) * nk / p.splits) - t.kb0;
  return t;
}

__device__ __forceinline__ float exp_fast(float x) {  // e^x within 2 ulp of 2^(x log2 e)
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// (maximum, sum of exponentials) of two sets of logits
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float M = fmaxf(m, m2), base = M == -INFINITY ? 0.f : M;
  s = s * exp_fast(m - base) + s2 * exp_fast(m2 - base);
  m = M;
}

// bits of two bf16, and what their rounding left over
__device__ __forceinline__ uint32_t take_bf16(float& a, float& b) {
  const uint32_t w = pack2_bf16(a, b);
  a -= __uint_as_float(w << 16);
  b -= __uint_as_float(w & 0xffff0000u);
  return w;
}

// 32 rows (a lane each) x 64 bf16 columns, w[j] holding columns 2j and 2j + 1:
// staged in the tensor map's 128-byte swizzle, stored by TMA.
__device__ __forceinline__ void store_slab16(const CUtensorMap* map, uint32_t stg, int lane,
                                             const uint32_t (&w)[32], int c0, int r0, int plane) {
  if (lane == 0) bulk_wait_read();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                     stg + (uint32_t)lane * 128u + ((uint32_t)(j ^ (lane & 7)) << 4)),
                 "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                 : "memory");
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_3d(map, stg, c0, r0, plane);
    bulk_commit();
  }
}

// 32 rows (a lane each) x 32 columns of float32 through the warp's staging tile,
// element (row, j) at j ^ row: no bank conflicts by rows or by columns.  `lane` is
// hidden from the compiler, which otherwise keeps all 32 addresses in registers
// across the tiles.
__device__ __forceinline__ void stage_slab(float* stage, int lane, const float* v) {
  asm volatile("" : "+r"(lane));
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) stage[lane * 32 + (j ^ lane)] = v[j];
  __syncwarp();
}
__device__ __forceinline__ float staged(const float* stage, int lane, int row) {
  return stage[row * 32 + (lane ^ row)];
}

// Sum over the warp's lanes of column `lane` of their 32 values each: in five
// steps a lane hands over the half of its columns that its partner keeps.
template <int N>
__device__ __forceinline__ float column_sum_of(const float* v, int lane) {
  if constexpr (N == 1) {
    return v[0];
  } else {
    float k[N / 2];
    const bool up = lane & (N / 2);
#pragma unroll
    for (int j = 0; j < N / 2; ++j)
      k[j] = (up ? v[j + N / 2] : v[j]) + __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + N / 2], N / 2);
    return column_sum_of<N / 2>(k, lane);
  }
}
__device__ __forceinline__ float column_sum(const float* v, int lane) { return column_sum_of<32>(v, lane); }

// A: x, g or x^T ...; TA 0: stored [M][K], 1: [K][M].  TB 0: B stored [K][N], 1: [N][K].
template <int CG, int TA, int TB, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    vocab_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmC, const TileParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* staging = smem + RING_BYTES;
  uint64_t* full = (uint64_t*)(staging + EPI_WARPS * STG_TILE);  // [stages] loads of both CTAs -> MMA
  uint64_t* empty = full + MAX_STAGES;                           // [stages] MMA -> each producer
  uint64_t* acc_full = empty + MAX_STAGES;                       // [2] MMA -> each epilogue
  uint64_t* acc_free = acc_full + 2;                             // [2] both epilogues -> MMA
  uint32_t* tmem_slot = (uint32_t*)(acc_free + 2);

  constexpr int TM = 128 * CG;  // rows of a tile
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = p.splits * ((p.M + TM - 1) / TM) * ((p.N + p.nt - 1) / p.nt);
  const int step = (int)gridDim.x / CG, first = (int)blockIdx.x / CG;

  if (threadIdx.x == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmB) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_free[b]), CG * EPI_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(tmem_slot)),
                   "r"(TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(tmem_slot)),
                   "r"(TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  fence_before();
  sync_ctas<CG>();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_previous_kernel();

  // The stage ring (s, with the parity of its turn) and the two accumulators (cg)
  // run on across tiles, so the next tile's loads and MMAs overlap this one's
  // epilogue.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      const uint32_t full0 = CG == 2 ? mapa_shared(smem_u32(&full[0]), 0) : smem_u32(&full[0]);
      bool ok = true;
      int s = 0;
      uint32_t turn = 0;
      for (int g = first; g < tiles && ok; g += step) {
        const Tile t = tile_of<TM>(p, g);
        const int m0 = t.m0 + 128 * (int)rank, n0 = t.n0 + p.nt / CG * (int)rank;
        // rows of A that do not exist are not loaded: their results are not kept,
        // whatever the stage holds there
        const bool have_a = m0 < p.M;
        const uint32_t a_bytes = TA == 0 ? (uint32_t)p.a_rows * 128u : (uint32_t)TILE_BYTES;
        const uint32_t bytes = (CG == 2 && t.m0 + 128 < p.M ? 2u : 1u) * a_bytes + (uint32_t)p.nt * 128u;
        for (int c = 0; c < t.nk && ok; c += p.kc) {
          const int cend = min(c + p.kc, t.nk);
          for (int q = 0; q < p.terms && ok; ++q) {
            const int pa = p.terms == 1 ? 0 : kTermA[q], pb = p.terms == 1 ? 0 : kTermB[q];
            for (int kb = c; kb < cend; ++kb) {
              if (turn > 0 && !mbar_wait(smem_u32(&empty[s]), (turn & 1) ^ 1)) {
                ok = false;
                break;
              }
              const uint32_t sA = smem_u32(smem + s * p.stage_bytes), sB = sA + (uint32_t)p.b_at;
              const uint32_t fb = full0 + 8u * (uint32_t)s;
              if (leader) mbar_expect_tx(smem_u32(&full[s]), bytes);
              const int k0 = (t.kb0 + kb) * BK;
              if (!have_a) {
              } else if constexpr (TA == 0) {
                load_box<CG>(sA, &tmA, fb, k0, m0, pa);
              } else {
                load_box<CG>(sA, &tmA, fb, m0, k0, pa);
                load_box<CG>(sA + 8192, &tmA, fb, m0 + 64, k0, pa);
              }
              if constexpr (TB == 1) {
                load_box<CG>(sB, &tmB, fb, k0, n0, pb);
              } else {
                load_box<CG>(sB, &tmB, fb, n0, k0, pb);
                if (p.nt / CG > 64) load_box<CG>(sB + 8192, &tmB, fb, n0 + 64, k0, pb);
              }
              if (++s == p.stages) {
                s = 0;
                ++turn;
              }
            }
          }
        }
      }
      // gave up: nobody leaves while the stages' last copies are on their way (the
      // leader's barriers count both CTAs'; the wait is bounded)
      bool landed = !ok && leader;
      for (int i = 0; i < p.stages && landed; ++i)
        if (i < s || turn > 0) landed = mbar_wait(smem_u32(&full[i]), (i < s ? turn : turn - 1) & 1);
    }
    if (warp == 1 && leader && lane == 0) {
      // -------------------------------------------------------- MMA (leader)
      const uint32_t id = idesc<CG, TA, 1 - TB>(p.nt);
      const uint64_t a0 = tile_desc<TA>(smem_u32(smem));
      const uint64_t b0 = tile_desc<1 - TB>(smem_u32(smem) + (uint32_t)p.b_at);
      const uint64_t stage16 = (uint64_t)(p.stage_bytes >> 4);
      const uint32_t full_bar = smem_u32(full), empty_bar = smem_u32(empty);
      uint64_t a_desc = a0, b_desc = b0;
      bool ok = true;
      int s = 0;
      uint32_t turn = 0, cg = 0;
      for (int g = first; g < tiles && ok; g += step) {
        const Tile t = tile_of<TM>(p, g);
        for (int c = 0; c < t.nk && ok; c += p.kc, ++cg) {
          const int n = (min(c + p.kc, t.nk) - c) * p.terms;
          const uint32_t b = cg & 1, acc = tmem + b * 256;
          if (cg >= 2 && !mbar_wait(smem_u32(&acc_free[b]), ((cg >> 1) - 1) & 1)) {
            ok = false;
            break;
          }
          fence_after();
          for (int i = 0; i < n; ++i) {
            if (!mbar_wait(full_bar + 8u * (uint32_t)s, turn & 1)) {
              ok = false;
              break;
            }
            fence_after();
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              mma<CG>(acc, a_desc + k * kStep<TA>, b_desc + k * kStep<1 - TB>, id,
                      (i == 0 && k == 0) ? 0u : 1u);
            commit<CG>(empty_bar + 8u * (uint32_t)s);
            a_desc += stage16;
            b_desc += stage16;
            if (++s == p.stages) {
              s = 0;
              ++turn;
              a_desc = a0;
              b_desc = b0;
            }
          }
          commit<CG>(smem_u32(&acc_full[b]));
        }
      }
    }
    if (EPI == kGrad && warp == 2 && blockIdx.x == 0 && p.scale_out) {
      int n = 0;
#pragma unroll 4
      for (int i = lane; i < p.M; i += 32) n += class_index(p.target, p.index_type, i, p.classes) >= 0;
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0)
        *p.scale_out = (p.upstream ? *p.upstream : 1.f) / (p.divisor > 0.f ? p.divisor : fmaxf(1.f, (float)n));
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
    // ----------------------------------------------------------- epilogue
    const int e = warp - 4, quarter = warp & 3, group = e >> 2;
    const uint32_t free0 = CG == 2 ? mapa_shared(smem_u32(&acc_free[0]), 0) : smem_u32(&acc_free[0]);
    const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(group * CW);
    float* stage = reinterpret_cast<float*>(staging + e * STG_TILE);
    const uint32_t stg = smem_u32(stage);
    float v[CW];
    float2 row_stats = make_float2(-INFINITY, 0.f);  // kStats, CG 1: of this CTA's tiles
    bool ok = true;
    uint32_t cg = 0;
    for (int g = first; g < tiles && ok; g += step) {
      const Tile t = tile_of<TM>(p, g);
#pragma unroll
      for (int j = 0; j < CW; ++j) v[j] = 0.f;
      for (int c = 0; c < t.nk; c += p.kc, ++cg) {
        const uint32_t b = cg & 1;
        if (!mbar_wait(smem_u32(&acc_full[b]), (cg >> 1) & 1)) {
          ok = false;
          break;
        }
        fence_after();
        __syncwarp();
#pragma unroll
        for (int q = 0; q < CW / 16; ++q) {
          float r[16];
          tmem_ld16(tbase + b * 256 + q * 16, r);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[q * 16 + j] += r[j];
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2)
            mbar_arrive_cluster(free0 + 8u * b);
          else
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(free0 + 8u * b) : "memory");
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int r0 = t.m0 + 128 * (int)rank + quarter * 32, row = r0 + lane;
      const int n0 = t.n0 + group * CW;
      const int cols = min(min(CW, p.nt - group * CW), p.N - n0);  // of this warp; may be <= 0
      if (r0 >= p.M || cols <= 0) continue;
      const bool live = row < p.M;

      if constexpr (EPI == kStats || EPI == kGrad) {
        if (p.bias) {
          const float* b = p.bias + n0;
          if (cols == CW && ((uintptr_t)b & 15) == 0) {
#pragma unroll
            for (int j = 0; j < CW; j += 4) {
              const float4 q = __ldg(reinterpret_cast<const float4*>(b + j));
              v[j] += q.x; v[j + 1] += q.y; v[j + 2] += q.z; v[j + 3] += q.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < CW; ++j)
              if (j < cols) v[j] += __ldg(b + j);
          }
        }
        const int cls = live ? (int)class_index(p.target, p.index_type, row, p.classes) : -1;
        const int target = cls < 0 ? -1 : cls - p.col0 - n0;  // in this warp's columns
        if constexpr (EPI == kStats) {
          if (cols < CW) {
#pragma unroll
            for (int j = 0; j < CW; ++j)
              if (j >= cols) v[j] = -INFINITY;
          }
          float m = v[0];
#pragma unroll
          for (int j = 1; j < CW; ++j) m = fmaxf(m, v[j]);
          const float base = m == -INFINITY ? 0.f : m;
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < CW; ++j) s += exp_fast(v[j] - base);
          if constexpr (CG == 1)
            join(row_stats.x, row_stats.y, m, s);
          if (live) {
            if constexpr (CG == 2)
              p.part[(int64_t)(t.n0 / p.nt * (p.nt > CW ? 2 : 1) + group) * p.part_ld + row] = make_float2(m, s);
            if (target >= 0 && target < cols) {
              float z = 0.f;
#pragma unroll
              for (int j = 0; j < CW; ++j) z = j == target ? v[j] : z;
              p.zt[row] = z;
            }
          }
        } else {
          // g = p - onehot; 0 for rows without a target
          const bool counts = cls >= 0;
          const float lse = counts ? p.lse[row] : INFINITY;
          // nothing left of the row: p = 0, as for the rows that do not count
          const float off = lse == -INFINITY ? INFINITY : lse;
          float* cs = p.colsum ? p.colsum + (int64_t)(r0 >> 5) * p.N + n0 : nullptr;
#pragma unroll
          for (int sl = 0; sl < CW / 64; ++sl) {  // one slab after the other: registers
            if (64 * sl >= cols) break;
            float* u = v + 64 * sl;
#pragma unroll
            for (int j = 0; j < 64; ++j) u[j] = exp_fast(u[j] - off);
            if (!counts) {  // a NaN or infinite logit included
#pragma unroll
              for (int j = 0; j < 64; ++j) u[j] = 0.f;
            }
            if (target >= 64 * sl && target < min(cols, 64 * sl + 64)) {
#pragma unroll
              for (int j = 0; j < 64; ++j) u[j] -= j == target - 64 * sl ? 1.f : 0.f;
            }
            if (cs) {  // before g is rounded
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float s = column_sum(u + 32 * h, lane);
                const int c = 64 * sl + 32 * h + lane;
                if (c < cols) cs[c] = s;
                asm volatile("" ::: "memory");
              }
            }
            for (int pl = 0; pl < p.planes; ++pl) {
              uint32_t w[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = take_bf16(u[2 * j], u[2 * j + 1]);
              store_slab16(&tmC, stg, lane, w, n0 + 64 * sl, r0, pl);
            }
            asm volatile("" ::: "memory");
          }
        }
      } else if constexpr (EPI == kSum) {
#pragma unroll
        for (int sl = 0; sl < CW / 32; ++sl) {
          if (32 * sl >= cols) break;
          if (lane == 0) bulk_wait_read();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            st_shared_v4(stg + (uint32_t)lane * 128u + ((uint32_t)(j ^ (lane & 7)) << 4), v[32 * sl + 4 * j],
                         v[32 * sl + 4 * j + 1], v[32 * sl + 4 * j + 2], v[32 * sl + 4 * j + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (p.add)
              tma_add_3d(&tmC, stg, n0 + 32 * sl, r0, t.split);
            else
              tma_store_3d(&tmC, stg, n0 + 32 * sl, r0, t.split);
            bulk_commit();
          }
        }
      } else {
        const float scale = *p.scale;
        if (p.tma_out) {
          if (p.out_bf16) {
#pragma unroll
            for (int sl = 0; sl < CW / 64; ++sl) {
              if (64 * sl >= cols) break;
              uint32_t w[32];
#pragma unroll
              for (int j = 0; j < 32; ++j)
                w[j] = pack2_bf16(scale * v[64 * sl + 2 * j], scale * v[64 * sl + 2 * j + 1]);
              store_slab16(&tmC, stg, lane, w, n0 + 64 * sl, r0, 0);
              asm volatile("" ::: "memory");
            }
          } else {
#pragma unroll
            for (int sl = 0; sl < CW / 32; ++sl) {
              if (32 * sl >= cols) break;
              uint32_t w[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(scale * v[32 * sl + j]);
              store_slab16(&tmC, stg, lane, w, n0 + 32 * sl, r0, 0);
              asm volatile("" ::: "memory");
            }
          }
        } else {
          // any alignment, or adding to what is there: through shared memory,
          // a row's 32 columns per access
#pragma unroll
          for (int sl = 0; sl < CW / 32; ++sl) {
            if (32 * sl >= cols) break;
            stage_slab(stage, lane, v + 32 * sl);
            const int c = 32 * sl + lane, rows = min(32, p.M - r0);
            if (c >= cols) continue;
            const int64_t at = (int64_t)r0 * p.ldo + n0 + c;
#pragma unroll 4
            for (int r = 0; r < rows; ++r) {
              const float q = scale * staged(stage, lane, r);
              if (p.out_bf16) {
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + at + r * p.ldo;
                *o = __float2bfloat16_rn(p.accumulate ? __bfloat162float(*o) + q : q);
              } else {
                float* o = static_cast<float*>(p.out) + at + r * p.ldo;
                *o = p.accumulate ? *o + q : q;
              }
            }
          }
        }
      }
    }
    if constexpr (EPI == kStats && CG == 1) {  // every tile has all rows: one partial per CTA
      if (group == 0 && quarter * 32 + lane < p.M)
        p.part[(int64_t)blockIdx.x * p.part_ld + quarter * 32 + lane] = row_stats;
    }
    if (lane == 0) bulk_wait_all();  // the staging outlives every TMA store's read
    __syncwarp();
  }
  fence_before();
  sync_ctas<CG>();  // neither CTA frees tensor memory or exits while the pair works
  if (warp == 1) {
    fence_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS)
                   : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS)
                   : "memory");
  }
}

// Scratch words before the arrays; joined (blocks done) is zero between calls.
struct Head {
  unsigned joined;
  float scale;  // backward: upstream / divisor
};

struct Targets {
  const void* p;
  int type;
  int64_t rows, classes;
  __device__ __forceinline__ int64_t at(int64_t r) const { return class_index(p, type, r, classes); }
};

// Rows with a target, by one block; every thread gets the count.
__device__ __forceinline__ int64_t count_targets(const Targets& t, long long* sh) {
  long long n = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < t.rows; i += blockDim.x) n += t.at(i) >= 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (unsigned i = 0; i < blockDim.x / 32; ++i) n += sh[i];
  return n;
}

// Joins a piece's partials of R rows per block, NT / R threads a row; the last
// piece writes lse and the losses, and the last block the mean (the only block:
// from its own rows' losses, without a ticket).
template <int R, int NT>
__global__ void __launch_bounds__(NT) join_kernel(const float2* part, int64_t part_ld, int slots,
                                                   Targets target, const float* zt, float2* run,
                                                   int first, int last, float divisor,
                                                   float* row_loss, float* lse, float* loss,
                                                   Head* head) {
  constexpr int L = NT / R, NW = NT / 32;
  __shared__ float2 sh[L][R + 1];
  __shared__ unsigned ticket;
  __shared__ long long shn[NW];
  __shared__ double shd[NW];
  wait_for_previous_kernel();
  const int r = threadIdx.x % R, l = threadIdx.x / R;
  const int64_t row = (int64_t)blockIdx.x * R + r, rows = target.rows;
  const bool writes = l == 0 && row < rows;
  const bool counts = writes && last && target.at(row) >= 0;
  const float z = counts ? zt[row] : 0.f;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
    const float2* q = part + row;
    int i = l;
    constexpr int K = NT == 256 ? 4 : 8;  // loads on their way
    for (; i + (K - 1) * L < slots; i += K * L) {
      float2 v[K];
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = __ldcs(q + (int64_t)(i + k * L) * part_ld);
      float M = m;
#pragma unroll
      for (int k = 0; k < K; ++k) M = fmaxf(M, v[k].x);
      const float base = M == -INFINITY ? 0.f : M;
      s *= exp_fast(m - base);
#pragma unroll
      for (int k = 0; k < K; ++k) s += v[k].y * exp_fast(v[k].x - base);
      m = M;
    }
#pragma unroll 2
    for (; i < slots; i += L) {
      const float2 v = __ldcs(q + (int64_t)i * part_ld);
      join(m, s, v.x, v.y);
    }
  }
  sh[l][r] = make_float2(m, s);
  for (int h = L / 2; h > 0; h >>= 1) {
    __syncthreads();
    if (l < h) {
      join(m, s, sh[l + h][r].x, sh[l + h][r].y);
      sh[l][r] = make_float2(m, s);
    }
  }
  float row_v = 0.f;
  if (writes) {
    if (!first) join(m, s, run[row].x, run[row].y);
    if (!last) {
      run[row] = make_float2(m, s);
    } else {
      const float log_s = logf(s);  // a row of -inf: -inf
      if (lse) lse[row] = m + log_s;
      // (m - z) + log s: lse - z would round lse first
      if (counts) row_v = z == -INFINITY ? INFINITY : (m - z) + log_s;
      row_loss[row] = row_v;
    }
  }
  if (!last || !loss) return;
  if (gridDim.x == 1) {
    const double own = warp_sum((double)row_v);
    if ((threadIdx.x & 31) == 0) shd[threadIdx.x >> 5] = own;
    const int n = __syncthreads_count(counts);
    if (threadIdx.x == 0) {
      double t = 0.0;
      for (int i = 0; i < (R + 31) / 32; ++i) t += shd[i];  // the warps with l == 0
      *loss = (float)(t / (double)(divisor > 0.f ? divisor : fmaxf(1.f, (float)n)));
    }
    return;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) ticket = atomicAdd(&head->joined, 1u);
  __syncthreads();
  if (ticket != gridDim.x - 1) return;
  __threadfence();
  double t = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < rows; i += NT) t += (double)__ldcg(row_loss + i);
  t = warp_sum(t);
  if ((threadIdx.x & 31) == 0) shd[threadIdx.x >> 5] = t;
  const int64_t n = divisor > 0.f ? 1 : count_targets(target, shn);
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.0;
    for (int i = 0; i < NW; ++i) t += shd[i];
    const float d = divisor > 0.f ? divisor : fmaxf(1.f, (float)n);
    *loss = (float)(t / (double)d);
    head->joined = 0u;
  }
}

}  // namespace
}  // namespace tl

#include "linear_ce_few.cuh"

namespace tl {
namespace {

// Eight elements of a row from any element offset, those past `left` zero.
__device__ __forceinline__ void load8(const float* p, int64_t left, float (&v)[8]) {
  if (left >= 8 && ((uintptr_t)p & 15) == 0) {
    const float4 a = ld_stream4(p), b = ld_stream4(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int64_t left, float (&v)[8]) {
  if (left >= 9) {  // words of two; where p lies between words, up to element 8
    const uint32_t* q = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
    const bool odd = ((uintptr_t)p & 2) != 0;
    uint32_t w[5];
    w[0] = odd ? (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16 : __ldg(q);
#pragma unroll
    for (int i = 1; i < 4; ++i) w[i] = __ldg(q + i);
    w[4] = odd ? __ldg(q + 4) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = odd ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
      v[2 * i] = __uint_as_float(x << 16);
      v[2 * i + 1] = __uint_as_float(x & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? __bfloat162float(p[i]) : 0.f;
  }
}

// The terms of a matrix as bf16 planes [planes][rows][ld], columns past `cols`
// zero: three that sum to a float32 matrix exactly, or a copy of a bf16 one
// whose rows TMA cannot address.  ld is a multiple of 8.  Rows without a target
// (where keep.p is not null) come out as zeros.
template <typename T, typename Index>
__global__ void __launch_bounds__(256) planes_kernel(const T* __restrict__ X, int64_t ldx, int64_t rows,
                                                     int64_t cols, int planes,
                                                     __nv_bfloat16* __restrict__ out, int64_t ld,
                                                     const Targets keep) {
  wait_for_previous_kernel();
  const int64_t plane = rows * ld;
  const Index vecs = (Index)(ld / 8), n = (Index)rows * vecs, step = (Index)gridDim.x * 256;
  for (Index i = (Index)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const Index r = i / vecs;
    const int64_t c = 8 * (int64_t)(i - r * vecs);
    float v[8];
    const bool kept = !keep.p || keep.at((int64_t)r) >= 0;
    load8(X + (int64_t)r * ldx + c, kept ? cols - c : 0, v);
    __nv_bfloat16* dst = out + (int64_t)r * ld + c;
    for (int p = 0; p < planes; ++p)
      *reinterpret_cast<uint4*>(dst + p * plane) =
          make_uint4(take_bf16(v[0], v[1]), take_bf16(v[2], v[3]), take_bf16(v[4], v[5]),
                     take_bf16(v[6], v[7]));
  }
}

// dx = scale * (sum of the splits' sums) (+ dx); a block a row, four columns a
// thread (ld is a multiple of 4).
template <typename T>
__global__ void __launch_bounds__(256) dx_kernel(const float* __restrict__ sums, int splits, int64_t rows,
                                                 int64_t cols, int64_t ld, const float* scale, T* dx,
                                                 int64_t lddx, int accumulate) {
  wait_for_previous_kernel();
  const float k = *scale;
  const bool vec = cols % 4 == 0 && lddx % 4 == 0 && ((uintptr_t)dx & 15) == 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    T* o = dx + r * lddx;
    for (int64_t c = 4 * (int64_t)threadIdx.x; c < cols; c += 1024) {
      float4 s = __ldcs(reinterpret_cast<const float4*>(sums + r * ld + c));
      for (int p = 1; p < splits; ++p) {
        const float4 q = __ldcs(reinterpret_cast<const float4*>(sums + ((int64_t)p * rows + r) * ld + c));
        s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
      }
      float v[4] = {k * s.x, k * s.y, k * s.z, k * s.w};
      const int n = (int)min((int64_t)4, cols - c);
      if (accumulate) {
        for (int i = 0; i < n; ++i) v[i] += to_f32(o[c + i]);
      }
      if (vec) {
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<float4*>(o + c) = make_float4(v[0], v[1], v[2], v[3]);
        else
          *reinterpret_cast<uint2*>(o + c) = make_uint2(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) from_f32(o + c + i, v[i]);
      }
    }
  }
}

// dbias of a piece: the row groups' column sums in order, four chains.
__global__ void __launch_bounds__(256) dbias_kernel(const float* __restrict__ colsum, int64_t groups,
                                                    int64_t cols, const float* scale, float* dbias,
                                                    int accumulate) {
  __shared__ float sh[8][33];
  wait_for_previous_kernel();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (int64_t g = w; g < groups; g += 8) s += colsum[g * cols + c];
  sh[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) s += sh[i][lane];
    dbias[c] = (accumulate ? dbias[c] : 0.f) + *scale * s;
  }
}

// ------------------------------------------------------------- host side ---
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeTiled)f;
  }();
  return fn;
}

// [planes][rows][cols] with row stride ld and plane stride rows * ld, boxes of
// box_c x box_r x 1 in the 128-byte swizzle.
bool make_map3(CUtensorMap* m, const void* base, bool f32, int64_t planes, int64_t rows, int64_t cols,
               int64_t ld, uint32_t box_c, uint32_t box_r) {
  const EncodeTiled enc = encode_tiled();
  if (!enc) return false;
  const int64_t es = f32 ? 4 : 2;
  // a single row or plane is never stepped over, but strides must be multiples of 16
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * es), (cuuint64_t)(rows * ld * es)};
  const cuuint32_t box[3] = {box_c, box_r, 1}, one[3] = {1, 1, 1};
  return enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int64_t up_to(int64_t n, int64_t k) { return (n + k - 1) / k * k; }

// An operand in memory that TMA can address: bf16 planes.
struct Planes {
  const __nv_bfloat16* p;
  int64_t planes, rows, cols, ld;
};
// as the K-major operand (stored [MN][K]) or the MN-major one ([K][MN])
bool k_major(CUtensorMap* m, const Planes& x, int box_rows) {
  return make_map3(m, x.p, false, x.planes, x.rows, x.cols, x.ld, 64, (uint32_t)box_rows);
}
bool mn_major(CUtensorMap* m, const Planes& x) {
  return make_map3(m, x.p, false, x.planes, x.rows, x.cols, x.ld, 64, 64);
}

// Whether a product's tiles are one CTA's: A's rows fit one (K-major A).
bool one_cta(int64_t M) { return M <= 128; }

// Columns of a tile: 256 (one CTA: 128), except
//  - where half-size tiles still fit one wave: the narrowest that do (steps are
//    what the epilogue's slabs and B's boxes allow);
//  - between one and four waves of a K-major B: fewer where that ends sooner (a
//    wave costs its tiles' columns and a fixed part worth about 32).  A training pass,
//    with this and with 256 columns, us: 256 x 19456 x 4096 235 and 242, 256 x 38000 x
//    2048 210 and 217, 1537 x 50021 x 1000 690 and 705 (dx); scoring by pairs is
//    bound by memory and gains nothing (200 x 32768 x 4096 65.2 and 65.0).
//    An MN-major B's boxes are 64 columns of 128 bytes: scoring 200 x 65536 x 2048
//    takes 98 us with 128-column tiles of CTA pairs, 71 with 256.
//    Tiles of one CTA gain nothing (1 token: 112 columns 60.9 us, 128 60.2): their
//    loads share the memory's rate, so a wave with fewer tiles ends sooner anyway.
template <int EPI>
int tile_columns(int64_t M, int64_t N, int splits, bool b_mn_major, bool one) {
  const int wide = one ? 128 : 256;
  const int64_t slots = std::max(1, one ? sm_count() : sm_count() / 2);
  const int64_t mt = (one ? (M + 127) / 128 : (M + 255) / 256) * splits;
  const int64_t tiles = mt * ((N + wide - 1) / wide);
  if (tiles >= 4 * slots) return wide;
  const int step = b_mn_major ? wide / 2 : EPI == kStats ? (one ? 16 : 32) : EPI == kSum ? 32 : 64;
  if (2 * tiles <= slots) {
    for (int nt = std::max(step, 64); nt < wide; nt += step)
      if (mt * ((N + nt - 1) / nt) <= slots) return nt;
    return wide;
  }
  if (b_mn_major || one) return wide;
  int best = wide;
  int64_t cost = INT64_MAX;
  for (int nt = wide; nt >= wide / 4 * 3; nt -= step) {
    const int64_t waves = (mt * ((N + nt - 1) / nt) + slots - 1) / slots, c = waves * (nt + 32);
    if (c < cost) {
      cost = c;
      best = nt;
    }
  }
  return best;
}

template <int CG, int TA, int TB, int EPI>
int launch_tiles_of(const Planes& A, const Planes& B, const CUtensorMap& c, TileParams p, cudaStream_t st) {
  constexpr auto kern = vocab_tile_kernel<CG, TA, TB, EPI>;
  TL_TRY((allow_smem<kern, SMEM_BYTES>()));
  constexpr int TM = 128 * CG;
  p.nt = tile_columns<EPI>(p.M, p.N, p.splits, TB == 0, CG == 1);
  p.a_rows = TA == 0 ? (int)std::min<int64_t>(128, up_to(p.M, 8)) : 128;
  // the MMA reads 128 rows of A from a stage's start: past the loaded ones what
  // follows in shared memory, whose products are not kept
  p.b_at = p.a_rows * 128;
  p.stage_bytes = p.b_at + p.nt / CG * 128;
  p.stages = std::min(MAX_STAGES, RING_BYTES / p.stage_bytes);
  CUtensorMap a, b;
  if (!(TA == 0 ? k_major(&a, A, p.a_rows) : mn_major(&a, A)) ||
      !(TB == 1 ? k_major(&b, B, p.nt / CG) : mn_major(&b, B)))
    return TL_ERR_UNSUPPORTED;
  const int64_t tiles = (int64_t)p.splits * ((p.M + TM - 1) / TM) * ((p.N + p.nt - 1) / p.nt);
  if (tiles > INT32_MAX / 2) return TL_ERR_UNSUPPORTED;
  const int64_t slots = std::max(1, sm_count() / CG);
  return launch_in_clusters(CG, kern, dim3((unsigned)(CG * std::min(tiles, slots))), THREADS, SMEM_BYTES, st, a,
                            b, c, p);
}
template <int TA, int TB, int EPI>
int launch_tiles(const Planes& A, const Planes& B, const CUtensorMap& c, const TileParams& p,
                 cudaStream_t st) {
  if constexpr (TA == 0) {
    if (one_cta(p.M)) return launch_tiles_of<1, TA, TB, EPI>(A, B, c, p, st);
  }
  return launch_tiles_of<2, TA, TB, EPI>(A, B, c, p, st);
}

// The partials a product of kStats leaves per row: one for each epilogue warp's
// columns, none for columns that do not exist; tiles of one CTA: one for each CTA.
int stat_slots(int64_t M, int64_t N, bool b_mn_major) {
  const int nt = tile_columns<kStats>(M, N, 1, b_mn_major, one_cta(M));
  if (one_cta(M)) return (int)std::min<int64_t>((N + nt - 1) / nt, std::max(1, sm_count()));
  const int64_t before = (N - 1) / nt;
  return (int)(before * (nt > CW ? 2 : 1) + (N - before * nt > CW ? 2 : 1));
}

struct Call {
  int dtype, trans_w, index_type;
  int64_t rows, classes, width;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  const float* bias;
  const void* target;
  float divisor;
  char* scratch;
  cudaStream_t st;
  Targets targets() const { return {target, index_type, rows, classes}; }
  bool f32() const { return dtype == TL_F32; }
  int planes() const { return f32() ? 3 : 1; }
  int terms() const { return f32() ? kTerms : 1; }
  // chunks of K per accumulator: 1024 deep, or 256 (x 6 products)
  int kc() const { return f32() ? 4 : 16; }
};

// Few rows of float32: W as it is (linear_ce_few.cuh, with the figures).
bool few(int dtype, int64_t rows, int64_t classes, int64_t width) {
  constexpr int64_t kMost = 1 << 22;  // of the grids' second dimension, and the kept logits
  return dtype == TL_F32 && rows <= kFewRows && classes <= kMost && width <= kMost;
}

// How a call is cut: classes per piece, and where its arrays are in scratch.
struct Plan {
  int64_t fpiece, bpiece;          // classes per piece, forward and backward
  int64_t dpiece;                  // the forward's where W is read where it is
  int64_t part_ld;                 // rows of the forward's partials
  int splits;                      // of K in dx
  int64_t xplanes, wplanes, zt, run, row_loss, part, g, sums, colsum, total;  // offsets
  // few rows: logits and g [rows][zld], the logits in zsplits sums
  bool few;
  int zsplits;
  int64_t z, zld;
};

// splits of K that let few tiles of dx fill the GPU: whole waves of clusters
int dx_splits(int64_t rows, int64_t width, int64_t piece) {
  const bool one = one_cta(rows);
  const int64_t tiles = one ? (width + 127) / 128 : ((rows + 255) / 256) * ((width + 255) / 256);
  const int64_t slots = std::max(1, one ? sm_count() : sm_count() / 2), nk = piece / BK;
  int best = 1;
  double eff = 0;
  for (int s = 1; s <= 16 && (s == 1 || nk / s >= 8); ++s) {
    const int64_t n = tiles * s, waves = (n + slots - 1) / slots;
    const double f = (double)n / (double)(waves * slots);
    if (f > eff + 0.02) {
      eff = f;
      best = s;
    }
    if (n >= 4 * slots) break;
  }
  return best;
}

Plan make_plan(int dtype, int trans_w, int64_t rows, int64_t classes, int64_t width, bool backward) {
  Plan q{};
  const int64_t P = dtype == TL_F32 ? 3 : 1, all = up_to(classes, 256);
  auto piece = [&](int64_t bytes_per_class, int64_t cap) {
    return std::min<int64_t>(all, std::max<int64_t>(256, cap / std::max<int64_t>(1, bytes_per_class) / 256 * 256));
  };
  q.part_ld = up_to(rows, 32);
  const int64_t cap = 512LL << 20;
  // the partials (8 bytes per row and 128 classes) and the terms of W
  q.dpiece = piece(q.part_ld * 8 / CW, cap);
  q.fpiece = std::min(q.dpiece, piece(width * 2 * P, cap));
  q.bpiece = std::min(piece(rows * 2 * P, cap), piece(width * 2 * P, cap));
  q.splits = backward ? dx_splits(rows, width, q.bpiece) : 1;
  int64_t at = 1024;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at = up_to(at + bytes, 1024);
    return o;
  };
  q.few = few(dtype, rows, classes, width);
  if (q.few) {
    q.zsplits = trans_w ? rowdot_splits(classes, width) : coldot_splits(width, classes);
    q.splits = trans_w ? coldot_splits(classes, width) : rowdot_splits(width, classes);
    q.zld = up_to(classes, 32);
    q.zt = take(rows * 4);
    q.row_loss = take(rows * 4);
    q.part = take(kStatBlocks * q.part_ld * 8);
    q.z = take((int64_t)q.zsplits * rows * q.zld * 4);
    q.g = take(backward ? rows * q.zld * 4 : 0);
    q.sums = take(backward ? (int64_t)q.splits * rows * up_to(width, 4) * 4 : 0);
    q.total = at;
    return q;
  }
  q.xplanes = take(P * rows * up_to(width, 64) * 2);
  const int64_t wp = backward ? std::max(q.fpiece, q.bpiece) : q.fpiece;
  q.wplanes = take(P * (trans_w ? wp * up_to(width, 64) : width * up_to(wp, 64)) * 2);
  const int64_t common = at;
  q.zt = take(rows * 4);
  q.run = take(rows * 8);
  q.row_loss = take(rows * 4);
  // two per tile: of 256 columns, or of at least 64 where there are few tiles
  // (tile_columns: less than 2 * sm_count() of 256)
  const int64_t few = 16 * std::max(1, sm_count()) / ((rows + 255) / 256) + 8;
  q.part = take((q.dpiece / CW + few) * q.part_ld * 8);
  q.total = at;
  if (backward) {
    at = common;
    q.g = take(P * rows * q.bpiece * 2);
    q.sums = take((int64_t)q.splits * rows * up_to(width, 4) * 4);
    q.colsum = take(up_to(rows, 32) / 32 * q.bpiece * 4);
    q.total = std::max(q.total, at);
  }
  return q;
}

template <typename T>
int write_planes(const T* X, int64_t ldx, int64_t rows, int64_t cols, int planes, __nv_bfloat16* out,
                 int64_t ld, const Targets& keep, cudaStream_t st) {
  const int64_t vecs = rows * (ld / 8);
  const dim3 grid((unsigned)std::min<int64_t>((vecs + 255) / 256, 32LL * sm_count()));
  // the index steps past the end by at most the grid's threads
  return vecs < (1LL << 31)
             ? launch(planes_kernel<T, uint32_t>, grid, 256, 0, st, X, ldx, rows, cols, planes, out, ld, keep)
             : launch(planes_kernel<T, uint64_t>, grid, 256, 0, st, X, ldx, rows, cols, planes, out, ld, keep);
}

// Whether TMA can address a matrix of the call's type as it is.
bool direct(const Call& c, const void* X, int64_t ldx) {
  return !c.f32() && ldx % 8 == 0 && aligned_to(X, 16);
}

// rows x cols of X as planes: itself where TMA can address it, else (or with
// `copy`) a copy, without the rows that `keep` names no class for.  A copy's rows
// start at multiples of 128 bytes: a box's rows of 128 bytes then are one cache
// line each, not two.
int as_planes(const Call& c, const void* X, int64_t ldx, int64_t rows, int64_t cols, int64_t scratch_at,
              bool copy, const Targets& keep, Planes* out) {
  if (!copy && direct(c, X, ldx)) {
    *out = {static_cast<const __nv_bfloat16*>(X), 1, rows, cols, ldx};
    return TL_OK;
  }
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(c.scratch + scratch_at);
  *out = {dst, c.planes(), rows, cols, up_to(cols, 64)};
  if (c.f32())
    return write_planes(static_cast<const float*>(X), ldx, rows, cols, 3, dst, out->ld, keep, c.st);
  return write_planes(static_cast<const __nv_bfloat16*>(X), ldx, rows, cols, 1, dst, out->ld, keep, c.st);
}

// classes c0 .. c0 + n of W
int w_planes(const Call& c, const Plan& q, int64_t c0, int64_t n, Planes* out) {
  const int64_t es = (int64_t)elem_bytes(c.dtype);
  const char* w = static_cast<const char*>(c.w) + (c.trans_w ? c0 * c.ldw : c0) * es;
  return c.trans_w ? as_planes(c, w, c.ldw, n, c.width, q.wplanes, false, Targets{}, out)
                   : as_planes(c, w, c.ldw, c.width, n, q.wplanes, false, Targets{}, out);
}
// x, read by every tile: a copy where its rows straddle cache lines, and rows and
// classes are many enough for that to pay (as it is and copied, width 1000, us:
// 4000 rows x 32000 classes 214 and 205; a training pass's products of 1537 x 50021
// 142 and 136, 170 and 159; 4000 x 6000 66.3 and 67.5, 5000 x 600 118 and 136; near
// the limits either is within 4%: 2000 x 8200 41.7 and 43.3, 400 x 50021 58.6 and 56.8).  For dW a copy always, with zeros in the rows without a target: their
// g is 0, but 0 times an infinity or NaN in a padded row is NaN in all of dW.
int x_planes(const Call& c, const Plan& q, bool for_dw, Planes* out) {
  const bool straddles = c.ldx % 64 || !aligned_to(c.x, 128);
  return as_planes(c, c.x, c.ldx, c.rows, c.width, q.xplanes,
                   for_dw || (straddles && c.rows >= 512 && c.classes >= 8192),
                   for_dw ? c.targets() : Targets{}, out);
}

// The logits' product over classes c0 .. c0 + n, with epilogue EPI.
template <int EPI>
int logits(const Call& c, const Planes& x, const Planes& w, const CUtensorMap& out, TileParams p,
           int64_t c0, int64_t n) {
  p.M = (int)c.rows;
  p.N = (int)n;
  p.K = (int)c.width;
  p.terms = c.terms();
  p.kc = c.kc();
  p.splits = 1;
  p.bias = c.bias ? c.bias + c0 : nullptr;
  p.target = c.target;
  p.index_type = c.index_type;
  p.classes = c.classes;
  p.col0 = (int)c0;
  return c.trans_w ? launch_tiles<0, 1, EPI>(x, w, out, p, c.st)
                   : launch_tiles<0, 0, EPI>(x, w, out, p, c.st);
}

// z [split][rows][zld] = x W, without the bias
int few_logits(const Call& c, const Plan& q) {
  float* z = reinterpret_cast<float*>(c.scratch + q.z);
  const float *x = static_cast<const float*>(c.x), *w = static_cast<const float*>(c.w);
  return c.trans_w ? few_product(true, w, c.ldw, c.classes, c.width, x, c.ldx, c.rows, z, q.zld, c.st)
                   : few_product(false, w, c.ldw, c.width, c.classes, x, c.ldx, c.rows, z, q.zld, c.st);
}

int few_forward(const Call& c, const Plan& q, float* loss, float* row_loss, float* lse) {
  TL_TRY(few_logits(c, q));
  float2* part = reinterpret_cast<float2*>(c.scratch + q.part);
  float* zt = reinterpret_cast<float*>(c.scratch + q.zt);
  if (!row_loss) row_loss = reinterpret_cast<float*>(c.scratch + q.row_loss);
  const int blocks = (int)std::min<int64_t>(kStatBlocks, (c.classes + 2047) / 2048);
  TL_TRY(launch(few_stats_kernel, dim3((unsigned)c.rows, (unsigned)blocks), 256, 0, c.st,
                reinterpret_cast<const float*>(c.scratch + q.z), q.zsplits, q.zld, c.bias, c.targets(), part,
                q.part_ld, zt));
  auto join_rows = [&](auto kern) {
    return launch(kern, dim3(1), 1024, 0, c.st, part, q.part_ld, blocks, c.targets(), zt, nullptr, 1, 1, c.divisor,
                  row_loss, lse, loss, reinterpret_cast<Head*>(c.scratch));
  };
  return c.rows <= 4 ? join_rows(join_kernel<4, 1024>) : join_rows(join_kernel<32, 1024>);
}

int few_backward(const Call& c, const Plan& q, const float* lse, const float* upstream, void* dx, int64_t lddx,
                 void* dW, int64_t lddw, float* dbias, int accumulate) {
  float* scale = &reinterpret_cast<Head*>(c.scratch)->scale;
  float* g = reinterpret_cast<float*>(c.scratch + q.g);
  float* sums = reinterpret_cast<float*>(c.scratch + q.sums);
  const float *x = static_cast<const float*>(c.x), *w = static_cast<const float*>(c.w);
  TL_TRY(few_logits(c, q));
  TL_TRY(launch(few_grad_kernel, dim3((unsigned)((c.classes + 255) / 256)), 256, 0, c.st,
                reinterpret_cast<const float*>(c.scratch + q.z), q.zsplits, q.zld, c.bias, c.targets(), lse,
                c.divisor, upstream, scale, g, q.zld, dbias, accumulate & TL_ACC_DBIAS));
  if (dx) {
    const int64_t ld = up_to(c.width, 4);
    TL_TRY(c.trans_w ? few_product(false, w, c.ldw, c.classes, c.width, g, q.zld, c.rows, sums, ld, c.st)
                     : few_product(true, w, c.ldw, c.width, c.classes, g, q.zld, c.rows, sums, ld, c.st));
    TL_TRY(launch(dx_kernel<float>, dim3((unsigned)c.rows), 256, 0, c.st, sums, q.splits, c.rows, c.width, ld, scale,
                  static_cast<float*>(dx), lddx, accumulate & TL_ACC_DX));
  }
  if (dW) {
    const int64_t R = c.trans_w ? c.classes : c.width, C = c.trans_w ? c.width : c.classes;
    const float *p = c.trans_w ? g : x, *r = c.trans_w ? x : g;
    const int64_t ldp = c.trans_w ? q.zld : c.ldx, ldr = c.trans_w ? c.ldx : q.zld;
    TL_TRY(few_rows(c.rows, lddw % 4 == 0 && aligned_to(dW, 16), [&](auto tt, auto v) {
      return launch(few_outer_kernel<decltype(tt)::value, decltype(v)::value>,
                    dim3((unsigned)((C + 127) / 128), (unsigned)((R + kFewOuterRows - 1) / kFewOuterRows)),
                    kFewThreads, 0, c.st, p, ldp, r, ldr, (int)c.rows, c.targets(), R, C, scale,
                    static_cast<float*>(dW), lddw, accumulate & TL_ACC_DW);
    }));
  }
  return TL_OK;
}

int forward(const Call& c, const Plan& q, float* loss, float* row_loss, float* lse) {
  if (q.few) return few_forward(c, q, loss, row_loss, lse);
  Planes x, w;
  TL_TRY(x_planes(c, q, false, &x));
  TileParams p{};
  p.part = reinterpret_cast<float2*>(c.scratch + q.part);
  p.part_ld = q.part_ld;
  p.zt = reinterpret_cast<float*>(c.scratch + q.zt);
  if (!row_loss) row_loss = reinterpret_cast<float*>(c.scratch + q.row_loss);
  CUtensorMap none;
  memset(&none, 0, sizeof(none));
  const int64_t piece = direct(c, c.w, c.ldw) ? q.dpiece : q.fpiece;
  for (int64_t c0 = 0; c0 < c.classes; c0 += piece) {
    const int64_t n = std::min(piece, c.classes - c0);
    TL_TRY(w_planes(c, q, c0, n, &w));
    TL_TRY(logits<kStats>(c, x, w, none, p, c0, n));
    auto join_rows = [&](auto kern, int64_t r, int threads) {
      return launch(kern, dim3((unsigned)((c.rows + r - 1) / r)), threads, 0, c.st, p.part, q.part_ld,
                    stat_slots(c.rows, n, !c.trans_w), c.targets(), p.zt,
                    reinterpret_cast<float2*>(c.scratch + q.run), c0 == 0, c0 + n == c.classes,
                    c.divisor, row_loss, lse, loss, reinterpret_cast<Head*>(c.scratch));
    };
    // tiles of one CTA leave at most sm_count() partials a row: one block joins them
    // (a partial per tile and several blocks took 8 us longer for 96 tokens x 65536
    // classes x 2048, 4 us for 1 x 32768 x 4096); else few rows: more threads for each
    TL_TRY(c.rows <= 4          ? join_rows(join_kernel<4, 1024>, 4, 1024)
           : c.rows <= 32       ? join_rows(join_kernel<32, 1024>, 32, 1024)
           : one_cta(c.rows)    ? join_rows(join_kernel<128, 1024>, 128, 1024)
           : c.rows < 4096      ? join_rows(join_kernel<4, 256>, 4, 256)
                                : join_rows(join_kernel<32, 256>, 32, 256));
  }
  return TL_OK;
}

int backward(const Call& c, const Plan& q, const float* lse, const float* upstream, void* dx, int64_t lddx,
             void* dW, int64_t lddw, float* dbias, int accumulate) {
  if (q.few) return few_backward(c, q, lse, upstream, dx, lddx, dW, lddw, dbias, accumulate);
  float* scale = &reinterpret_cast<Head*>(c.scratch)->scale;
  Planes x, w;
  TL_TRY(x_planes(c, q, dW != nullptr, &x));
  const int64_t es = (int64_t)elem_bytes(c.dtype);
  float* sums = reinterpret_cast<float*>(c.scratch + q.sums);
  float* colsum = reinterpret_cast<float*>(c.scratch + q.colsum);
  const int64_t sums_ld = up_to(c.width, 4);
  for (int64_t c0 = 0; c0 < c.classes; c0 += q.bpiece) {
    const int64_t n = std::min(q.bpiece, c.classes - c0);
    TL_TRY(w_planes(c, q, c0, n, &w));
    const Planes g{reinterpret_cast<__nv_bfloat16*>(c.scratch + q.g), c.planes(), c.rows, n, q.bpiece};
    CUtensorMap o;
    if (!make_map3(&o, g.p, false, g.planes, g.rows, g.cols, g.ld, 64, 32)) return TL_ERR_UNSUPPORTED;
    TileParams p{};
    p.lse = lse;
    p.planes = c.planes();
    p.divisor = c.divisor;
    p.upstream = upstream;
    p.scale_out = c0 == 0 ? scale : nullptr;
    p.colsum = dbias ? colsum : nullptr;
    TL_TRY(logits<kGrad>(c, x, w, o, p, c0, n));
    p = TileParams{};
    p.terms = c.terms();
    p.kc = c.kc();
    p.scale = scale;
    if (dx) {  // sums[rows][width] += g W^T
      p.M = (int)c.rows;
      p.N = (int)c.width;
      p.K = (int)n;
      p.splits = q.splits;
      p.add = c0 > 0;
      if (!make_map3(&o, sums, true, q.splits, c.rows, c.width, sums_ld, 32, 32))
        return TL_ERR_UNSUPPORTED;
      TL_TRY((c.trans_w ? launch_tiles<0, 0, kSum>(g, w, o, p, c.st)
                        : launch_tiles<0, 1, kSum>(g, w, o, p, c.st)));
    }
    if (dW) {  // [classes][width] = g^T x, or [width][classes] = x^T g
      p.M = (int)(c.trans_w ? n : c.width);
      p.N = (int)(c.trans_w ? c.width : n);
      p.K = (int)c.rows;
      p.splits = 1;
      p.out = static_cast<char*>(dW) + (c.trans_w ? c0 * lddw : c0) * es;
      p.ldo = lddw;
      p.out_bf16 = !c.f32();
      p.accumulate = (accumulate & TL_ACC_DW) != 0;
      memset(&o, 0, sizeof(o));
      p.tma_out = !p.accumulate && (lddw * es) % 16 == 0 && aligned_to(p.out, 16) &&
                  make_map3(&o, p.out, c.f32(), 1, p.M, p.N, lddw, c.f32() ? 32 : 64, 32);
      const Planes& A = c.trans_w ? g : x;
      const Planes& B = c.trans_w ? x : g;
      TL_TRY((launch_tiles<1, 0, kOut>(A, B, o, p, c.st)));
    }
    if (dbias) {
      TL_TRY(launch(dbias_kernel, dim3((unsigned)((n + 31) / 32)), 256, 0, c.st, colsum, up_to(c.rows, 32) / 32,
                    n, scale, dbias + c0, accumulate & TL_ACC_DBIAS));
    }
  }
  if (dx) {
    const int64_t blocks = std::min<int64_t>(c.rows, 32LL * sm_count());
    if (c.f32())
      TL_TRY(launch(dx_kernel<float>, dim3((unsigned)blocks), 256, 0, c.st, sums, q.splits, c.rows, c.width,
                    sums_ld, scale, static_cast<float*>(dx), lddx, accumulate & TL_ACC_DX));
    else
      TL_TRY(launch(dx_kernel<__nv_bfloat16>, dim3((unsigned)blocks), 256, 0, c.st, sums, q.splits, c.rows,
                    c.width, sums_ld, scale, static_cast<__nv_bfloat16*>(dx), lddx, accumulate & TL_ACC_DX));
  }
  return TL_OK;
}

int check(const Call& c, size_t scratch_bytes, bool backward) {
  if (!dtype_ok(c.dtype) || !index_ok(c.index_type)) return TL_ERR_INVALID_ARG;
  if (c.trans_w != 0 && c.trans_w != 1) return TL_ERR_INVALID_ARG;
  if (c.rows < 0 || c.classes <= 0 || c.width <= 0) return TL_ERR_INVALID_ARG;
  if (c.rows > INT32_MAX / 2 || c.classes > INT32_MAX / 2 || c.width > INT32_MAX / 2)
    return TL_ERR_UNSUPPORTED;
  if (c.rows > 0 && (!c.x || !c.w || !c.target)) return TL_ERR_INVALID_ARG;
  if (c.ldx < c.width || c.ldw < (c.trans_w ? c.width : c.classes)) return TL_ERR_INVALID_ARG;
  if (!(c.divisor >= 0.f)) return TL_ERR_INVALID_ARG;
  if (!c.scratch || !aligned_to(c.scratch, 16) ||
      scratch_bytes < tl_linear_ce_scratch_bytes(c.dtype, c.trans_w, c.rows, c.classes, c.width, backward))
    return TL_ERR_INVALID_ARG;
  return TL_OK;
}

}  // namespace

int linear_ce_device_error(int* code, int reset) { return read_device_error(code, reset); }

}  // namespace tl

extern "C" {

size_t tl_linear_ce_scratch_bytes(int dtype, int trans_w, int64_t rows, int64_t classes, int64_t width,
                                  int backward) {
  if (!tl::dtype_ok(dtype) || rows < 0 || classes <= 0 || width <= 0) return 0;
  return (size_t)tl::make_plan(dtype, trans_w, std::max<int64_t>(rows, 1), classes, width, backward != 0)
      .total;
}

int tl_linear_ce(int dtype, int trans_w, int64_t rows, int64_t classes, int64_t width, const void* x,
                 int64_t ldx, const void* W, int64_t ldw, const float* bias, const void* target,
                 int index_type, float divisor, float* loss, float* row_loss, float* lse, void* scratch,
                 size_t scratch_bytes, void* stream) {
  tl::Call c{dtype, trans_w, index_type, rows, classes, width, x, ldx, W, ldw, bias, target, divisor,
             static_cast<char*>(scratch), nullptr};
  TL_TRY(tl::check(c, scratch_bytes, false));
  if (rows > 0 && !loss && !row_loss && !lse) return TL_ERR_INVALID_ARG;
  c.st = tl::stream_or_default(stream);
  if (rows == 0) {
    if (loss) TL_CUDA_TRY(cudaMemsetAsync(loss, 0, sizeof(float), c.st));
    return TL_OK;
  }
  return tl::forward(c, tl::make_plan(dtype, trans_w, rows, classes, width, false), loss, row_loss, lse);
}

int tl_linear_ce_backward(int dtype, int trans_w, int64_t rows, int64_t classes, int64_t width,
                          const void* x, int64_t ldx, const void* W, int64_t ldw, const float* bias,
                          const void* target, int index_type, float divisor, const float* lse,
                          const float* upstream, void* dx, int64_t lddx, void* dW, int64_t lddw,
                          float* dbias, int accumulate, void* scratch, size_t scratch_bytes,
                          void* stream) {
  tl::Call c{dtype, trans_w, index_type, rows, classes, width, x, ldx, W, ldw, bias, target, divisor,
             static_cast<char*>(scratch), nullptr};
  TL_TRY(tl::check(c, scratch_bytes, true));
  if (rows > 0 && (!lse || (!dx && !dW && !dbias))) return TL_ERR_INVALID_ARG;
  if (accumulate & ~(TL_ACC_DX | TL_ACC_DW | TL_ACC_DBIAS)) return TL_ERR_INVALID_ARG;
  if ((dx && lddx < width) || (dW && lddw < (trans_w ? width : classes))) return TL_ERR_INVALID_ARG;
  // the gradients are written piece by piece, while x and W are still read
  if ((dx && (dx == x || dx == W)) || (dW && (dW == W || dW == x)) || (dx && dx == dW))
    return TL_ERR_INVALID_ARG;
  c.st = tl::stream_or_default(stream);
  if (rows == 0) {  // sums over no rows
    const size_t es = tl::elem_bytes(dtype);
    if (dW && !(accumulate & TL_ACC_DW))
      TL_CUDA_TRY(cudaMemset2DAsync(dW, lddw * es, 0, (trans_w ? width : classes) * es,
                                    trans_w ? classes : width, c.st));
    if (dbias && !(accumulate & TL_ACC_DBIAS))
      TL_CUDA_TRY(cudaMemsetAsync(dbias, 0, classes * sizeof(float), c.st));
    return TL_OK;
  }
  return tl::backward(c, tl::make_plan(dtype, trans_w, rows, classes, width, true), lse, upstream, dx, lddx,
                      dW, lddw, dbias, accumulate);
}

}  // extern "C"
