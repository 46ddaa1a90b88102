// Linear layer on 8-bit integers, the W8A8 counterpart of bbh_linear:
//   C[m, n] = round16( a_scale[m] * w_scale[n] * sum_k A[m, k] W[n, k] + bias[n] )  (+ erf-GELU)
// The sum is exact (tcgen05.mma kind::i8, int32 accumulators in TMEM; |sum| <= 128^2 K < 2^31
// for K <= 131071), so the result does not depend on tile shape, split or order.
//
// Three kernels:
//  * linear_i8_pair_kernel -- many rows: persistent SM pairs (cta_group::2) on 256 x BN tiles,
//    two TMEM accumulators so that the epilogue of a tile runs under the MMAs of the next;
//  * linear_i8_small_kernel -- few rows: the weights are the MMA's 128-row operand and BN tokens
//    its columns, K split over the CTAs of a cluster, partial sums added in shared memory
//    (int32: exact in any order); both fed by 128-byte-swizzled TMA tiles of 128 int8 along K;
//  * linear_i8_few_kernel -- one to 16 tokens: the weights straight from memory into registers.
// A launch starts while the one in front still runs (griddepcontrol), and that one may write any operand: global
// memory is read after pdl_wait() only, and never through the non-coherent path (__ldg, const __restrict__),
// which is for what stays constant as long as the kernel lives.
// Every wait is bounded (mbar_wait); one that runs out sets the device error word and the
// kernel returns.
#include "common.cuh"
#include "epilogue.cuh"
#include "internal.h"
#include "../../include/bbh.h"

#include <cuda_bf16.h>

#include <atomic>
#include <cfloat>
#include <string>

namespace bbh {

// (16 bytes more of arguments made a launch of the one-token kernel 0.35 us longer for the host: 3.8 instead of 3.45)
struct I8Params {
  const float* a_scale;    // [M]
  const float* w_scale;    // [N]
  const uint16_t* bias;    // [N] or null, the output's type
  uint16_t* C;
  int64_t ldc;
  int M, N, K;
  int prefetch;  // few rows: W to L2 while the kernel in front still runs (see kPrefetchBytes)
};

// Weights are constants of a model and, one token after the other, come from HBM: the kernels for few rows ask
// for theirs before they wait for the kernel in front of them. That brings bytes to L2 and reads none, so what
// that kernel may still write to W is seen after the wait. 16 pairs of quantize_i8 and linear_i8 with weights of
// 4096 x 4096 each, one token: 106 -> 96 us; 16 tokens 119 -> 107, 64 tokens 143 -> 137. Where the weights are in
// L2 already it costs 0 to 0.2 us a launch; with much more of them than L2 takes it only changes the order of
// the reads (16384 x 4096: 12.4 -> 13.4 us).
constexpr int64_t kPrefetchBytes = int64_t(32) << 20;
constexpr int kPrefetchBlocks = 4;  // k-blocks of a CTA, few-rows kernel (all of them: twice the loss, little more gain)

__device__ int g_i8_err;  // first device error of these kernels (kDevWaitTimeout)

// D[tmem] (+)= A[smem] * B[smem]^T, kind::i8 (int8 in, int32 accumulate).
__device__ __forceinline__ void tc_mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tc_mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive once on the mbarrier at this shared-memory offset in BOTH CTAs of the pair when the pair
// MMAs issued so far by this thread have finished (one commit: each costs the issuing thread time).
__device__ __forceinline__ void tc_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// The two halves of a cluster's barrier. The relaxed arrival orders no memory accesses: with .release the
// barrier took 1,200 cycles, with outstanding stores or none.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// One lane of a converged warp. The loops that issue copies and MMAs run under it and not under
// `lane == 0`: it tells the compiler that a single lane runs them, and their descriptors and addresses
// stay in uniform registers. An MMA then takes its thread 30 cycles instead of 60 and a k-block of
// the few-rows kernel 245 to 316 instead of 460 (which it took for any number of tokens).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// `bytes` (a multiple of 16, at a multiple of 16) to L2.
__device__ __forceinline__ void l2_prefetch(const void* at, uint32_t bytes) {
  if (bytes) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(bytes) : "memory");
}

// Instruction descriptor, kind::i8: signed A and B, int32 D, both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

constexpr int kBK = 128;  // int8 per k-block: one 128-byte swizzle row
constexpr int kMmaK = 32;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// min(|x|, 16) that keeps a NaN (fminf drops it)
__device__ __forceinline__ float abs_to_16(float x) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(x)), "f"(16.f));
  return d;
}

// erf-GELU, x Phi(x) = max(x, 0) - |x| Phi(-|x|), of N pairs of fp32 values side by side (which hides
// the fmas' latency). log2 Phi(-a) is close to a parabola and is evaluated as a polynomial of degree 10
// in a (this project's own least-squares fit on [0, 5.75], weighted by what an error means to the
// output and reweighted to equal ripple): Phi(-a) is within 1.8e-7 of itself up to a = 4, 2e-6 up to 5.75;
// beyond, the polynomial keeps falling until ex2 gives 0 (from a = 11.5 on); a ends at 16, because infinity times that
// 0 would be NaN: +inf stays +inf, -inf gives 0, and only NaN gives NaN. With the roundings of the sum and of ex2
// the output is within 2e-7 max(|x|, 1).
// Why this degree: of normal x 0.009 % of the fp16 outputs are the other neighbour of the exact value, 0.018 %
// with fp32's erf. Degree 7 (Phi within 5.8e-6) has 0.20 %, and a quantiser behind the layer then rounds ten times
// as many of its integers the other way, each of which the next layer spreads over a row; degree 9 0.018 to
// 0.03 %. 68451 x 1536 x 384: 68.9 us with degree 7 one value at a time, here, in packed pairs (half the
// issue slots), 74.3; degree 9 72.9; degree 10 one value at a time 82.3.
template <int N>
__device__ __forceinline__ void gelu2(unsigned long long (&x)[N]) {
  constexpr float kPhi[11] = {-0.999999881f,    -1.15111041f,    -0.459175467f,   -0.052566696f,
                              0.00711826188f,   -0.000130872504f, -0.000220343485f, 6.01809223e-05f,
                              -8.31889884e-06f, 6.23994595e-07f, -2.01010462e-08f};
  unsigned long long a[N], p[N];
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float2 r = f2_split(x[q]);
    a[q] = f2(abs_to_16(r.x), abs_to_16(r.y));
    x[q] = f2(fmaxf(r.x, 0.f), fmaxf(r.y, 0.f));
  }
#pragma unroll
  for (int q = 0; q < N; ++q) p[q] = f2_fma(f2(kPhi[10], kPhi[10]), a[q], f2(kPhi[9], kPhi[9]));
#pragma unroll
  for (int i = 8; i >= 0; --i)
#pragma unroll
    for (int q = 0; q < N; ++q) p[q] = f2_fma(p[q], a[q], f2(kPhi[i], kPhi[i]));
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float2 r = f2_split(x[q]), e = f2_split(p[q]), m = f2_split(a[q]);
    x[q] = f2(fmaf(-m.x, ex2(e.x), r.x), fmaf(-m.y, ex2(e.y), r.y));
  }
}

// N pairs of outputs (with GELU) rounded to 16 bits, packed (the low half first).
template <bool BF16, bool GELU, int N>
__device__ __forceinline__ void finish2(unsigned long long (&y)[N], uint32_t (&w)[N]) {
  if constexpr (GELU) gelu2(y);
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float2 v = f2_split(y[q]);
    if constexpr (BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
      w[q] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      w[q] = pack_half2(v.x, v.y);
    }
  }
}

template <bool BF16>
__device__ __forceinline__ float bias_f32(const uint16_t* b) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(*b) << 16);
  return __half2float(*reinterpret_cast<const __half*>(b));
}

// (acc * a_scale) * w_scale + bias of two outputs, the same in both kernels (bit for bit)
__device__ __forceinline__ unsigned long long dequant2(int acc0, int acc1, unsigned long long sa,
                                                       unsigned long long sw, unsigned long long bias) {
  return f2_fma(f2_mul(f2(__int2float_rn(acc0), __int2float_rn(acc1)), sa), sw, bias);
}

// 32 lanes x 32 columns of TMEM, the load only; tmem_wait32 makes the registers valid.
__device__ __forceinline__ void tmem_issue32(uint32_t taddr, int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait32(int (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// 16 lanes x 32 columns of TMEM in the 16x256b shape, the load only (tmem_wait16 makes the registers
// valid): thread t gets rows t / 4 (r[4j], r[4j+1]) and t / 4 + 8 (r[4j+2], r[4j+3]) of columns
// 8 j + 2 (t % 4) and the next, j = 0 .. 3.
__device__ __forceinline__ void tmem_issue16(uint32_t taddr, int (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait16(int (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])
               :
               : "memory");
}

// Four 8 x 8 matrices of 16-bit elements to shared memory: matrix i from w[i] of every thread (row t / 4,
// elements 2 (t % 4) and the next), its row r at the address that lane 8 i + r gives.
__device__ __forceinline__ void stmatrix4(uint32_t addr, const uint32_t (&w)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3])
               : "memory");
}

// ====================================================================== many rows: SM pairs

// COLS: columns per epilogue warp.
template <int BN, int COLS>
struct I8PairCfg {
  static constexpr int BM = 128;         // accumulator rows per CTA (256 per pair)
  static constexpr int B_ROWS = BN / 2;  // W rows held by each CTA
  static constexpr int A_BYTES = BM * kBK;
  static constexpr int B_BYTES = B_ROWS * kBK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int EPI_WARPS = 4 * BN / COLS;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STAGING_BYTES = EPI_WARPS * 4096;   // per epilogue warp: two chunks of 16 rows x 64 columns
  static constexpr int COLS_BYTES = EPI_WARPS * 8 * COLS;  // per epilogue warp: COLS scales and biases
  static constexpr int AUX_BYTES = 512 /*barriers*/ + COLS_BYTES;
  static constexpr int STAGES = (227 * 1024 - 1024 - STAGING_BYTES - AUX_BYTES) / STAGE_BYTES;
  static constexpr int NACC = 2;
  static constexpr int TMEM_COLS = 512;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + STAGING_BYTES + AUX_BYTES;
  static_assert(BN % COLS == 0 && COLS % 64 == 0 && BN <= 256 && NACC * BN <= TMEM_COLS, "pair tile");
  static_assert(STAGES >= 4 && SMEM <= 227 * 1024, "shared memory");
  static_assert((2 * STAGES + 2 * NACC) * 8 + 8 <= 512, "barriers");
};

// TMA_C: C is written with TMA stores (16-byte aligned rows of whole 16 bytes); otherwise row by row from the
// staging buffer with 2-byte stores, which any N and alignment allows.
template <int BN, int COLS, bool BF16, bool GELU, bool TMA_C>
__global__ void __launch_bounds__(I8PairCfg<BN, COLS>::THREADS, 1)
    linear_i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmC, const I8Params p) {
  using Cfg = I8PairCfg<BN, COLS>;
  constexpr int STAGES = Cfg::STAGES;
  constexpr int NACC = Cfg::NACC;

  extern __shared__ uint8_t smem_raw[];
  // the same 1024-aligned offsets in both CTAs: the pair MMA reads both at one address
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint8_t* s_stage = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_stage + Cfg::STAGING_BYTES);  // used in the even CTA
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* accf_bar = empty_bar + STAGES;
  uint64_t* acce_bar = accf_bar + NACC;  // used in the even CTA
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acce_bar + NACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* s_cols = reinterpret_cast<float*>(s_stage + Cfg::STAGING_BYTES + 512);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const bool leader = crank == 0;
  const int half = static_cast<int>(crank);  // which 128 rows of the pair tile

  pdl_launch_dependents();
  const int n_tiles = (p.N - 1) / BN + 1;  // (not + BN - 1: M and N may be near 2^31)
  const int k_blocks = (p.K + kBK - 1) / kBK;
  const int num_tiles = ((p.M - 1) / (2 * Cfg::BM) + 1) * n_tiles;
  const int first_tile = static_cast<int>(blockIdx.x) / 2;
  const int tile_step = static_cast<int>(gridDim.x) / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);   // the even CTA's producer arrival (+ both CTAs' bytes)
      mbar_init(&empty_bar[s], 1);  // one commit from the MMA thread
    }
    for (int a = 0; a < NACC; ++a) {
      mbar_init(&accf_bar[a], 1);
      mbar_init(&acce_bar[a], 2 * Cfg::EPI_WARPS);  // every epilogue warp of both CTAs
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (TMA_C) tma_prefetch_desc(&tmC);
  }
  if (warp == 1) tmem_alloc_pair(tmem_holder, Cfg::TMEM_COLS);
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  cluster_arrive_relaxed();  // both CTAs' barriers initialised (fence_barrier_init), TMEM allocated
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  // Tiles t in n-fastest order: rows m * 256 + 128 * half, columns n * BN.
  struct Tile {
    int t, m, n;
  };
  const int m_step = tile_step / n_tiles, n_step = tile_step % n_tiles;
  const Tile tile0{first_tile, first_tile / n_tiles, first_tile % n_tiles};
  auto next = [&](const Tile& c) {
    Tile d{c.t + tile_step, c.m + m_step, c.n + n_step};
    if (d.n >= n_tiles) {
      d.n -= n_tiles;
      ++d.m;
    }
    return d;
  };
  auto tile_m0 = [&](const Tile& c) { return c.m * (2 * Cfg::BM) + half * Cfg::BM; };
  auto tile_n0 = [&](const Tile& c) { return c.n * BN; };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (elect_one()) {
      const uint32_t full0 = mapa_shared(smem_u32(full_bar), 0);
      int stage = 0;
      uint32_t phase = 0;
      for (Tile tile = tile0; tile.t < num_tiles && !*abort_flag; tile = next(tile)) {
        const int m0 = tile_m0(tile);
        const int nb = tile_n0(tile) + half * Cfg::B_ROWS;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, &g_i8_err)) break;
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);
          const uint32_t fb = full0 + stage * 8;
          tma_load_2d_pair(sA + stage * Cfg::A_BYTES, &tmA, fb, kb * kBK, m0);
          tma_load_2d_pair(sB + stage * Cfg::B_BYTES, &tmB, fb, kb * kBK, nb);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    if (leader && elect_one()) {
      constexpr uint32_t idesc = idesc_i8(2 * Cfg::BM, BN);
      const uint64_t a_desc0 = sw128_kmajor_desc(smem_u32(sA)), b_desc0 = sw128_kmajor_desc(smem_u32(sB));
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      // k-blocks whose slot is filled again; the others are not announced, so that no arrival is on its way to
      // a CTA that has left
      const int refilled = first_tile < num_tiles ? ((num_tiles - 1 - first_tile) / tile_step + 1) * k_blocks - STAGES : 0;
      int block = 0;
      for (int tile = first_tile; tile < num_tiles && !*abort_flag; tile += tile_step) {
        if (!mbar_wait(&acce_bar[acc], acc_phase ^ 1, abort_flag, &g_i8_err)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        bool ok = true;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag, &g_i8_err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t a_desc = a_desc0 + stage * (Cfg::A_BYTES >> 4), b_desc = b_desc0 + stage * (Cfg::B_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < kBK / kMmaK; ++k)
            tc_mma_i8_pair(d_tmem, a_desc + k * (kMmaK >> 4), b_desc + k * (kMmaK >> 4), idesc, (kb | k) != 0 ? 1u : 0u);
          // the slot is free in both CTAs once these MMAs have read it
          if (block++ < refilled) tc_commit_both(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        tc_commit_both(&accf_bar[acc]);
        if (++acc == NACC) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quad = warp & 3;         // TMEM lane quadrant this warp may access
    const int part = (warp - 2) >> 2;  // which COLS columns of the tile
    const int we = warp - 2;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    // Two chunks of 16 rows x 64 columns (row half 0 and 1), 16-byte piece c of row r at piece c ^ (r & 7).
    uint8_t* buf = s_stage + we * 4096;
    float* s_sw = s_cols + we * 2 * COLS;  // this warp's channel scales, then biases
    float* s_b = s_sw + COLS;
    const uint32_t acce0 = mapa_shared(smem_u32(acce_bar), 0);
    const int row_t = lane >> 2, col_t = 2 * (lane & 3);  // this thread's place in an 8 x 8 block
    // this lane's row and piece parity of the four blocks that one stmatrix4 writes: rows 0-7, 8-15 of a
    // 16-byte piece, then of the next
    const int row_m = (lane & 7) + (lane & 8), piece_m = lane >> 4;
    // The scales and biases of a tile are fetched while the previous tile is worked on: the rows row_t + 8 i,
    // and columns lane + 32 i for the warp's table.
    float sa_next[4], sw_next[COLS / 32], b_next[COLS / 32];
    auto fetch = [&](const Tile& t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = tile_m0(t) + quad * 32 + row_t + 8 * i;
        sa_next[i] = row < p.M ? p.a_scale[row] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < COLS / 32; ++i) {
        const int c = tile_n0(t) + part * COLS + 32 * i + lane;
        sw_next[i] = c < p.N ? p.w_scale[c] : 0.f;
        b_next[i] = p.bias && c < p.N ? bias_f32<BF16>(p.bias + c) : 0.f;
      }
    };
    if (first_tile < num_tiles) fetch(tile0);
    int acc = 0;
    uint32_t acc_phase = 0;
    Tile ahead = tile0;
    for (Tile tile = tile0; tile.t < num_tiles; tile = ahead) {
      const int row0 = tile_m0(tile) + quad * 32;
      const int c0 = tile_n0(tile) + part * COLS;
      __syncwarp();  // every lane has read the previous tile's scales and biases
      float sa[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = sa_next[i];
#pragma unroll
      for (int i = 0; i < COLS / 32; ++i) {
        s_sw[32 * i + lane] = sw_next[i];
        s_b[32 * i + lane] = b_next[i];
      }
      __syncwarp();
      ahead = next(tile);
      if (ahead.t < num_tiles) fetch(ahead);
      if (!mbar_wait(&accf_bar[acc], acc_phase, abort_flag, &g_i8_err)) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + lane_off + acc * BN + part * COLS;
      // steps of 16 rows x 32 columns (row half h of 32 columns, then the other half), the next one's
      // TMEM load under way during each
      constexpr int STEPS = COLS / 16;
      int v[2][16];
      tmem_issue16(tacc, v[0]);
      unsigned long long sw[4], b[4];  // of this thread's 8 of the 32 columns
#pragma unroll
      for (int step = 0; step < STEPS; ++step) {
        const int h = step & 1, cs = step >> 1;
        tmem_wait16(v[step & 1]);
        if (step < STEPS - 1) {
          tmem_issue16(tacc + (static_cast<uint32_t>(16 * ((step + 1) & 1)) << 16) + 32 * ((step + 1) >> 1),
                       v[(step + 1) & 1]);
        } else {
          // accumulator read: release it to the even CTA's MMA thread, if that will use it again
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && tile.t + NACC * tile_step < num_tiles) mbar_arrive_cluster(acce0 + acc * 8);
        }
        if (h == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sw[j] = *reinterpret_cast<const unsigned long long*>(s_sw + 32 * cs + 8 * j + col_t);
            b[j] = *reinterpret_cast<const unsigned long long*>(s_b + 32 * cs + 8 * j + col_t);
          }
        }
        if (TMA_C && cs % 2 == 0) {
          // the last store of this half's chunk has read it (half 1's was issued last)
          if (lane == 0) {
            if (h == 0) bulk_wait_read<1>();
            else bulk_wait_read<0>();
          }
          __syncwarp();
        }
        const int(&x)[16] = v[step & 1];
        const unsigned long long sa0 = f2(sa[2 * h], sa[2 * h]), sa1 = f2(sa[2 * h + 1], sa[2 * h + 1]);
        const uint32_t dst = smem_u32(buf + h * 2048 + row_m * 128);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          unsigned long long y[4];
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int* a = &x[4 * (j + k)];
            y[2 * k] = dequant2(a[0], a[1], sa0, sw[j + k], b[j + k]);
            y[2 * k + 1] = dequant2(a[2], a[3], sa1, sw[j + k], b[j + k]);
          }
          finish2<BF16, GELU>(y, w);
          stmatrix4(dst + (((4 * (cs & 1) + j + piece_m) ^ (lane & 7)) << 4), w);
        }
        if (cs % 2 == 1) {
          // 16 rows x 64 columns are in place
          const int col = c0 + 32 * (cs - 1), row = row0 + 16 * h;
          if constexpr (TMA_C) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
              if (col < p.N && row < p.M) tma_store_2d(&tmC, buf + h * 2048, col, row);
              bulk_commit();  // one group per chunk, empty ones too: bulk_wait_read counts them
            }
          } else {
            // row by row: 32 neighbouring 2-byte stores at a time
            __syncwarp();
            const int rows = min(16, p.M - row);
            for (int r = 0; r < rows; ++r) {
              const uint8_t* line = buf + h * 2048 + r * 128;
              uint16_t* c = p.C + static_cast<int64_t>(row + r) * p.ldc + col;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int e = 32 * i + lane;
                const uint16_t o =
                    *reinterpret_cast<const uint16_t*>(line + (((e >> 3) ^ (r & 7)) << 4) + (e & 7) * 2);
                if (col + e < p.N) c[e] = o;
              }
            }
            __syncwarp();
          }
        }
      }
      if (++acc == NACC) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (TMA_C && lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == 0 && lane == 0) {
    // Let in-flight TMA copies land before the CTA's shared memory is released.
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 1000000ull) {
    }
  }
  __syncthreads();
  // Both CTAs are done with the accumulators. Every arrival, copy and MMA that one made in the other has been
  // waited for above, so nothing is left to be ordered.
  cluster_arrive_relaxed();
  cluster_wait();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
}

// ====================================================================== few rows: split K

template <int BN>
struct I8SmallCfg {
  static constexpr int A_BYTES = 128 * kBK;  // 128 output channels of W
  static constexpr int B_BYTES = BN * kBK;   // BN tokens
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // partial sums of the tokens that a CTA finishes, from every CTA of the cluster: int32
  // [splits][tokens / 4][128 channels][4], at least 4 tokens a CTA, at most 8 CTAs
  static constexpr int RED_BYTES = (BN < 32 ? 32 : BN) * 512;
  static constexpr int STAGES = (204 * 1024 - RED_BYTES) / STAGE_BYTES > 8 ? 8 : (204 * 1024 - RED_BYTES) / STAGE_BYTES;
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int PARTS = BN < 64 ? 1 : 2;  // epilogue warps per TMEM lane quadrant, BN / PARTS tokens each
  static constexpr int THREADS = 64 + 128 * PARTS;
  static constexpr int SMEM = STAGES * STAGE_BYTES + RED_BYTES + 1024 + 256 + 4 * BN;
  static_assert((BN & (BN - 1)) == 0 && BN >= 16 && BN <= 128, "token tile");
  // more than half an SM's shared memory: one CTA per SM, so TMEM can always be had
  static_assert(SMEM > 114 * 1024 && SMEM <= 227 * 1024, "shared memory");
};

// grid: x = cluster size (2^log_splits) * channel tiles, y = token tiles. Rank r of a cluster sums the
// r-th part of the k-blocks and finishes the r-th `per` tokens of the tile.
template <int BN, bool BF16, bool GELU>
__global__ void __launch_bounds__(I8SmallCfg<BN>::THREADS, 1)
    linear_i8_small_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                           const I8Params p, const int log_splits, const int8_t* W, const int64_t ldw) {
  using Cfg = I8SmallCfg<BN>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint8_t* red = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(red + Cfg::RED_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_bar = empty_bar + STAGES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* s_sa = reinterpret_cast<float*>(red + Cfg::RED_BYTES + 256);  // [BN] token scales

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int splits = 1 << log_splits;
  const int rank = log_splits ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = (static_cast<int>(blockIdx.x) >> log_splits) * 128;
  const int m0 = static_cast<int>(blockIdx.y) * BN;
  const int k_blocks = (p.K + kBK - 1) / kBK;
  const int kb0 = (k_blocks * rank) >> log_splits;
  const int kb1 = (k_blocks * (rank + 1)) >> log_splits;
  const int tokens = min(BN, p.M - m0);

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(acc_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) tmem_alloc(tmem_holder, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  if (p.prefetch && blockIdx.y == 0 && warp >= 2 && warp < 6) {  // not by TMA, which takes its orders one after the other
    const int row = n0 + static_cast<int>(threadIdx.x) - 64;
    if (row < p.N) {
      for (int kb = kb0; kb < min(kb1, kb0 + kPrefetchBlocks); ++kb)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(W + row * ldw + kb * kBK));
    }
  }
  pdl_wait();
  if (log_splits) cluster_arrive_relaxed();  // this CTA runs: its shared memory may be written (waited for below)

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, &g_i8_err)) break;
        mbar_arrive_expect_tx(&full_bar[stage], Cfg::STAGE_BYTES);
        tma_load_2d(sA + stage * Cfg::A_BYTES, &tmW, &full_bar[stage], kb * kBK, n0);
        tma_load_2d(sB + stage * Cfg::B_BYTES, &tmX, &full_bar[stage], kb * kBK, m0);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_i8(128, BN);
      const uint64_t a_desc0 = sw128_kmajor_desc(smem_u32(sA)), b_desc0 = sw128_kmajor_desc(smem_u32(sB));
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag, &g_i8_err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t a_desc = a_desc0 + stage * (Cfg::A_BYTES >> 4), b_desc = b_desc0 + stage * (Cfg::B_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < kBK / kMmaK; ++k)
          tc_mma_i8(tmem, a_desc + k * (kMmaK >> 4), b_desc + k * (kMmaK >> 4), idesc, (kb != kb0 || k) ? 1u : 0u);
        tc_commit(&empty_bar[stage]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (ok) tc_commit(acc_bar);
    }
    __syncwarp();
  }

  // Epilogue threads: TMEM lane = output channel, column = token. Each thread has one channel and
  // works on groups of four tokens.
  const bool epi = warp >= 2;
  const int quad = warp & 3;
  const int part = epi ? (warp - 2) >> 2 : 0;
  const int ch = quad * 32 + lane;
  const int n = n0 + ch;
  unsigned long long sw = 0, bias = 0;
  // G groups of four tokens from t on of this thread's channel: 2-byte stores, 32 neighbouring channels a
  // warp (four channels a store, after a transposition between lanes, took longer). G groups side by
  // side: the epilogue's time is the latency of its chain of steps.
  auto put = [&](int t, const auto& a) {
    constexpr int G = sizeof(a) / sizeof(int4);
    unsigned long long y[2 * G];
    uint32_t w[2 * G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const ulonglong2 sa = *reinterpret_cast<const ulonglong2*>(s_sa + t + 4 * g);
      y[2 * g] = dequant2(a[g].x, a[g].y, sa.x, sw, bias);
      y[2 * g + 1] = dequant2(a[g].z, a[g].w, sa.y, sw, bias);
    }
    finish2<BF16, GELU>(y, w);
    uint16_t* c = p.C + static_cast<int64_t>(m0 + t) * p.ldc + n;
    const int rows = n < p.N ? tokens - t : 0;
#pragma unroll
    for (int i = 0; i < 4 * G; ++i) {
      if (i < rows) *c = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      c += p.ldc;
    }
  };
  // partial sums: int4 g (tokens 4 g ..) of channel ch from rank src at [src][g][ch]
  const int log_per = max(2, (31 - __clz(BN)) - log_splits);  // tokens a CTA finishes: 2^log_per
  const int pieces = 1 << (log_per - 2);
  bool ok = true;
  if (epi) {
    const int e = threadIdx.x - 64;
    if (e < BN) s_sa[e] = e < tokens ? p.a_scale[m0 + e] : 0.f;
    if (n < p.N) {
      const float s = p.w_scale[n];
      const float b = p.bias ? bias_f32<BF16>(p.bias + n) : 0.f;
      sw = f2(s, s);
      bias = f2(b, b);
    }
    named_barrier(1, 128 * Cfg::PARTS);  // the token scales are in place
    ok = mbar_wait(acc_bar, 0, abort_flag, &g_i8_err);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
  }
  if (log_splits) cluster_wait();  // every CTA of the cluster runs
  if (epi && ok) {
    const uint32_t tacc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const int t_end = min(tokens, (part + 1) * (BN / Cfg::PARTS));
#pragma unroll 1
    for (int c = part * (BN / Cfg::PARTS); c < t_end; c += 32) {  // BN = 16: the upper 16 columns are not used
      int v[32];
      tmem_issue32(tacc + c, v);
      tmem_wait32(v);
      int4 a[8];
#pragma unroll
      for (int g = 0; g < 8; ++g) a[g] = make_int4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
      if (log_splits == 0) {
        if constexpr (BN >= 32) {
          put(c, a);
        } else {
          const int4 low[4] = {a[0], a[1], a[2], a[3]};
          put(c, low);
        }
      } else {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const int t = c + 4 * g;
          if (t < tokens) {
            const int piece = (t & ((1 << log_per) - 1)) >> 2;
            int4* at = reinterpret_cast<int4*>(red) + (rank * pieces + piece) * 128 + ch;
            if (t >> log_per == rank) {
              *at = a[g];
              continue;
            }
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_shared(smem_u32(at), t >> log_per)),
                         "r"(a[g].x), "r"(a[g].y), "r"(a[g].z), "r"(a[g].w)
                         : "memory");
          }
        }
      }
    }
  }
  if (log_splits) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();  // all partial sums are in place
    if (epi) {
      auto sum = [&](int g, auto& a) {
        constexpr int G = sizeof(a) / sizeof(int4);
#pragma unroll
        for (int i = 0; i < G; ++i) a[i] = make_int4(0, 0, 0, 0);
        for (int src = 0; src < splits; ++src) {
          const int4* x = reinterpret_cast<const int4*>(red) + (src * pieces + g) * 128 + ch;
#pragma unroll
          for (int i = 0; i < G; ++i) {
            const int4 u = x[i * 128];
            a[i] = make_int4(a[i].x + u.x, a[i].y + u.y, a[i].z + u.z, a[i].w + u.w);
          }
        }
      };
      const int mine = max(pieces / Cfg::PARTS, 1);  // this warp's pieces, from `first` on
      const int first = part * mine;
      const int t0 = rank << log_per;
      if (first < pieces) {
        if (mine >= 4) {
          for (int g = first; g < first + mine && t0 + 4 * g < tokens; g += 4) {
            int4 a[4];
            sum(g, a);
            put(t0 + 4 * g, a);
          }
        } else {
          for (int g = first; g < first + mine && t0 + 4 * g < tokens; ++g) {
            int4 a[1];
            sum(g, a);
            put(t0 + 4 * g, a);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    // Let in-flight TMA copies land before the CTA's shared memory is released.
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 1000000ull) {
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

// ======================================================================== one to 16 tokens

// Single tokens and decoding batches: the weights' bytes are the work, and a launch's fixed costs (TMEM,
// barriers, a cluster) are as long as their transfer. So no staging: a CTA has 16 output channels, its
// eight warps every eighth 64 bytes of K, loaded straight into the fragments of mma.sync m16n8k32 (the
// order of k is free as long as both operands have the same, so a lane's 16 consecutive bytes are four
// of its fragments' words), and the partial sums meet in shared memory. 1 x 4096 x 4096: 3.3 us = 5.1 TB/s
// of weights when they are in L2, 4.8 = 3.5 TB/s when they come from HBM; 1 x 8192 x 2048 3.3 and 4.8.
constexpr int kFewWarps = 8;

__device__ __forceinline__ void mma_i8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of an int8 row from k on, zeros behind its end (and nothing read there).
__device__ __forceinline__ uint4 load_k16(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
  const int r = k < K ? K - k : 0;  // 0 .. 15 bytes: an 8-, a 4-, a 2- and a 1-byte load
  const int8_t* at = row + k;
  uint64_t lo = 0, rest = 0;
  if (r & 8) lo = *reinterpret_cast<const uint64_t*>(at);
  at += r & 8;
  if (r & 4) rest = *reinterpret_cast<const uint32_t*>(at);
  at += r & 4;
  if (r & 2) rest |= static_cast<uint64_t>(*reinterpret_cast<const uint16_t*>(at)) << (8 * (r & 4));
  at += r & 2;
  if (r & 1) rest |= static_cast<uint64_t>(static_cast<uint8_t>(*at)) << (8 * (r & 6));
  const uint64_t hi = r & 8 ? rest : 0;
  lo = r & 8 ? lo : rest;
  return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
                    static_cast<uint32_t>(hi >> 32));
}

// MT: token tiles of 8. U: 64-byte steps in flight per warp.
template <int MT, int U, bool BF16, bool GELU>
__global__ void __launch_bounds__(32 * kFewWarps)
    linear_i8_few_kernel(const int8_t* A, const int64_t lda, const int8_t* W,
                         const int64_t ldw, const I8Params p) {
  __shared__ int part[kFewWarps][MT * 128];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  // rows behind the last channel or token repeat the last one; their sums are not used
  const int8_t* w0 = W + min(n0 + g, static_cast<int64_t>(p.N) - 1) * ldw;
  const int8_t* w1 = W + min(n0 + g + 8, static_cast<int64_t>(p.N) - 1) * ldw;
  const int8_t* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = A + static_cast<int64_t>(min(8 * t + g, p.M - 1)) * lda;
  int acc[MT][4] = {};
  if (p.prefetch && threadIdx.x < 16 && n0 + threadIdx.x < p.N) l2_prefetch(W + (n0 + threadIdx.x) * ldw, p.K & ~15);
  pdl_wait();
  for (int k0 = 64 * warp; k0 < p.K; k0 += 64 * kFewWarps * U) {
    uint4 a[U], b[U], v[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + 64 * kFewWarps * u + 16 * q;
      a[u] = load_k16(w0, k, p.K);
      b[u] = load_k16(w1, k, p.K);
#pragma unroll
      for (int t = 0; t < MT; ++t) v[u][t] = load_k16(x[t], k, p.K);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        mma_i8(acc[t], a[u].x, b[u].x, a[u].y, b[u].y, v[u][t].x, v[u][t].y);
        mma_i8(acc[t], a[u].z, b[u].z, a[u].w, b[u].w, v[u][t].z, v[u][t].w);
      }
  }
  // acc[t]: channels g (0, 1) and g + 8 (2, 3), tokens 8 t + 2 q and the next; part[warp][token][channel]
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][(8 * t + 2 * q + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[t][i];
  __syncthreads();
  // one thread a token and two neighbouring channels
  const int tok = threadIdx.x >> 3, c = 2 * (threadIdx.x & 7);
  if (tok >= p.M || tok >= 8 * MT) return;
  int s0 = 0, s1 = 0;
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    const int2 u = *reinterpret_cast<const int2*>(&part[w][tok * 16 + c]);
    s0 += u.x;
    s1 += u.y;
  }
  const int64_t n = n0 + c;
  const bool one = n < p.N, two = n + 1 < p.N;
  const float sa = p.a_scale[tok];
  const float b0 = p.bias && one ? bias_f32<BF16>(p.bias + n) : 0.f, b1 = p.bias && two ? bias_f32<BF16>(p.bias + n + 1) : 0.f;
  unsigned long long y[1] = {dequant2(s0, s1, f2(sa, sa), f2(one ? p.w_scale[n] : 0.f, two ? p.w_scale[n + 1] : 0.f),
                                      f2(b0, b1))};
  uint32_t o[1];
  finish2<BF16, GELU>(y, o);
  uint16_t* out = p.C + tok * p.ldc + n;
  if (one) out[0] = static_cast<uint16_t>(o[0]);
  if (two) out[1] = static_cast<uint16_t>(o[0] >> 16);
}

// ======================================================================== host side
namespace {

// What is asked or set once per device, by whichever thread comes first (several may: all find the same).
using OncePerDevice = std::atomic<int>[64];

// Once per device and kernel: opt in to the kernel's shared memory.
template <typename K>
cudaError_t opt_in(K kern, int smem, OncePerDevice& done, int dev) {
  if (done[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) done[dev] = 1;
  return e;
}

// Clusters of `size` CTAs that can run at once, asked once per device and kernel.
template <typename K>
int max_clusters(K kern, int size, int threads, int smem, int sms, OncePerDevice& cache, int dev) {
  if (const int known = cache[dev]) return known;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(sms / size * size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = sms / size;
  }
  cache[dev] = n;
  return n;
}

struct I8Maps {
  CUtensorMap A, W, C;
  const int8_t* w;
  int64_t ldw;
};

template <int BN, int COLS, bool BF16, bool GELU, bool TMA_C>
cudaError_t launch_pair_i8(const I8Maps& m, const I8Params& p, int dev, int sms, cudaStream_t s) {
  using Cfg = I8PairCfg<BN, COLS>;
  static OncePerDevice done;
  auto kern = linear_i8_pair_kernel<BN, COLS, BF16, GELU, TMA_C>;
  const cudaError_t e = opt_in(kern, Cfg::SMEM, done, dev);
  if (e != cudaSuccess) return e;
  static OncePerDevice pairs_of;
  const int64_t tiles = (int64_t(p.M) + 255) / 256 * ((p.N - 1) / BN + 1);
  const int most = max_clusters(kern, 2, Cfg::THREADS, Cfg::SMEM, sms, pairs_of, dev);
  const int pairs = static_cast<int>(tiles < most ? tiles : most);
  return launch_ex(kern, dim3(2 * pairs), dim3(Cfg::THREADS), Cfg::SMEM, s, true, 2, m.A, m.W, m.C, p);
}

template <int BN, int COLS, bool GELU>
cudaError_t launch_pair_cols(const I8Maps& m, const I8Params& p, bool bf16, bool tma_c, int dev, int sms,
                             cudaStream_t s) {
  if (bf16)
    return tma_c ? launch_pair_i8<BN, COLS, true, GELU, true>(m, p, dev, sms, s)
                 : launch_pair_i8<BN, COLS, true, GELU, false>(m, p, dev, sms, s);
  return tma_c ? launch_pair_i8<BN, COLS, false, GELU, true>(m, p, dev, sms, s)
               : launch_pair_i8<BN, COLS, false, GELU, false>(m, p, dev, sms, s);
}

// Columns of an epilogue warp. For the 256-wide tile, eight warps of 128 columns leave room for a fifth stage;
// sixteen of 64 columns finish a tile sooner, which counts when the GELU takes longer than the tile's MMAs: 8192 x
// 4096 with GELU, K = 384: 25.5 us with sixteen, 27.5 with eight; K = 768: 30.1 / 32.8; K = 1024: 34.9 / 36.4;
// K = 4096: 107.9 / 100.3. Without GELU eight are as fast at K = 384 (50.5 us for 68451 x 1536) and faster above.
int pair_cols(int bn, int K, bool gelu) { return bn < 256 || (gelu && K < 1280) ? 64 : 128; }

cudaError_t launch_pair_any(const I8Maps& m, const I8Params& p, int bn, int cols, bool bf16, bool gelu, bool tma_c,
                            int dev, int sms, cudaStream_t s) {
  if (bn == 128)
    return gelu ? launch_pair_cols<128, 64, true>(m, p, bf16, tma_c, dev, sms, s)
                : launch_pair_cols<128, 64, false>(m, p, bf16, tma_c, dev, sms, s);
  if (bn == 192)
    return gelu ? launch_pair_cols<192, 64, true>(m, p, bf16, tma_c, dev, sms, s)
                : launch_pair_cols<192, 64, false>(m, p, bf16, tma_c, dev, sms, s);
  if (!gelu) return launch_pair_cols<256, 128, false>(m, p, bf16, tma_c, dev, sms, s);
  return cols == 128 ? launch_pair_cols<256, 128, true>(m, p, bf16, tma_c, dev, sms, s)
                     : launch_pair_cols<256, 64, true>(m, p, bf16, tma_c, dev, sms, s);
}

template <int BN, bool BF16, bool GELU>
cudaError_t launch_small_i8(const I8Maps& m, const I8Params& p, int splits, int dev, cudaStream_t s) {
  using Cfg = I8SmallCfg<BN>;
  static OncePerDevice done;
  auto kern = linear_i8_small_kernel<BN, BF16, GELU>;
  const cudaError_t e = opt_in(kern, Cfg::SMEM, done, dev);
  if (e != cudaSuccess) return e;
  int log_splits = 0;
  while ((1 << log_splits) < splits) ++log_splits;
  const dim3 grid(static_cast<unsigned>(((p.N - 1) / 128 + 1) << log_splits), static_cast<unsigned>((p.M - 1) / BN + 1));
  return launch_ex(kern, grid, dim3(Cfg::THREADS), Cfg::SMEM, s, true, splits, m.W, m.A, p, log_splits,
                   m.w, m.ldw);
}

template <int BN>
cudaError_t launch_small_bn(const I8Maps& m, const I8Params& p, bool bf16, bool gelu, int splits, int dev,
                            cudaStream_t s) {
  if (bf16)
    return gelu ? launch_small_i8<BN, true, true>(m, p, splits, dev, s)
                : launch_small_i8<BN, true, false>(m, p, splits, dev, s);
  return gelu ? launch_small_i8<BN, false, true>(m, p, splits, dev, s)
              : launch_small_i8<BN, false, false>(m, p, splits, dev, s);
}

template <int MT, int U>
cudaError_t launch_few(const int8_t* A, int64_t lda, const int8_t* W, int64_t ldw, const I8Params& p, bool bf16,
                       bool gelu, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((int64_t(p.N) + 15) / 16));
  auto go = [&](auto kern) { return launch_ex(kern, grid, dim3(32 * kFewWarps), 0, s, true, 1, A, lda, W, ldw, p); };
  if (bf16) return gelu ? go(linear_i8_few_kernel<MT, U, true, true>) : go(linear_i8_few_kernel<MT, U, true, false>);
  return gelu ? go(linear_i8_few_kernel<MT, U, false, true>) : go(linear_i8_few_kernel<MT, U, false, false>);
}

// Steps in flight of the kernel for one to 16 tokens: as many as a warp has (512 bytes of K each), where the CTAs are
// too few to keep memory busy otherwise. One token, us with 2 / 4 / 8 steps and the weights in L2: 4096 x 4096 4.4 /
// 4.0 / 3.3, 4096 x 1536 3.3 / 2.9 / 4.6, 384 x 384 1.6 / 2.3 / 3.5, 8192 x 2048 (512 CTAs) 3.3 / 4.3 / 7.6; in HBM
// 5.9 / 5.3 / 4.8, 3.9 / 3.7 / 5.2, 2.1 / 3.1 / 5.0, 4.8 / 6.3 / 9.2. At the border, N = 32 SMs: 4700 x 3500 5.0 /
// 4.7 / 3.9, 5000 x 3300 5.2 / 4.7 / 6.1.
int few_steps(int M, int N, int K, int sms) {
  if (M > 8 || K <= 1024 || N > 32 * sms) return 2;
  return K <= 2048 ? 4 : 8;
}

cudaError_t launch_few_any(const int8_t* A, int64_t lda, const int8_t* W, int64_t ldw, const I8Params& p, int tiles,
                           int steps, bool bf16, bool gelu, cudaStream_t s) {
  if (tiles == 2) return launch_few<2, 2>(A, lda, W, ldw, p, bf16, gelu, s);
  if (steps == 2) return launch_few<1, 2>(A, lda, W, ldw, p, bf16, gelu, s);
  return steps == 4 ? launch_few<1, 4>(A, lda, W, ldw, p, bf16, gelu, s)
                    : launch_few<1, 8>(A, lda, W, ldw, p, bf16, gelu, s);
}

// Whether that kernel takes less time than the tcgen05 one (us, few rows / tcgen05), with the weights in L2: 1 x 4096
// x 4096 3.3 / 4.2; 1 x 2048 x 8192 4.7 / 4.4; 4 x 16384 x 4096 8.8 / 8.7; 8 x 4096 x 4096 3.6 / 4.1; 8 x 16384 x
// 4096 9.3 / 7.3; 16 x 1536 x 384 2.3 / 2.3; 16 x 1024 x 1024 2.1 / 2.9; 16 x 1024 x 4096 3.8 / 3.3; 16 x 4096 x 4096
// 5.6 / 4.0; and in HBM, where a model's weights are for single tokens, K = 4096 and N = 4096, 5120, 6144, 8192, 11008,
// 16384: one token 4.7 / 5.2, 6.6 / 6.6, 7.0 / 7.0, 7.8 / 7.9, 12.1 / 9.8, 14.0 / 12.3; eight 5.3 / 5.2, 7.1 / 6.9,
// 7.6 / 7.3, 8.4 / 8.1, 12.7 / 9.9, 14.6 / 12.5. So nothing is lost from 16 Mi weights on.
bool few_is_faster(int M, int N, int K, int sms) {
  const int64_t weights = int64_t(N) * K;
  if (M <= 8) return weights <= (int64_t(16) << 20) && (K <= 4096 || N > 16 * sms);
  return M <= 16 && K <= 2048 && weights <= (int64_t(4) << 20);
}

// Which kernel a call runs: BBH_I8_FEW with `tile` 8-token tiles and `part` steps in flight, BBH_I8_SPLIT with `tile`
// tokens a tile and K in `part` (a power of two) CTAs, BBH_I8_PAIR with `tile` columns a tile and `part` a warp of
// the epilogue.
struct I8Plan {
  int kernel, tile, part;
};

// CTAs of the few-rows kernel that run at once in clusters of 2^log_splits, in clusters (all token tiles
// have an SM to themselves, so one of them answers for all): 148, 74, 33 and 15 on a B200, whose parts
// do not all hold a whole number of large clusters.
int cluster_room(int log_splits, int sms, int dev) {
  using Cfg = I8SmallCfg<64>;
  static OncePerDevice done;
  static OncePerDevice room[4];
  if (log_splits == 0) return sms;
  auto kern = linear_i8_small_kernel<64, false, false>;
  if (opt_in(kern, Cfg::SMEM, done, dev) != cudaSuccess) return sms >> log_splits;
  return max_clusters(kern, 1 << log_splits, Cfg::THREADS, Cfg::SMEM, sms, room[log_splits], dev);
}

// The kernel and tile that take the least time by this model of a launch, in us, fitted to 1,700 times of
// back-to-back launches on a B200 (17 to 68,451 rows, 384 to 8192 columns, K to 8192; within 8 % rms of them; its
// choice is 1 % slower than the fastest on average, 14 % at most):
//   few rows: 1.88 + 0.012 bn (with GELU 0.0175) + (0.107 + 0.0005 bn) k-blocks per CTA, and 0.57 + 0.0035 bn
//     log2(splits) for a split K (the cluster's barrier and the exchange of partial sums), all clusters running
//     at once;
//   pairs: a tile's MMAs take k-blocks (0.024 + 0.00103 bn), its epilogue 0.00613 bn - 0.26 (with GELU 0.0115 bn
//     - 0.23), the longer of them in every round of tiles but one, in which both count; 2.32 a launch, 0.55 a round.
// E.g. 64 x 4096 x 4096: bn 64 in 4 parts 5.4 us, bn 32 in 2 parts 5.5, bn 64 whole 6.4; 1024 x 1024 x 4096: bn 64
// whole 6.8 us, bn 128 in 2 parts 7.7, pairs with bn 256 12.8; pairs, 1024 x 4096 x 1024 with GELU: bn 128 7.3 us,
// 192 8.9, 256 8.3; 4096 x 4096 x 1024 with GELU: 17.8, 17.1, 18.1; 8192 x 4096 x 4096: 91.6, 90.0, 83.4.
I8Plan choose_plan(int M, int N, int K, bool gelu, int sms, int dev) {
  if (few_is_faster(M, N, K, sms)) return {BBH_I8_FEW, M > 8 ? 2 : 1, few_steps(M, N, K, sms)};
  const int k_blocks = (K + kBK - 1) / kBK;
  I8Plan best{};
  double best_us = DBL_MAX;
  auto consider = [&](double us, const I8Plan& plan) {
    if (us >= best_us) return;
    best_us = us;
    best = plan;
  };
  for (int bn = 256; bn >= 128; bn -= 64) {
    const int64_t tiles = (int64_t(M) + 255) / 256 * ((N - 1) / bn + 1);
    const double rounds = static_cast<double>((tiles - 1) / (sms / 2) + 1);
    const double mma = k_blocks * (0.024 + 0.00103 * bn), epi = gelu ? 0.0115 * bn - 0.23 : 0.00613 * bn - 0.26;
    consider(2.32 + mma + epi + (rounds - 1) * (mma > epi ? mma : epi) + 0.55 * rounds, {BBH_I8_PAIR, bn, pair_cols(bn, K, gelu)});
  }
  const int64_t ch_tiles = (N - 1) / 128 + 1;
  for (int bn = 16; bn <= 128; bn *= 2) {
    const int64_t tiles = ch_tiles * ((int64_t(M) + bn - 1) / bn);
    if (tiles > sms) continue;
    for (int ls = 0; ls <= 3 && (1 << ls) <= k_blocks && tiles <= cluster_room(ls, sms, dev); ++ls) {
      const int blocks = (k_blocks + (1 << ls) - 1) >> ls;
      consider(1.88 + (gelu ? 0.0175 : 0.012) * bn + (0.107 + 0.0005 * bn) * blocks + (ls ? 0.57 + 0.0035 * bn * ls : 0),
               {BBH_I8_SPLIT, bn, 1 << ls});
    }
  }
  return best;
}

}  // namespace
}  // namespace bbh

extern "C" {

int bbh_linear_i8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* W, int64_t ldw,
                  const float* w_scale, const uint16_t* bias, uint16_t* C, int64_t ldc, int M, int N, int K, int gelu,
                  int dtype, void* stream) {
  using namespace bbh;
  if (M < 0 || N < 0 || K < 1 || K > BBH_LINEAR_I8_MAX_K)
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: M and N must be >= 0 and K in [1, 131071]");
  if (dtype != BBH_F16 && dtype != BBH_BF16)
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: dtype must be BBH_F16 or BBH_BF16");
  if (M == 0 || N == 0) return BBH_OK;
  if (!A || !a_scale || !W || !w_scale || !C) return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: null pointer");
  if (lda < K || ldw < K || ldc < N)
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: a row stride is smaller than its row");
  auto bits = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  if (((bits(A) | bits(W)) & 15) || lda % 16 || ldw % 16)
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: A and W must be 16-byte aligned with row strides of whole 16 bytes");
  if (((bits(a_scale) | bits(w_scale)) & 3) || ((bits(C) | bits(bias)) & 1))
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: a pointer is not aligned to its elements");
  const Span c = span(C, ldc, M, N, 2);
  if (overlap(c, span(A, lda, M, K, 1)) || overlap(c, span(W, ldw, N, K, 1)) || overlap(c, span(a_scale, 1, M, 1, 4)) ||
      overlap(c, span(w_scale, 1, N, 1, 4)) || (bias && overlap(c, span(bias, N, 1, N, 2))))
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8: the output overlaps an input");
  int dev = 0, sms = 0;
  int rc = unit_device(&dev, &sms);
  if (rc) return rc;

  I8Params p{a_scale, w_scale, bias, C, ldc, M, N, K, int64_t(N) * K <= kPrefetchBytes};
  const bool bf16 = dtype == BBH_BF16, g = gelu != 0;
  // N % 8: a TMA store ends at a 16-byte boundary, not inside one (it overwrote up to 7 elements of padding)
  const bool tma_c = !(bits(C) & 15) && ldc % 8 == 0 && N % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  I8Maps maps;
  cudaError_t e;
  const I8Plan plan = choose_plan(M, N, K, g, sms, dev);
  if (plan.kernel == BBH_I8_FEW) {
    e = launch_few_any(A, lda, W, ldw, p, plan.tile, plan.part, bf16, g, s);
  } else if (plan.kernel == BBH_I8_SPLIT) {
    maps.w = W;
    maps.ldw = ldw;
    rc = encode_2d_bytes(&maps.W, W, N, K, ldw, 1, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = encode_2d_bytes(&maps.A, A, M, K, lda, 1, kBK, plan.tile, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return internal_fail(rc, "bbh_linear_i8: tensor map encoding failed");
    switch (plan.tile) {
      case 16: e = launch_small_bn<16>(maps, p, bf16, g, plan.part, dev, s); break;
      case 32: e = launch_small_bn<32>(maps, p, bf16, g, plan.part, dev, s); break;
      case 64: e = launch_small_bn<64>(maps, p, bf16, g, plan.part, dev, s); break;
      default: e = launch_small_bn<128>(maps, p, bf16, g, plan.part, dev, s); break;
    }
  } else {
    rc = encode_2d_bytes(&maps.A, A, M, K, lda, 1, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = encode_2d_bytes(&maps.W, W, N, K, ldw, 1, kBK, plan.tile / 2, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc)
      rc = tma_c ? encode_2d_bytes(&maps.C, C, M, N, ldc, 2, 64, 16, CU_TENSOR_MAP_SWIZZLE_128B)
                 : (maps.C = maps.A, BBH_OK);
    if (rc) return internal_fail(rc, "bbh_linear_i8: tensor map encoding failed");
    e = launch_pair_any(maps, p, plan.tile, plan.part, bf16, g, tma_c, dev, sms, s);
  }
  if (e != cudaSuccess) return internal_fail(BBH_ERR_CUDA, std::string("bbh_linear_i8: ") + cudaGetErrorString(e));
  return BBH_OK;
}

int bbh_linear_i8_plan(int M, int N, int K, int gelu, int* plan) {
  using namespace bbh;
  if (M < 1 || N < 1 || K < 1 || K > BBH_LINEAR_I8_MAX_K || !plan)
    return internal_fail(BBH_ERR_ARG, "bbh_linear_i8_plan: M and N must be >= 1, K in [1, 131071], plan not null");
  int dev = 0, sms = 0;
  const int rc = unit_device(&dev, &sms);
  if (rc) return rc;
  const I8Plan p = choose_plan(M, N, K, gelu != 0, sms, dev);
  plan[0] = p.kernel;
  plan[1] = p.tile;
  plan[2] = p.part;
  return BBH_OK;
}

int bbh_linear_i8_device_error(int reset) {
  int v = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, bbh::g_i8_err, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && reset && v) e = cudaMemcpyToSymbol(bbh::g_i8_err, &zero, sizeof(int));
  if (e != cudaSuccess)
    return bbh::internal_fail(BBH_ERR_CUDA, std::string("bbh_linear_i8_device_error: ") + cudaGetErrorString(e));
  return v;
}

}  // extern "C"
