// Linear layer on 8-bit integers, the W8A8 counterpart of bbh_linear:
//   C[m, n] = round16( a_scale[m] * w_scale[n] * sum_k A[m, k] W[n, k] + bias[n] )  (+ erf-GELU)
// The sum is exact (tcgen05.mma kind::i8, int32 accumulators in TMEM; |sum| <= 128^2 K < 2^31
// for K <= 131071), so the result does not depend on tile shape, split or order.
//
// Two kernels, both fed by 128-byte-swizzled TMA tiles of 128 int8 along K:
//  * linear_i8_pair_kernel -- many rows: persistent SM pairs (cta_group::2) on 256 x BN tiles,
//    two TMEM accumulators so that the epilogue of a tile runs under the MMAs of the next;
//  * linear_i8_small_kernel -- few rows: the weights are the MMA's 128-row operand and BN tokens
//    its columns, K split over the CTAs of a cluster, partial sums added in shared memory
//    (int32: exact in any order).
// Every wait is bounded (mbar_wait); one that runs out sets the device error word and the
// kernel returns.
#include "common.cuh"
#include "epilogue.cuh"
#include "internal.h"
#include "../../include/bbh.h"

#include <cuda_bf16.h>

#include <string>

namespace bbh {

struct I8Params {
  const float* a_scale;    // [M]
  const float* w_scale;    // [N]
  const uint16_t* bias;    // [N] or null, the output's type
  uint16_t* C;
  int64_t ldc;
  int M, N, K;
};

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

// Instruction descriptor, kind::i8: signed A and B, int32 D, both K-major.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

constexpr int kBK = 128;  // int8 per k-block: one 128-byte swizzle row
constexpr int kMmaK = 32;

// erf-GELU of the layer's output. fp16: gelu_half2, the one of bbh_linear. bf16: the same fit,
//   y(x) = x p(x^2), gelu = x/2 (1 + tanh y), evaluated in fp32 (no clamp: p > 0 everywhere).
__device__ __forceinline__ float gelu_f32(float x) {
  const float u = x * x;
  float z = fmaf(1.19315286e-06f, u, -3.22934132e-05f);
  z = fmaf(z, u, -1.12335663e-04f);
  z = fmaf(z, u, 3.64356497e-02f);
  z = fmaf(z, u, 7.97853484e-01f);
  float t;
  asm("tanh.approx.f32 %0, %1;" : "=f"(t) : "f"(z * x));
  return fmaf(0.5f * x, t, 0.5f * x);
}

// Two outputs rounded to 16 bits, packed (a in the low half).
template <bool BF16, bool GELU>
__device__ __forceinline__ uint32_t finish2(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = GELU ? __floats2bfloat162_rn(gelu_f32(a), gelu_f32(b)) : __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const uint32_t w = pack_half2(a, b);
  return GELU ? gelu_half2(w) : w;
}

template <bool BF16>
__device__ __forceinline__ float bias_f32(const uint16_t* b) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(*b) << 16);
  return __half2float(*reinterpret_cast<const __half*>(b));
}

// (acc * a_scale) * w_scale + bias, the same in both kernels (bit for bit)
__device__ __forceinline__ float dequant(int acc, float sa, float sw, float bias) {
  return fmaf(__int2float_rn(acc) * sa, sw, bias);
}

// ====================================================================== many rows: SM pairs

template <int BN>
struct I8PairCfg {
  static constexpr int BM = 128;         // accumulator rows per CTA (256 per pair)
  static constexpr int B_ROWS = BN / 2;  // W rows held by each CTA
  static constexpr int A_BYTES = BM * kBK;
  static constexpr int B_BYTES = B_ROWS * kBK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int PARTS = BN / 64;  // epilogue warps per TMEM lane quadrant, 64 columns each
  static constexpr int EPI_WARPS = 4 * PARTS;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STAGING_BYTES = EPI_WARPS * 4096;  // per epilogue warp: 32 rows x 128 B
  static constexpr int COLS_BYTES = EPI_WARPS * 512;      // per epilogue warp: 64 scales, 64 biases
  static constexpr int AUX_BYTES = 512 /*barriers*/ + COLS_BYTES;
  static constexpr int RING_BYTES = 227 * 1024 - 1024 - STAGING_BYTES - AUX_BYTES;
  static constexpr int STAGES = RING_BYTES / STAGE_BYTES;
  static constexpr int NACC = 2;
  static constexpr int TMEM_COLS = 512;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + STAGING_BYTES + AUX_BYTES;
  static_assert(BN % 64 == 0 && BN <= 256 && NACC * BN <= TMEM_COLS, "pair tile");
  static_assert(STAGES >= 3 && SMEM <= 227 * 1024, "shared memory");
  static_assert((2 * STAGES + 2 * NACC) * 8 + 8 <= 512, "barriers");
};

// TMA_C: C is written with TMA stores (16-byte aligned rows); otherwise row by row from the
// staging buffer with 2-byte stores, which any N and alignment allows.
template <int BN, bool BF16, bool GELU, bool TMA_C>
__global__ void __launch_bounds__(I8PairCfg<BN>::THREADS, 1)
    linear_i8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmC, const I8Params p) {
  using Cfg = I8PairCfg<BN>;
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
  cluster_sync_all();  // both CTAs' barriers initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  auto tile_m0 = [&](int t) { return (t / n_tiles) * (2 * Cfg::BM) + half * Cfg::BM; };
  auto tile_n0 = [&](int t) { return (t % n_tiles) * BN; };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      const uint32_t full0 = mapa_shared(smem_u32(full_bar), 0);
      int stage = 0;
      uint32_t phase = 0;
      for (int tile = first_tile; tile < num_tiles && !*abort_flag; tile += tile_step) {
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
    if (leader && lane == 0) {
      constexpr uint32_t idesc = idesc_i8(2 * Cfg::BM, BN);
      const uint32_t empty_peer = mapa_shared(smem_u32(empty_bar), 1);
      const uint32_t accf_peer = mapa_shared(smem_u32(accf_bar), 1);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
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
          const uint32_t a_addr = smem_u32(sA + stage * Cfg::A_BYTES);
          const uint32_t b_addr = smem_u32(sB + stage * Cfg::B_BYTES);
#pragma unroll
          for (int k = 0; k < kBK / kMmaK; ++k)
            tc_mma_i8_pair(d_tmem, sw128_kmajor_desc(a_addr + k * kMmaK), sw128_kmajor_desc(b_addr + k * kMmaK), idesc,
                           (kb | k) != 0 ? 1u : 0u);
          tc_commit_pair(smem_u32(&empty_bar[stage]));
          tc_commit_pair(empty_peer + stage * 8);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        tc_commit_pair(smem_u32(&accf_bar[acc]));
        tc_commit_pair(accf_peer + acc * 8);
        if (++acc == NACC) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quad = warp & 3;         // TMEM lane quadrant this warp may access
    const int part = (warp - 2) >> 2;  // which 64 columns of the tile
    const int we = warp - 2;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    ChunkStore cst{s_stage + we * 4096, &tmC, lane};
    float* s_sw = s_cols + we * 128;  // this warp's 64 channel scales, then 64 biases
    float* s_b = s_sw + 64;
    const uint32_t acce0 = mapa_shared(smem_u32(acce_bar), 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
      const int row0 = tile_m0(tile) + quad * 32;
      const int c0 = tile_n0(tile) + part * 64;
      // this tile's scales, fetched while the MMAs run
      const float sa = row0 + lane < p.M ? __ldg(p.a_scale + row0 + lane) : 0.f;
      __syncwarp();  // the previous tile's reads of s_sw / s_b are done
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 32 * h + lane;
        s_sw[32 * h + lane] = c < p.N ? __ldg(p.w_scale + c) : 0.f;
        s_b[32 * h + lane] = p.bias && c < p.N ? bias_f32<BF16>(p.bias + c) : 0.f;
      }
      __syncwarp();
      if (!mbar_wait(&accf_bar[acc], acc_phase, abort_flag, &g_i8_err)) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + lane_off + acc * BN + part * 64;
      float v[64];  // int32 accumulators
      tmem_ld64(tacc, tacc + 32, v);
      // accumulator read: release it to the even CTA's MMA thread
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acce0 + acc * 8);
      uint32_t w[32];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float4 sw = *reinterpret_cast<const float4*>(s_sw + 4 * j);
        const float4 b = *reinterpret_cast<const float4*>(s_b + 4 * j);
        const float y0 = dequant(__float_as_int(v[4 * j]), sa, sw.x, b.x);
        const float y1 = dequant(__float_as_int(v[4 * j + 1]), sa, sw.y, b.y);
        const float y2 = dequant(__float_as_int(v[4 * j + 2]), sa, sw.z, b.z);
        const float y3 = dequant(__float_as_int(v[4 * j + 3]), sa, sw.w, b.w);
        w[2 * j] = finish2<BF16, GELU>(y0, y1);
        w[2 * j + 1] = finish2<BF16, GELU>(y2, y3);
      }
      if constexpr (TMA_C) {
        if (c0 < p.N && row0 < p.M) cst.put64(w, c0, row0);
      } else {
        // 32 rows x 64 columns through the staging buffer (16-byte piece c of row r at piece
        // c ^ (r & 7)), then row by row: 32 neighbouring 2-byte stores at a time
        uint8_t* rowp = cst.buf + lane * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(rowp + ((c ^ (lane & 7)) << 4)) =
              make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        __syncwarp();
        const int rows = min(32, p.M - row0);
        for (int r = 0; r < rows; ++r) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = 32 * h + lane;
            const uint16_t o = *reinterpret_cast<const uint16_t*>(cst.buf + r * 128 + (((col >> 3) ^ (r & 7)) << 4) +
                                                                  (col & 7) * 2);
            if (c0 + col < p.N) p.C[static_cast<int64_t>(row0 + r) * p.ldc + c0 + col] = o;
          }
        }
        __syncwarp();
      }
      if (++acc == NACC) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (TMA_C) cst.drain();
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
  cluster_sync_all();  // the peer no longer reads or signals this CTA's memory
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
  static constexpr int RED_BYTES = BN * 512;  // partial sums of this CTA's tokens from every CTA of the cluster
  static constexpr int STAGES = (204 * 1024 - RED_BYTES) / STAGE_BYTES > 8 ? 8 : (204 * 1024 - RED_BYTES) / STAGE_BYTES;
  static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  static constexpr int THREADS = 64 + 128;
  static constexpr int SMEM = STAGES * STAGE_BYTES + RED_BYTES + 1024 + 256;
  static_assert((BN & (BN - 1)) == 0 && BN >= 16 && BN <= 128, "token tile");
  // One CTA per SM (so TMEM, 128 columns at most, can always be had), see launch_small.
  static_assert(SMEM > 114 * 1024 && SMEM <= 227 * 1024, "shared memory");
};

// grid: x = cluster size * channel tiles, y = token tiles; rank r of a cluster sums the r-th part
// of the k-blocks and finishes the tokens t = r (mod cluster size) of the tile.
template <int BN, bool BF16, bool GELU>
__global__ void __launch_bounds__(I8SmallCfg<BN>::THREADS, 1)
    linear_i8_small_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                           const I8Params p, const int splits) {
  using Cfg = I8SmallCfg<BN>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  int* red = reinterpret_cast<int*>(smem + STAGES * Cfg::STAGE_BYTES);  // [splits][BN / splits][128]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::RED_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* acc_bar = empty_bar + STAGES;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / splits * 128;
  const int m0 = static_cast<int>(blockIdx.y) * BN;
  const int k_blocks = (p.K + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(k_blocks) * rank / splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(k_blocks) * (rank + 1) / splits);

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
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync_all();  // every CTA of the cluster runs: its shared memory may be written
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int tokens = min(BN, p.M - m0);

  if (warp == 0) {
    if (lane == 0) {
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
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(128, BN);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag, &g_i8_err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(sA + stage * Cfg::A_BYTES);
        const uint32_t b_addr = smem_u32(sB + stage * Cfg::B_BYTES);
#pragma unroll
        for (int k = 0; k < kBK / kMmaK; ++k)
          tc_mma_i8(tmem, sw128_kmajor_desc(a_addr + k * kMmaK), sw128_kmajor_desc(b_addr + k * kMmaK), idesc,
                    (kb != kb0 || k) ? 1u : 0u);
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

  // Epilogue threads: lane of TMEM = output channel, column = token.
  const int quad = warp & 3;
  const int ch = quad * 32 + lane;
  const int n = n0 + ch;
  const bool epi = warp >= 2;
  bool ok = false;
  float sw = 0.f, bias = 0.f;
  if (epi) {
    if (n < p.N) {
      sw = __ldg(p.w_scale + n);
      bias = p.bias ? bias_f32<BF16>(p.bias + n) : 0.f;
    }
    ok = mbar_wait(acc_bar, 0, abort_flag, &g_i8_err);
    __syncwarp();
    tc_fence_after();
  }
  // two tokens of one channel: 2-byte stores, 32 neighbouring channels per warp
  auto put = [&](int t, int a0, int a1) {
    const float s0 = __ldg(p.a_scale + m0 + t);
    const bool two = t + splits < tokens;
    const float s1 = two ? __ldg(p.a_scale + m0 + t + splits) : 0.f;
    const uint32_t w = finish2<BF16, GELU>(dequant(a0, s0, sw, bias), dequant(a1, s1, sw, bias));
    uint16_t* c = p.C + static_cast<int64_t>(m0 + t) * p.ldc + n;
    if (n < p.N) {
      c[0] = static_cast<uint16_t>(w);
      if (two) c[splits * p.ldc] = static_cast<uint16_t>(w >> 16);
    }
  };
  const uint32_t tacc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const bool all_ok = __all_sync(0xffffffffu, ok);
  if (epi && all_ok) {
#pragma unroll 1
    for (int c = 0; c < tokens; c += 32) {  // BN = 16: the 16 columns behind the tile are not used
      float v[32];
      tmem_ld32(tacc + c, v);
      if (splits == 1) {
#pragma unroll
        for (int t = 0; t < 32; t += 2)
          if (c + t < tokens) put(c + t, __float_as_int(v[t]), __float_as_int(v[t + 1]));
      } else {
        const uint32_t own = smem_u32(red + (rank * (BN / splits)) * 128 + ch);
#pragma unroll
        for (int t = 0; t < 32; ++t)
          if (c + t < tokens) {
            const int to = (c + t) & (splits - 1), slot = (c + t) / splits;
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(mapa_shared(own + slot * 512, to)),
                         "r"(__float_as_int(v[t]))
                         : "memory");
          }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync_all();  // all partial sums are in place
    if (epi) {
      const int mine = (tokens - rank + splits - 1) / splits;  // tokens rank, rank + splits, ...
      for (int s = 0; s < mine; s += 2) {
        int a0 = 0, a1 = 0;
        for (int src = 0; src < splits; ++src) {
          const int* part = red + (src * (BN / splits) + s) * 128 + ch;
          a0 += part[0];
          if (s + 1 < mine) a1 += part[128];
        }
        put(rank + s * splits, a0, a1);
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

// ======================================================================== host side
namespace {

// Once per device and kernel: opt in to the kernel's shared memory.
template <typename K>
cudaError_t opt_in(K kern, int smem, bool (&done)[64], int dev) {
  if (done[dev]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) done[dev] = true;
  return e;
}

// Pairs of SMs that can run a kernel at once, asked once per device and kernel.
template <typename K>
int max_pairs(K kern, int threads, int smem, int sms, int (&cache)[64], int dev) {
  if (cache[dev]) return cache[dev];
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(sms & ~1);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = sms / 2;
  }
  return cache[dev] = n;
}

struct I8Maps {
  CUtensorMap A, W, C;
};

template <int BN, bool BF16, bool GELU, bool TMA_C>
cudaError_t launch_pair_i8(const I8Maps& m, const I8Params& p, int dev, int sms, cudaStream_t s) {
  using Cfg = I8PairCfg<BN>;
  static bool done[64] = {};
  auto kern = linear_i8_pair_kernel<BN, BF16, GELU, TMA_C>;
  const cudaError_t e = opt_in(kern, Cfg::SMEM, done, dev);
  if (e != cudaSuccess) return e;
  static int pairs_of[64] = {};
  const int64_t tiles = (int64_t(p.M) + 255) / 256 * ((p.N - 1) / BN + 1);
  const int most = max_pairs(kern, Cfg::THREADS, Cfg::SMEM, sms, pairs_of, dev);
  const int pairs = static_cast<int>(tiles < most ? tiles : most);
  return launch_ex(kern, dim3(2 * pairs), dim3(Cfg::THREADS), Cfg::SMEM, s, true, 2, m.A, m.W, m.C, p);
}

template <int BN>
cudaError_t launch_pair_bn(const I8Maps& m, const I8Params& p, bool bf16, bool gelu, bool tma_c, int dev, int sms,
                           cudaStream_t s) {
  switch ((bf16 ? 4 : 0) + (gelu ? 2 : 0) + (tma_c ? 1 : 0)) {
    case 0: return launch_pair_i8<BN, false, false, false>(m, p, dev, sms, s);
    case 1: return launch_pair_i8<BN, false, false, true>(m, p, dev, sms, s);
    case 2: return launch_pair_i8<BN, false, true, false>(m, p, dev, sms, s);
    case 3: return launch_pair_i8<BN, false, true, true>(m, p, dev, sms, s);
    case 4: return launch_pair_i8<BN, true, false, false>(m, p, dev, sms, s);
    case 5: return launch_pair_i8<BN, true, false, true>(m, p, dev, sms, s);
    case 6: return launch_pair_i8<BN, true, true, false>(m, p, dev, sms, s);
    default: return launch_pair_i8<BN, true, true, true>(m, p, dev, sms, s);
  }
}

template <int BN, bool BF16, bool GELU>
cudaError_t launch_small_i8(const I8Maps& m, const I8Params& p, int splits, int dev, cudaStream_t s) {
  using Cfg = I8SmallCfg<BN>;
  static bool done[64] = {};
  auto kern = linear_i8_small_kernel<BN, BF16, GELU>;
  const cudaError_t e = opt_in(kern, Cfg::SMEM, done, dev);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>(splits * ((p.N - 1) / 128 + 1)), static_cast<unsigned>((p.M - 1) / BN + 1));
  return launch_ex(kern, grid, dim3(Cfg::THREADS), Cfg::SMEM, s, true, splits, m.W, m.A, p, splits);
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

  I8Params p{a_scale, w_scale, bias, C, ldc, M, N, K};
  const bool bf16 = dtype == BBH_BF16, g = gelu != 0;
  const bool tma_c = !(bits(C) & 15) && ldc % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  I8Maps maps;
  cudaError_t e;
  const int ch_tiles = (N - 1) / 128 + 1;
  const int64_t small128 = int64_t(ch_tiles) * ((M - 1) / 128 + 1);
  if (small128 <= sms) {
    // few rows
    const int bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const int k_blocks = (K + kBK - 1) / kBK;
    const int tiles = ch_tiles * ((M - 1) / bn + 1);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 <= k_blocks) splits *= 2;
    rc = encode_2d_bytes(&maps.W, W, N, K, ldw, 1, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = encode_2d_bytes(&maps.A, A, M, K, lda, 1, kBK, bn, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return internal_fail(rc, "bbh_linear_i8: tensor map encoding failed");
    e = bn == 16   ? launch_small_bn<16>(maps, p, bf16, g, splits, dev, s)
        : bn == 32 ? launch_small_bn<32>(maps, p, bf16, g, splits, dev, s)
        : bn == 64 ? launch_small_bn<64>(maps, p, bf16, g, splits, dev, s)
                   : launch_small_bn<128>(maps, p, bf16, g, splits, dev, s);
  } else {
    const int bn = N % 256 && N % 192 == 0 ? 192 : 256;
    rc = encode_2d_bytes(&maps.A, A, M, K, lda, 1, kBK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = encode_2d_bytes(&maps.W, W, N, K, ldw, 1, kBK, bn / 2, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc)
      rc = tma_c ? encode_2d_bytes(&maps.C, C, M, N, ldc, 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B)
                 : (maps.C = maps.A, BBH_OK);
    if (rc) return internal_fail(rc, "bbh_linear_i8: tensor map encoding failed");
    e = bn == 192 ? launch_pair_bn<192>(maps, p, bf16, g, tma_c, dev, sms, s)
                  : launch_pair_bn<256>(maps, p, bf16, g, tma_c, dev, sms, s);
  }
  if (e != cudaSuccess) return internal_fail(BBH_ERR_CUDA, std::string("bbh_linear_i8: ") + cudaGetErrorString(e));
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
