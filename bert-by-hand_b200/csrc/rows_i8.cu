// Row operators of the 8-bit linear path: root-mean-square norm (with the residual added,
// 16-bit or 8-bit output), quantisation of rows to int8 and its inverse.
//
//   v = x + residual (fp32, not rounded)      sum = round16(v)
//   y = v * rstd * w,  rstd = 1 / sqrt(mean(v^2) + eps)
//   q = rint(y / scale), scale = max|y| / 127     (y = x for bbh_quantize_i8)
//
// One pass: a row stays in the registers of its threads between the loads and the stores.
// rstd cancels out of q (q = rint(v w * 127 / max|v w|), scale = max|v w| * rstd / 127), so the
// sum of squares and the maximum are reduced together, with one exchange between the warps
// of a row. All arithmetic is fp32; the only roundings are those of the outputs.
// Bound: HBM bytes (x, residual, sum, y or q; each moved once).
#include "common.cuh"
#include "internal.h"
#include "../../include/bbh.h"

#include <cuda_bf16.h>

#include <cfloat>
#include <climits>

namespace bbh {

enum RowMode : int { kRowNorm = 0, kRowNormI8 = 1, kRowQuant = 2 };

struct RowParams {
  const uint16_t* x;
  const uint16_t* residual;  // null: none
  const uint16_t* weight;    // null: ones
  uint16_t* y;               // kRowNorm
  int8_t* q;                 // 8-bit modes
  float* scale;              // 8-bit modes
  uint16_t* sum;             // written when residual is given and sum is not null
  int64_t ldx, ldr, ldy, ldq, lds;
  int rows, D;
  int group;  // threads of a row: a power of two, 16 .. 512
  float eps;
};

constexpr int kRowBlock = 128;  // threads of a block when a row takes fewer
constexpr int kRowMaxBlock = 512;  // leaves 128 registers a thread: no spills at any width

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(a, b);
}

// max that keeps a NaN of either side (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A thread's 8 values of chunk j. VEC 8: eight consecutive elements, one 16-byte access
// (rows 16-byte aligned, D a multiple of 8). VEC 1: elements a group's width apart, 2-byte
// accesses, which any alignment and width allows.
template <int VEC>
__device__ __forceinline__ int elem(int j, int i, int t, int group) {
  return VEC == 8 ? 8 * (j * group + t) + i : (8 * j + i) * group + t;
}

template <int VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int j, int t, int group, int D) {
  uint4 u = make_uint4(0, 0, 0, 0);
  if constexpr (VEC == 8) {
    const int e = elem<8>(j, 0, t, group);
    if (e < D) u = *reinterpret_cast<const uint4*>(row + e);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = elem<1>(j, i, t, group);
      if (e < D) w[i >> 1] |= static_cast<uint32_t>(row[e]) << (16 * (i & 1));
    }
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return u;
}

template <int VEC, bool BF16>
__device__ __forceinline__ void store8(uint16_t* row, int j, int t, int group, int D, const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack16<BF16>(f[2 * i], f[2 * i + 1]);
  if constexpr (VEC == 8) {
    const int e = elem<8>(j, 0, t, group);
    if (e < D) *reinterpret_cast<uint4*>(row + e) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = elem<1>(j, i, t, group);
      if (e < D) row[e] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// rint(f * 127 / top) as the low byte of f * inv + 1.5 * 2^23 (rounded half to even there);
// |f * inv| <= 127 (1 + 2^-23), which rounds to 127 at most. Elements of a 16-bit row meet exact
// halves (top / 2 is 63.5 steps), which inv = 127 / top rounded to fp32 would push to either
// side: TIES adds the rest of 127 / top, so that f * 127 / top is right to fp32 and a half
// stays one (with 11-bit elements every other value is 2^-20 of itself or more away from a half).
template <bool TIES>
__device__ __forceinline__ uint32_t round_byte(float f, float inv, float inv_rest) {
  if constexpr (TIES) return __float_as_uint(fmaf(f, inv, f * inv_rest) + 12582912.f);
  return __float_as_uint(fmaf(f, inv, 12582912.f));
}

template <int VEC, bool TIES>
__device__ __forceinline__ void store_q8(int8_t* row, int j, int t, int group, int D, const float* f, float inv,
                                         float inv_rest) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = inv > 0.f ? round_byte<TIES>(f[i], inv, inv_rest) : 0u;
  if constexpr (VEC == 8) {
    const int e = elem<8>(j, 0, t, group);
    uint2 o;
    o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    if (e < D) *reinterpret_cast<uint2*>(row + e) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = elem<1>(j, i, t, group);
      if (e < D) row[e] = static_cast<int8_t>(b[i]);
    }
  }
}

// Sum of s and maximum of m over the `group` threads of a row (a power of two; groups of more
// than a warp exchange through shared memory). Every thread of the block calls it.
template <bool SUM, bool MAX>
__device__ __forceinline__ void group_reduce(float& s, float& m, int group) {
  __shared__ float2 part[kRowMaxBlock / 32];
  const int lane = threadIdx.x & 31;
  const int width = group < 32 ? group : 32;
  for (int o = width >> 1; o > 0; o >>= 1) {
    if (SUM) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (MAX) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  if (group > 32) {
    const int warps = group >> 5;
    const int warp = threadIdx.x >> 5;
    if (lane == 0) part[warp] = make_float2(s, m);
    __syncthreads();
    const float2 p = part[(warp & ~(warps - 1)) + (lane & (warps - 1))];
    s = p.x;
    m = p.y;
    for (int o = warps >> 1; o > 0; o >>= 1) {
      if (SUM) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (MAX) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
  }
}

// V: 8-element chunks a thread holds (D <= 8 * V * group).
template <int MODE, bool BF16, int V, int VEC>
__global__ void __launch_bounds__(kRowMaxBlock) row_kernel(const RowParams p) {
  pdl_launch_dependents();
  const int group = p.group;
  const int t = threadIdx.x & (group - 1);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x / group) + threadIdx.x / group;
  const bool live = r < p.rows;
  const int D = live ? p.D : 0;  // a group behind the last row loads and stores nothing
  pdl_wait();

  uint4 ux[V], ur[V], uw[V];
#pragma unroll
  for (int j = 0; j < V; ++j) ux[j] = load8<VEC>(p.x + r * p.ldx, j, t, group, D);
  if (MODE != kRowQuant && p.residual) {
#pragma unroll
    for (int j = 0; j < V; ++j) ur[j] = load8<VEC>(p.residual + r * p.ldr, j, t, group, D);
  }
  if (MODE != kRowQuant && p.weight) {
#pragma unroll
    for (int j = 0; j < V; ++j) uw[j] = load8<VEC>(p.weight, j, t, group, D);
  }

  float f[8 * V];
  float ss = 0.f, top = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float* v = f + 8 * j;
    const uint32_t* a = reinterpret_cast<const uint32_t*>(&ux[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = unpack16<BF16>(a[i]);
      v[2 * i] = u.x;
      v[2 * i + 1] = u.y;
    }
    if constexpr (MODE != kRowQuant) {
      if (p.residual) {
        const uint32_t* b = reinterpret_cast<const uint32_t*>(&ur[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 u = unpack16<BF16>(b[i]);
          v[2 * i] += u.x;
          v[2 * i + 1] += u.y;
        }
        if (p.sum) store8<VEC, BF16>(p.sum + r * p.lds, j, t, group, D, v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
      if (p.weight) {
        const uint32_t* b = reinterpret_cast<const uint32_t*>(&uw[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 u = unpack16<BF16>(b[i]);
          v[2 * i] *= u.x;
          v[2 * i + 1] *= u.y;
        }
      }
    }
    if constexpr (MODE != kRowNorm) {
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
    }
  }
  group_reduce<MODE != kRowQuant, MODE != kRowNorm>(ss, top, group);
  const float rstd = MODE == kRowQuant ? 1.f : rsqrtf(ss / static_cast<float>(p.D) + p.eps);

  if constexpr (MODE == kRowNorm) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[8 * j + i] *= rstd;
      store8<VEC, BF16>(p.y + r * p.ldy, j, t, group, D, f + 8 * j);
    }
  } else {
    // A row whose largest magnitude is below 2^-120 (127 / top would near the end of fp32) is
    // stored as zeros with scale 0; one with a NaN or an infinity as zeros with scale NaN, so
    // that whatever is computed from it is NaN too.
    const bool finite = top <= FLT_MAX;
    const float inv = finite && top >= 0x1p-120f ? 127.f / top : 0.f;
    const float rest = inv > 0.f ? fmaf(-inv, top, 127.f) / top : 0.f;
    if (live && t == 0)
      p.scale[r] = finite ? (inv > 0.f ? top / 127.f : 0.f) * rstd : __int_as_float(0x7fc00000);
#pragma unroll
    for (int j = 0; j < V; ++j) store_q8<VEC, MODE == kRowQuant>(p.q + r * p.ldq, j, t, group, D, f + 8 * j, inv, rest);
  }
}

// y = q * scale, one group of threads per row, four 8-element chunks in flight per thread.
struct DequantParams {
  const int8_t* q;
  const float* scale;
  uint16_t* y;
  int64_t ldq, ldy;
  int rows, D, group;
};

template <bool BF16, int VEC>
__global__ void __launch_bounds__(kRowMaxBlock) dequant_kernel(const DequantParams p) {
  pdl_launch_dependents();
  const int group = p.group;
  const int t = threadIdx.x & (group - 1);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x / group) + threadIdx.x / group;
  pdl_wait();
  if (r >= p.rows) return;
  const int8_t* q = p.q + r * p.ldq;
  uint16_t* y = p.y + r * p.ldy;
  const float s = p.scale[r];
  for (int j0 = 0; elem<VEC>(j0, 0, t, group) < p.D; j0 += 4) {
    uint2 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u[k] = make_uint2(0, 0);
      if constexpr (VEC == 8) {
        const int e = elem<8>(j0 + k, 0, t, group);
        if (e < p.D) u[k] = *reinterpret_cast<const uint2*>(q + e);
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = elem<1>(j0 + k, i, t, group);
          if (e < p.D) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(q[e])) << (8 * (i & 3));
        }
        u[k] = make_uint2(w[0], w[1]);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = i < 4 ? u[k].x : u[k].y;
        f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * (i & 3)))) * s;
      }
      store8<VEC, BF16>(y, j0 + k, t, group, p.D, f);
    }
  }
}

namespace {

// Threads of a row and 8-element chunks a thread: the smallest power of two that leaves at
// most four chunks a thread (eight in rows of more than 16,384 elements); with few rows, more threads a row (down to one chunk each), since
// the chip then waits on one row's loads and not on bandwidth.
int row_group(int rows, int D, int num_sms, int* chunks) {
  const int n = (D + 7) / 8;
  int g = 16;
  while (g < kRowMaxBlock && (n + g - 1) / g > 4) g *= 2;
  while (rows <= 2 * num_sms && g < kRowMaxBlock && (n + g - 1) / g > 1) g *= 2;
  *chunks = (n + g - 1) / g;
  return g;
}

template <int MODE, bool BF16, int VEC>
cudaError_t launch_rows(const RowParams& p, int chunks, cudaStream_t s) {
  const int block = p.group < kRowBlock ? kRowBlock : p.group;
  const int per = block / p.group;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.rows) + per - 1) / per));
  switch (chunks) {
    case 1: return launch_ex(row_kernel<MODE, BF16, 1, VEC>, grid, dim3(block), 0, s, true, 1, p);
    case 2: return launch_ex(row_kernel<MODE, BF16, 2, VEC>, grid, dim3(block), 0, s, true, 1, p);
    case 3: return launch_ex(row_kernel<MODE, BF16, 3, VEC>, grid, dim3(block), 0, s, true, 1, p);
    case 4: return launch_ex(row_kernel<MODE, BF16, 4, VEC>, grid, dim3(block), 0, s, true, 1, p);
    default: return launch_ex(row_kernel<MODE, BF16, 8, VEC>, grid, dim3(block), 0, s, true, 1, p);
  }
}

template <int MODE>
cudaError_t launch_mode(const RowParams& p, bool bf16, bool wide, int chunks, cudaStream_t s) {
  if (bf16) return wide ? launch_rows<MODE, true, 8>(p, chunks, s) : launch_rows<MODE, true, 1>(p, chunks, s);
  return wide ? launch_rows<MODE, false, 8>(p, chunks, s) : launch_rows<MODE, false, 1>(p, chunks, s);
}

bool off(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// An output may be an input itself (same rows, same stride: each element is read before it
// is written, by one thread); any other overlap is refused.
bool clash(const Span& out, const void* out_p, const Span& in, const void* in_p, bool same_ok) {
  if (!in_p || !out_p || !overlap(out, in)) return false;
  return !(same_ok && out.lo == in.lo && out.ld == in.ld);
}

int check_rows(const char* who, int rows, int D, int dtype) {
  if (rows < 0 || D < 1 || D > BBH_ROW_MAX_D)
    return internal_fail(BBH_ERR_ARG, std::string(who) + ": rows must be >= 0 and D in [1, 32768]");
  if (dtype != BBH_F16 && dtype != BBH_BF16)
    return internal_fail(BBH_ERR_ARG, std::string(who) + ": dtype must be BBH_F16 or BBH_BF16");
  return BBH_OK;
}

int run_rows(const char* who, int mode, RowParams p, int dtype, void* stream) {
  const std::string w(who);
  int rc = check_rows(who, p.rows, p.D, dtype);
  if (rc) return rc;
  if (p.rows == 0) return BBH_OK;
  const bool i8 = mode != kRowNorm;
  if (!p.x || (i8 ? (!p.q || !p.scale) : !p.y)) return internal_fail(BBH_ERR_ARG, w + ": null pointer");
  if (p.sum && !p.residual) return internal_fail(BBH_ERR_ARG, w + ": sum needs a residual");
  if (!(p.eps >= 0.f) || p.eps > FLT_MAX) return internal_fail(BBH_ERR_ARG, w + ": eps must be finite and >= 0");
  if (p.ldx < p.D || (p.residual && p.ldr < p.D) || (p.sum && p.lds < p.D) || (i8 ? p.ldq < p.D : p.ldy < p.D))
    return internal_fail(BBH_ERR_ARG, w + ": a row stride is smaller than D");
  if (off(p.x, 2) || off(p.residual, 2) || off(p.weight, 2) || off(p.sum, 2) || off(p.y, 2) || off(p.scale, 4))
    return internal_fail(BBH_ERR_ARG, w + ": a pointer is not aligned to its elements");
  const void* outs[3] = {i8 ? static_cast<void*>(p.q) : p.y, p.sum, p.scale};
  const Span so[3] = {i8 ? span(p.q, p.ldq, p.rows, p.D, 1) : span(p.y, p.ldy, p.rows, p.D, 2),
                      span(p.sum, p.lds, p.rows, p.D, 2), span(p.scale, 1, p.rows, 1, 4)};
  const void* ins[3] = {p.x, p.residual, p.weight};
  const Span si[3] = {span(p.x, p.ldx, p.rows, p.D, 2), span(p.residual, p.ldr, p.rows, p.D, 2),
                      span(p.weight, p.D, 1, p.D, 2)};
  for (int o = 0; o < 3; ++o) {
    for (int i = 0; i < 3; ++i)
      if (clash(so[o], outs[o], si[i], ins[i], i < 2 && (o == 1 || (o == 0 && !i8))))
        return internal_fail(BBH_ERR_ARG, w + ": an output overlaps an input");
    for (int i = o + 1; i < 3; ++i)
      if (clash(so[o], outs[o], so[i], outs[i], false))
        return internal_fail(BBH_ERR_ARG, w + ": two outputs overlap");
  }
  int dev = 0, sms = 0;
  rc = unit_device(&dev, &sms);
  if (rc) return rc;
  const bool wide = p.D % 8 == 0 && !off(p.x, 16) && !off(p.residual, 16) && !off(p.weight, 16) && !off(p.sum, 16) &&
                    !off(p.y, 16) && !off(p.q, 8) && p.ldx % 8 == 0 && (!p.residual || p.ldr % 8 == 0) &&
                    (!p.sum || p.lds % 8 == 0) && (i8 ? p.ldq % 8 == 0 : p.ldy % 8 == 0);
  int chunks = 0;
  p.group = row_group(p.rows, p.D, sms, &chunks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == BBH_BF16;
  const cudaError_t e = mode == kRowNorm     ? launch_mode<kRowNorm>(p, bf, wide, chunks, s)
                        : mode == kRowNormI8 ? launch_mode<kRowNormI8>(p, bf, wide, chunks, s)
                                             : launch_mode<kRowQuant>(p, bf, wide, chunks, s);
  if (e != cudaSuccess) return internal_fail(BBH_ERR_CUDA, w + ": " + cudaGetErrorString(e));
  return BBH_OK;
}

}  // namespace
}  // namespace bbh

extern "C" {

int bbh_rmsnorm(const uint16_t* x, int64_t ldx, const uint16_t* residual, int64_t ldr, const uint16_t* weight,
                uint16_t* y, int64_t ldy, uint16_t* sum, int64_t lds, int M, int D, float eps, int dtype,
                void* stream) {
  bbh::RowParams p{x, residual, weight, y, nullptr, nullptr, sum, ldx, ldr, ldy, 0, lds, M, D, 0, eps};
  return bbh::run_rows("bbh_rmsnorm", bbh::kRowNorm, p, dtype, stream);
}

int bbh_rmsnorm_i8(const uint16_t* x, int64_t ldx, const uint16_t* residual, int64_t ldr, const uint16_t* weight,
                   int8_t* q, int64_t ldq, float* scale, uint16_t* sum, int64_t lds, int M, int D, float eps,
                   int dtype, void* stream) {
  bbh::RowParams p{x, residual, weight, nullptr, q, scale, sum, ldx, ldr, 0, ldq, lds, M, D, 0, eps};
  return bbh::run_rows("bbh_rmsnorm_i8", bbh::kRowNormI8, p, dtype, stream);
}

int bbh_quantize_i8(const uint16_t* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int M, int D, int dtype,
                    void* stream) {
  bbh::RowParams p{x, nullptr, nullptr, nullptr, q, scale, nullptr, ldx, 0, 0, ldq, 0, M, D, 0, 0.f};
  return bbh::run_rows("bbh_quantize_i8", bbh::kRowQuant, p, dtype, stream);
}

int bbh_dequantize_i8(const int8_t* q, int64_t ldq, const float* scale, uint16_t* y, int64_t ldy, int M, int D,
                      int dtype, void* stream) {
  using namespace bbh;
  int rc = check_rows("bbh_dequantize_i8", M, D, dtype);
  if (rc) return rc;
  if (M == 0) return BBH_OK;
  if (!q || !scale || !y) return internal_fail(BBH_ERR_ARG, "bbh_dequantize_i8: null pointer");
  if (ldq < D || ldy < D) return internal_fail(BBH_ERR_ARG, "bbh_dequantize_i8: a row stride is smaller than D");
  if (off(scale, 4) || off(y, 2))
    return internal_fail(BBH_ERR_ARG, "bbh_dequantize_i8: a pointer is not aligned to its elements");
  const Span sy = span(y, ldy, M, D, 2);
  if (clash(sy, y, span(q, ldq, M, D, 1), q, false) || clash(sy, y, span(scale, 1, M, 1, 4), scale, false))
    return internal_fail(BBH_ERR_ARG, "bbh_dequantize_i8: the output overlaps an input");
  int dev = 0, sms = 0;
  rc = unit_device(&dev, &sms);
  if (rc) return rc;
  const bool wide = D % 8 == 0 && !off(q, 8) && !off(y, 16) && ldq % 8 == 0 && ldy % 8 == 0;
  int chunks = 0;
  DequantParams p{q, scale, y, ldq, ldy, M, D, row_group(M, D, sms, &chunks)};
  const int block = p.group < kRowBlock ? kRowBlock : p.group;
  const int per = block / p.group;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(M) + per - 1) / per));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == BBH_BF16;
  auto kern = bf ? (wide ? dequant_kernel<true, 8> : dequant_kernel<true, 1>)
                 : (wide ? dequant_kernel<false, 8> : dequant_kernel<false, 1>);
  const cudaError_t e = launch_ex(kern, grid, dim3(block), 0, s, true, 1, p);
  if (e != cudaSuccess)
    return internal_fail(BBH_ERR_CUDA, std::string("bbh_dequantize_i8: ") + cudaGetErrorString(e));
  return BBH_OK;
}

}  // extern "C"
