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
// Bound: HBM bytes (x, residual, sum, y or q; each moved once). On a B200 whose copies reach 6.5 TB/s, with tensors that
// change from call to call (more of them than L2 holds): 8192 x 4096 bf16 with a residual rmsnorm 41.7 us = 6.4 TB/s,
// rmsnorm_i8 37.4 = 6.3; without rmsnorm 22.1 = 6.1, rmsnorm_i8 22.0 = 4.6 (its arithmetic per byte is twice that with
// one); quantize_i8 18.2 = 5.5, dequantize_i8 17.6 = 5.7. 20000 x 1023 fp16, rows of every alignment: rmsnorm 18.6 =
// 4.4, rmsnorm_i8 23.9 = 2.6, quantize_i8 16.4 = 3.7 (kShifted below: the weight is realigned for every chunk of
// every row, and q goes through shared memory). The comparisons of variants further down were made with one set of
// tensors, which L2 holds in part: up to a quarter shorter.
#include "common.cuh"
#include "epilogue.cuh"
#include "internal.h"
#include "../../include/bbh.h"

#include <cuda_bf16.h>

#include <cfloat>
#include <climits>

namespace bbh {

enum RowMode : int { kRowNorm = 0, kRowNormI8 = 1, kRowQuant = 2 };

struct RowParams {  // 96 bytes: above, a launch takes the host 0.35 us longer
  const uint16_t* x;
  const uint16_t* residual;  // null: none
  const uint16_t* weight;    // null: ones
  void* out;                 // kRowNorm: 16-bit, else int8
  float* scale;              // 8-bit modes
  uint16_t* sum;             // written when residual is given and sum is not null
  int64_t ldx, ldr, ldo, lds;
  int rows, D;
  int group;  // threads of a row: a power of two, 16 .. 512
  float eps;
};

static_assert(sizeof(RowParams) == 96, "kernel arguments");

constexpr int kRowBlock = 128;  // threads of a block when a row takes fewer
// Leaves 128 registers a thread, 64 where row_kernel asks for two blocks an SM. Spilled: with 2-byte accesses from three
// or four chunks a thread on 100 to 220 bytes, at eight 550 to 1,580; kShifted with four chunks, or with a residual and
// eight, 4 to 48; nothing with aligned rows.
constexpr int kRowMaxBlock = 512;

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

// max(m, |a|, |b|) that keeps a NaN of any of them (fmaxf drops it)
__device__ __forceinline__ float max_abs_nan(float m, float a, float b) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// the same on a packed pair of 16-bit values
template <bool BF16>
__device__ __forceinline__ uint32_t max_abs_nan2(uint32_t m, uint32_t w) {
  uint32_t a = w & 0x7fff7fffu, d;
  if constexpr (BF16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(m), "r"(a));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(m), "r"(a));
  return d;
}

// How a row is cut for its threads, 8 elements a chunk; chunk c = j * group + t is thread t's j-th.
//  kAligned  chunk c is elements 8c .. 8c + 7, one 16-byte access: rows 16-byte aligned, D a multiple of 8.
//  kShifted  the 16-bit tensors' rows start anywhere, but all of them at the same distance from a 16-byte
//            boundary (contiguous tensors of any width do): chunk c is elements head + 8c .., one 16-byte
//            access; the `head` elements in front of the first chunk and the rest behind the last one go
//            to one thread each.
//  kSingle   any strides and alignments: elements `group` apart, 2-byte accesses.
enum Cut : int { kAligned, kShifted, kSingle };

// A thread's place in its row.
struct Place {
  int t, group, D;
  int head;    // elements in front of the first chunk (0 but for kShifted)
  int chunks;  // whole chunks (kAligned, kShifted)
  int edge;    // this thread's element outside the chunks, or -1 (kShifted)
};

template <int CUT>
__device__ __forceinline__ Place place(const uint16_t* row, int t, int group, int D) {
  Place p{t, group, D, 0, D / 8, -1};
  if constexpr (CUT == kShifted) {
    p.head = min(D, static_cast<int>(-(reinterpret_cast<uintptr_t>(row) >> 1) & 7));
    p.chunks = (D - p.head) / 8;
    const int tail = p.head + 8 * p.chunks;
    if (t < 8) {
      if (t < p.head) p.edge = t;
    } else if (t < 16 && tail + t - 8 < D) {
      p.edge = tail + t - 8;
    }
  }
  return p;
}

// First element of the thread's j-th chunk, or -1.
template <int CUT>
__device__ __forceinline__ int chunk_at(const Place& p, int j) {
  const int c = j * p.group + p.t;
  return c < p.chunks ? p.head + 8 * c : -1;
}
// Element i of chunk j, kSingle.
__device__ __forceinline__ int single_at(const Place& p, int j, int i) { return (8 * j + i) * p.group + p.t; }

template <int CUT>
__device__ __forceinline__ uint4 load8(const uint16_t* row, const Place& p, int j) {
  if constexpr (CUT == kSingle) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (single_at(p, j, i) < p.D) w[i >> 1] |= static_cast<uint32_t>(row[single_at(p, j, i)]) << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const int e = chunk_at<CUT>(p, j);
    return e >= 0 ? *reinterpret_cast<const uint4*>(row + e) : make_uint4(0, 0, 0, 0);
  }
}

template <int CUT>
__device__ __forceinline__ void store8(uint16_t* row, const Place& p, int j, uint4 u) {
  if constexpr (CUT == kSingle) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (single_at(p, j, i) < p.D) row[single_at(p, j, i)] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
  } else {
    const int e = chunk_at<CUT>(p, j);
    if (e >= 0) *reinterpret_cast<uint4*>(row + e) = u;
  }
}

// A chunk of the weight, which is 16-byte aligned where the rows may not be (kShifted): elements e .. e + 7
// lie in two neighbouring 16-byte pieces and are taken out of their eight words.
template <int CUT>
__device__ __forceinline__ uint4 load_weight8(const uint16_t* weight, const Place& p, int j) {
  if (CUT != kShifted || (p.head & 7) == 0) return load8<CUT>(weight, p, j);
  const int e = chunk_at<CUT>(p, j);
  if (e < 0) return make_uint4(0, 0, 0, 0);
  const int base = e - p.head;  // a multiple of 8
  const uint4 lo = *reinterpret_cast<const uint4*>(weight + base);
  uint4 hi;
  if (base + 16 <= p.D) {
    hi = *reinterpret_cast<const uint4*>(weight + base + 8);
  } else {  // the piece ends behind the weight
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < p.head; ++i) {
      const uint32_t b = static_cast<uint32_t>(weight[base + 8 + i]) << (16 * (i & 1));
      w[0] |= i < 2 ? b : 0u;
      w[1] |= i >> 1 == 1 ? b : 0u;
      w[2] |= i >> 1 == 2 ? b : 0u;
      w[3] |= i >> 1 == 3 ? b : 0u;
    }
    hi = make_uint4(w[0], w[1], w[2], w[3]);
  }
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  const int words = p.head >> 1;  // 0 .. 3
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = words & 2 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = words & 1 ? w[i + 1] : w[i];
  const uint32_t pick = p.head & 1 ? 0x5432u : 0x3210u;
  return make_uint4(__byte_perm(w[0], w[1], pick), __byte_perm(w[1], w[2], pick), __byte_perm(w[2], w[3], pick),
                    __byte_perm(w[3], w[4], pick));
}

template <bool BF16>
__device__ __forceinline__ float load1(const uint16_t* row, int e) {
  return unpack16<BF16>(row[e]).x;
}
template <bool BF16>
__device__ __forceinline__ void store1(uint16_t* row, int e, float f) {
  row[e] = static_cast<uint16_t>(pack16<BF16>(f, 0.f));
}

template <bool BF16>
__device__ __forceinline__ void unpack8(uint4 u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack16<BF16>(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack16<BF16>(f[0], f[1]), pack16<BF16>(f[2], f[3]), pack16<BF16>(f[4], f[5]),
                    pack16<BF16>(f[6], f[7]));
}

// v *= u, and ss += v[even]^2, ss1 += v[odd]^2, of eight values in packed pairs: half the instructions
// (8192 x 4096 rmsnorm_i8 20.4 us instead of 21.4).
__device__ __forceinline__ void mul8(float* v, const float* u) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 z = f2_split(f2_mul(f2(v[i], v[i + 1]), f2(u[i], u[i + 1])));
    v[i] = z.x;
    v[i + 1] = z.y;
  }
}
__device__ __forceinline__ void squares8(const float* v, float& ss, float& ss1) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const unsigned long long z = f2(v[i], v[i + 1]);
    const float2 t = f2_split(f2_fma(z, z, f2(ss, ss1)));
    ss = t.x;
    ss1 = t.y;
  }
}

// The low bytes of eight words.
__device__ __forceinline__ uint2 low_bytes(const uint32_t* b) {
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// 127 / top from the hardware's reciprocal (off by 2^-23 at most) and 3 * 2^-23 more, so that with its two
// roundings it is above 127 / top by 0 to 5 * 2^-23 of it. Above 2^126 (bf16) the reciprocal would be subnormal, with
// steps of up to 2^-21 of itself: such a top is divided by 16 first, and the quotient at the end.
template <bool BF16>
__device__ __forceinline__ float steps_per_unit(float top) {
  const float unit = BF16 && top > 0x1p125f ? 0x1p-4f : 1.f;
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(top * unit));
  return r * 127.f * (1.f + 3 * 0x1p-23f) * unit;
}

// 127 / top to half an ulp and a little: one Newton step, for values that do not meet exact halves (kRowNormI8).
// With the one above, five times further off, ten times as many values of a norm's output were rounded to the
// other neighbour of a half (about one in 100,000), each of which a layer behind it spreads over its whole row.
__device__ __forceinline__ float steps_per_unit_near(float top) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(top));
  const float inv = r * 127.f;
  return fmaf(fmaf(-inv, top, 127.f), r, inv);
}

// rint(f * 127 / top) of eight values as bytes: the low byte of f * inv + 1.5 * 2^23, one fma that
// rounds half to even, with inv from steps_per_unit; f * inv < 127.0001 rounds to 127.
//
// Elements of a 16-bit row (kRowQuant) meet exact halves, which an inexact inv pushes to either side.
// If 127 does not divide top's significand the only one is |f| = top / 2, 63.5 steps, and inv, being
// above, takes it to 64, the even neighbour; with 11-bit significands every other value is at least
// 2^-20 of itself away from a half, more than inv is off. If 127 divides it (`ties`), f * inv + f * rest,
// with rest what inv lacks of 127 / top, is right to fp32 and a half stays one.
// HALVES: whether exact halves occur (kRowQuant; without, packed pairs are faster, with them slower).
template <bool HALVES>
__device__ __forceinline__ uint2 quantize8(const float* f, float inv, float rest, bool ties) {
  uint32_t b[8];
  if constexpr (!HALVES) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 z = f2_split(f2_fma(f2(f[i], f[i + 1]), f2(inv, inv), f2(12582912.f, 12582912.f)));
      b[i] = __float_as_uint(z.x);
      b[i + 1] = __float_as_uint(z.y);
    }
  } else if (ties) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(fmaf(f[i], inv, f[i] * rest) + 12582912.f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(fmaf(f[i], inv, 12582912.f));
  }
  return low_bytes(b);
}
__device__ __forceinline__ uint8_t quantize1(float f, float inv, float rest, bool ties) {
  return static_cast<uint8_t>(__float_as_uint(ties ? fmaf(f, inv, f * rest) + 12582912.f : fmaf(f, inv, 12582912.f)));
}

// Sum of s and maximum of m over the `group` threads of a row (a power of two from 16 on; groups of
// more than a warp exchange through shared memory). Every thread of the block calls it.
template <bool SUM, bool MAX>
__device__ __forceinline__ void group_reduce(float& s, float& m, int group) {
  __shared__ float2 part[kRowMaxBlock / 32];
  auto step = [&](int o) {
    if (SUM) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (MAX) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  };
  if (group > 16) step(16);
  step(8);
  step(4);
  step(2);
  step(1);
  if (group > 32) {
    const int warps = group >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[warp] = make_float2(s, m);
    __syncthreads();
    const float2 p = part[(warp & ~(warps - 1)) + (lane & (warps - 1))];
    s = p.x;
    m = p.y;
    if (warps > 8) step(8);
    if (warps > 4) step(4);
    if (warps > 2) step(2);
    step(1);
  }
}

// V: 8-element chunks a thread holds. 64 registers up to four chunks (32 warps an SM: with 82, norm of
// 8192 x 4096 took 27.1 us instead of 22.9). RES: with a residual (a kernel of its own: without one 16384 x 1536
// rmsnorm takes 16.4 us instead of 17.4, 20000 x 1023 16.3 instead of 17.5). Where little is done to an element
// its packed form is kept and unpacked twice (16384 x 1536 rmsnorm 16.1; rmsnorm_i8, which would need
// the weight twice as well, 17.9 instead of 15.2).
template <int MODE, bool BF16, int V, int CUT, bool RES>
__global__ void __launch_bounds__(kRowMaxBlock, V <= 4 && CUT != kSingle ? 2 : 1) row_kernel(const RowParams p) {
  // whether the row stays packed in registers and is unpacked a second time for the output
  constexpr bool kTwice = MODE == kRowQuant || (MODE == kRowNorm && !RES);
  pdl_launch_dependents();
  const int group = p.group;
  const int t = threadIdx.x & (group - 1);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x / group) + threadIdx.x / group;
  const bool live = r < p.rows;
  const uint16_t* x = p.x + r * p.ldx;
  const uint16_t* residual = RES ? p.residual + r * p.ldr : nullptr;
  const uint16_t* weight = MODE != kRowQuant ? p.weight : nullptr;
  uint16_t* sum = p.sum + r * p.lds;
  const Place at = place<CUT>(x, t, group, live ? p.D : 0);  // a group behind the last row has no elements
  const bool edge = CUT == kShifted && at.edge >= 0;
  const float inv_D = MODE == kRowQuant ? 0.f : __frcp_rn(static_cast<float>(p.D));
  pdl_wait();

  uint4 ux[V], ur[RES ? V : 1];
#pragma unroll
  for (int j = 0; j < V; ++j) ux[j] = load8<CUT>(x, at, j);
  if constexpr (RES) {
#pragma unroll
    for (int j = 0; j < V; ++j) ur[j] = load8<CUT>(residual, at, j);
  }
  float fe = 0.f;  // the edge element
  if (edge) {
    fe = load1<BF16>(x, at.edge);
    if constexpr (RES) fe += load1<BF16>(residual, at.edge);
  }

  float f[kTwice ? 8 : 8 * V];
  float ss = 0.f, ss1 = 0.f, top = 0.f;
  uint32_t top2 = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float* v = kTwice ? f : f + 8 * j;
    if constexpr (MODE == kRowQuant) {  // the packed values are enough until the scale is known
      top2 = max_abs_nan2<BF16>(top2, ux[j].x);
      top2 = max_abs_nan2<BF16>(top2, ux[j].y);
      top2 = max_abs_nan2<BF16>(top2, ux[j].z);
      top2 = max_abs_nan2<BF16>(top2, ux[j].w);
    } else {
      unpack8<BF16>(ux[j], v);
      if constexpr (RES) {
        float u[8];
        unpack8<BF16>(ur[j], u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += u[i];
        if (p.sum) store8<CUT>(sum, at, j, pack8<BF16>(v));
      }
      squares8(v, ss, ss1);
    }
    if constexpr (MODE == kRowNormI8) {
      if (weight) {
        float u[8];
        unpack8<BF16>(load_weight8<CUT>(weight, at, j), u);
        mul8(v, u);
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2) top = max_abs_nan(top, v[i], v[i + 1]);
    }
  }
  if constexpr (MODE == kRowQuant) {
    const float2 m = unpack16<BF16>(top2);
    top = max_nan(m.x, m.y);
  }
  if (edge) {
    if (RES && p.sum) store1<BF16>(sum, at.edge, fe);
    ss1 = fmaf(fe, fe, ss1);
    if (weight) fe *= load1<BF16>(weight, at.edge);
    top = max_abs_nan(top, fe, 0.f);
  }
  ss += ss1;
  group_reduce<MODE != kRowQuant, MODE != kRowNorm>(ss, top, group);
  const float rstd = MODE == kRowQuant ? 1.f : rsqrtf(ss * inv_D + p.eps);

  // the packed values again: they take half the registers, and the compiler shall not keep the others
  auto again = [&](int j) {
    uint4 u = ux[j];
    asm volatile("" : "+r"(u.x), "+r"(u.y), "+r"(u.z), "+r"(u.w));
    unpack8<BF16>(u, f);
  };
  if constexpr (MODE == kRowNorm) {
    uint16_t* y = static_cast<uint16_t*>(p.out) + r * p.ldo;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float* v = kTwice ? f : f + 8 * j;
      if (kTwice) again(j);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= rstd;
      if (weight) {
        float u[8];
        unpack8<BF16>(load_weight8<CUT>(weight, at, j), u);
        mul8(v, u);
      }
      store8<CUT>(y, at, j, pack8<BF16>(v));
    }
    if (edge) store1<BF16>(y, at.edge, fe * rstd);
  } else {
    // A row whose largest magnitude is below 2^-120 (127 / top would near the end of fp32) is
    // stored as zeros with scale 0; one with a NaN or an infinity as zeros with scale NaN, so
    // that whatever is computed from it is NaN too.
    const bool finite = top <= FLT_MAX;
    const bool zero = !finite || top < 0x1p-120f;
    const float inv = MODE == kRowQuant ? steps_per_unit<BF16>(zero ? 1.f : top) : steps_per_unit_near(zero ? 1.f : top);
    bool ties = false;
    float rest = 0.f;
    if constexpr (MODE == kRowQuant) {
      ties = (((__float_as_uint(top) >> 13) & 0x3ffu) | 0x400u) % 127u == 0;
      if (ties) rest = fmaf(-inv, top, 127.f) / top;
    }
    if (live && t == 0) p.scale[r] = !finite ? __int_as_float(0x7fc00000) : zero ? 0.f : top / 127.f * rstd;
    int8_t* q = static_cast<int8_t*>(p.out) + r * p.ldo;
    if constexpr (CUT == kShifted) {
      // The bytes of a chunk are not where an aligned store of q wants them: through shared memory, element e
      // at byte e + sh, so that chunks are 8-byte pieces there. The rows of q are 8-byte aligned.
      extern __shared__ uint2 s_q[];
      uint2* row = s_q + (threadIdx.x / group) * (V * group + 2);
      const int sh = -at.head & 7, first = sh ? 1 : 0;  // the piece of chunk 0
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (kTwice) again(j);
        if (chunk_at<CUT>(at, j) >= 0) row[first + j * group + t] = quantize8<MODE == kRowQuant>(kTwice ? f : f + 8 * j, inv, rest, ties);
      }
      if (edge) reinterpret_cast<uint8_t*>(row)[at.edge + sh] = quantize1(fe, inv, rest, ties);
      __syncthreads();
      for (int c = t; 8 * c < at.D; c += group) {  // elements 8c ..: bytes sh .. of piece c, then of piece c + 1
        const uint2 a = row[c], b = row[c + 1];
        const uint64_t lo = static_cast<uint64_t>(a.y) << 32 | a.x, hi = static_cast<uint64_t>(b.y) << 32 | b.x;
        uint64_t o = sh ? lo >> (8 * sh) | hi << (64 - 8 * sh) : lo;
        if (zero) o = 0;
        if (8 * c + 8 <= at.D) {
          *reinterpret_cast<uint64_t*>(q + 8 * c) = o;
        } else {
          for (int i = 0; 8 * c + i < at.D; ++i) q[8 * c + i] = static_cast<int8_t>(o >> (8 * i));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (kTwice) again(j);
        uint2 o = quantize8<MODE == kRowQuant>(kTwice ? f : f + 8 * j, inv, rest, ties);
        if (zero) o = make_uint2(0, 0);
        if constexpr (CUT == kAligned) {
          const int e = chunk_at<CUT>(at, j);
          if (e >= 0) *reinterpret_cast<uint2*>(q + e) = o;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (single_at(at, j, i) < at.D)
              q[single_at(at, j, i)] = static_cast<int8_t>((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
        }
      }
    }
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

// Eight bytes of q, whose rows are 8-byte aligned, from element e = base + head on (base a multiple of 8).
__device__ __forceinline__ uint2 load_q8(const int8_t* q, int e, int head, int D) {
  const int base = e - head;
  const uint64_t lo = *reinterpret_cast<const uint64_t*>(q + base);
  uint64_t hi = 0;
  if (head) {
    if (base + 16 <= D) {
      hi = *reinterpret_cast<const uint64_t*>(q + base + 8);
    } else {
      for (int i = 0; i < head; ++i) hi |= static_cast<uint64_t>(static_cast<uint8_t>(q[base + 8 + i])) << (8 * i);
    }
  }
  const uint64_t o = head ? lo >> (8 * head) | hi << (64 - 8 * head) : lo;
  return make_uint2(static_cast<uint32_t>(o), static_cast<uint32_t>(o >> 32));
}

template <bool BF16, int CUT>
__global__ void __launch_bounds__(kRowMaxBlock) dequant_kernel(const DequantParams p) {
  pdl_launch_dependents();
  const int group = p.group;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x / group) + threadIdx.x / group;
  pdl_wait();
  if (r >= p.rows) return;
  const int8_t* q = p.q + r * p.ldq;
  uint16_t* y = p.y + r * p.ldy;
  const Place at = place<CUT>(y, threadIdx.x & (group - 1), group, p.D);
  const float s = p.scale[r];
  const int chunks = CUT == kSingle ? (p.D + 7) / 8 : at.chunks;
  for (int j0 = 0; j0 * group < chunks; j0 += 4) {
    uint2 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u[k] = make_uint2(0, 0);
      if constexpr (CUT == kSingle) {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (single_at(at, j0 + k, i) < p.D)
            w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(q[single_at(at, j0 + k, i)])) << (8 * (i & 3));
        u[k] = make_uint2(w[0], w[1]);
      } else {
        const int e = chunk_at<CUT>(at, j0 + k);
        if (e >= 0) u[k] = load_q8(q, e, CUT == kShifted ? at.head : 0, p.D);
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
      store8<CUT>(y, at, j0 + k, pack8<BF16>(f));
    }
  }
  if (CUT == kShifted && at.edge >= 0) store1<BF16>(y, at.edge, static_cast<float>(q[at.edge]) * s);
}

namespace {

// Threads of a row and 8-element chunks a thread: the smallest power of two that leaves at
// most four chunks a thread (eight in rows of more than 16,384 elements); with few rows, more threads
// a row (down to one chunk each), since the chip then waits on one row's loads and not on bandwidth:
// up to two rows an SM, and the norms, which have more to do, until there are 512 threads an SM
// (rmsnorm_i8 with a residual, 1024 x 1024: 3.2 us instead of 3.6, 2048 x 1024 3.8 / 4.5, 1000 x 1023 3.9 / 5.6;
// quantize_i8 of 1000 x 1023 would take 3.4 instead of 2.7).
// Two chunks instead of four at many rows: 8192 x 4096 rmsnorm_i8 22.7 -> 31.1 us.
int row_group(int rows, int D, int num_sms, bool norm, int* chunks) {
  const int n = (D + 7) / 8;
  int g = 16;
  while (g < kRowMaxBlock && (n + g - 1) / g > 4) g *= 2;
  auto few = [&] { return rows <= 2 * num_sms || (norm && int64_t(rows) * g < int64_t(512) * num_sms); };
  while (few() && g < kRowMaxBlock && (n + g - 1) / g > 1) g *= 2;
  *chunks = (n + g - 1) / g;
  return g;
}

template <int MODE, bool BF16, int CUT, bool RES>
cudaError_t launch_rows(const RowParams& p, int chunks, cudaStream_t s) {
  const int block = p.group < kRowBlock ? kRowBlock : p.group;
  const int per = block / p.group;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.rows) + per - 1) / per));
  auto go = [&](auto kern, int v) {
    const size_t smem = CUT == kShifted && MODE != kRowNorm ? size_t(per) * (v * p.group + 2) * 8 : 0;
    return launch_ex(kern, grid, dim3(block), smem, s, true, 1, p);
  };
  switch (chunks) {
    case 1: return go(row_kernel<MODE, BF16, 1, CUT, RES>, 1);
    case 2: return go(row_kernel<MODE, BF16, 2, CUT, RES>, 2);
    case 3: return go(row_kernel<MODE, BF16, 3, CUT, RES>, 3);
    case 4: return go(row_kernel<MODE, BF16, 4, CUT, RES>, 4);
    default: return go(row_kernel<MODE, BF16, 8, CUT, RES>, 8);
  }
}

template <int MODE, bool BF16, int CUT>
cudaError_t launch_cut(const RowParams& p, int chunks, cudaStream_t s) {
  if constexpr (MODE != kRowQuant)
    if (p.residual) return launch_rows<MODE, BF16, CUT, true>(p, chunks, s);
  return launch_rows<MODE, BF16, CUT, false>(p, chunks, s);
}

template <int MODE>
cudaError_t launch_mode(const RowParams& p, bool bf16, Cut cut, int chunks, cudaStream_t s) {
  switch (cut) {
    case kAligned:
      return bf16 ? launch_cut<MODE, true, kAligned>(p, chunks, s) : launch_cut<MODE, false, kAligned>(p, chunks, s);
    case kShifted:
      return bf16 ? launch_cut<MODE, true, kShifted>(p, chunks, s) : launch_cut<MODE, false, kShifted>(p, chunks, s);
    default:
      return bf16 ? launch_cut<MODE, true, kSingle>(p, chunks, s) : launch_cut<MODE, false, kSingle>(p, chunks, s);
  }
}

bool off(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// An output may be an input itself (same rows, same stride: each element is read before it
// is written, by one thread); any other overlap is refused.
bool clash(const Span& out, const void* out_p, const Span& in, const void* in_p, bool same_ok) {
  if (!in_p || !out_p || !overlap(out, in)) return false;
  return !(same_ok && out.lo == in.lo && out.step == in.step);
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
  if (!p.x || !p.out || (i8 && !p.scale)) return internal_fail(BBH_ERR_ARG, w + ": null pointer");
  if (p.sum && !p.residual) return internal_fail(BBH_ERR_ARG, w + ": sum needs a residual");
  if (!(p.eps >= 0.f) || p.eps > FLT_MAX) return internal_fail(BBH_ERR_ARG, w + ": eps must be finite and >= 0");
  if (p.ldx < p.D || (p.residual && p.ldr < p.D) || (p.sum && p.lds < p.D) || p.ldo < p.D)
    return internal_fail(BBH_ERR_ARG, w + ": a row stride is smaller than D");
  if (off(p.x, 2) || off(p.residual, 2) || off(p.weight, 2) || off(p.sum, 2) || (!i8 && off(p.out, 2)) || off(p.scale, 4))
    return internal_fail(BBH_ERR_ARG, w + ": a pointer is not aligned to its elements");
  const void* outs[3] = {p.out, p.sum, p.scale};
  const Span so[3] = {span(p.out, p.ldo, p.rows, p.D, i8 ? 1 : 2),
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
  // the cut that the operands allow (see Cut)
  bool aligned = p.D % 8 == 0, shifted = !off(p.weight, 16) && (!i8 || (!off(p.out, 8) && p.ldo % 8 == 0));
  auto look = [&](const uint16_t* q, int64_t ld) {
    if (!q) return;
    aligned = aligned && !off(q, 16) && ld % 8 == 0;
    shifted = shifted && ((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p.x)) & 15) == 0 &&
              (p.rows == 1 || (ld - p.ldx) % 8 == 0);
  };
  look(p.x, p.ldx);
  look(p.residual, p.ldr);
  look(p.sum, p.lds);
  if (!i8) look(static_cast<const uint16_t*>(p.out), p.ldo);
  aligned = aligned && shifted;
  const Cut cut = aligned ? kAligned : shifted ? kShifted : kSingle;
  int chunks = 0;
  p.group = row_group(p.rows, p.D, sms, mode != kRowQuant, &chunks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == BBH_BF16;
  const cudaError_t e = mode == kRowNorm     ? launch_mode<kRowNorm>(p, bf, cut, chunks, s)
                        : mode == kRowNormI8 ? launch_mode<kRowNormI8>(p, bf, cut, chunks, s)
                                             : launch_mode<kRowQuant>(p, bf, cut, chunks, s);
  if (e != cudaSuccess) return internal_fail(BBH_ERR_CUDA, w + ": " + cudaGetErrorString(e));
  return BBH_OK;
}

}  // namespace
}  // namespace bbh

extern "C" {

int bbh_rmsnorm(const uint16_t* x, int64_t ldx, const uint16_t* residual, int64_t ldr, const uint16_t* weight,
                uint16_t* y, int64_t ldy, uint16_t* sum, int64_t lds, int M, int D, float eps, int dtype,
                void* stream) {
  bbh::RowParams p{x, residual, weight, y, nullptr, sum, ldx, ldr, ldy, lds, M, D, 0, eps};
  return bbh::run_rows("bbh_rmsnorm", bbh::kRowNorm, p, dtype, stream);
}

int bbh_rmsnorm_i8(const uint16_t* x, int64_t ldx, const uint16_t* residual, int64_t ldr, const uint16_t* weight,
                   int8_t* q, int64_t ldq, float* scale, uint16_t* sum, int64_t lds, int M, int D, float eps,
                   int dtype, void* stream) {
  bbh::RowParams p{x, residual, weight, q, scale, sum, ldx, ldr, ldq, lds, M, D, 0, eps};
  return bbh::run_rows("bbh_rmsnorm_i8", bbh::kRowNormI8, p, dtype, stream);
}

int bbh_quantize_i8(const uint16_t* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int M, int D, int dtype,
                    void* stream) {
  bbh::RowParams p{x, nullptr, nullptr, q, scale, nullptr, ldx, 0, ldq, 0, M, D, 0, 0.f};
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
  const bool q8 = !off(q, 8) && ldq % 8 == 0;
  const Cut cut = q8 && D % 8 == 0 && !off(y, 16) && ldy % 8 == 0 ? kAligned : q8 ? kShifted : kSingle;
  int chunks = 0;
  DequantParams p{q, scale, y, ldq, ldy, M, D, row_group(M, D, sms, false, &chunks)};
  const int block = p.group < kRowBlock ? kRowBlock : p.group;
  const int per = block / p.group;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(M) + per - 1) / per));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_ex(kern, grid, dim3(block), 0, s, true, 1, p); };
  const bool bf = dtype == BBH_BF16;
  const cudaError_t e = cut == kAligned   ? (bf ? go(dequant_kernel<true, kAligned>) : go(dequant_kernel<false, kAligned>))
                        : cut == kShifted ? (bf ? go(dequant_kernel<true, kShifted>) : go(dequant_kernel<false, kShifted>))
                                          : (bf ? go(dequant_kernel<true, kSingle>) : go(dequant_kernel<false, kSingle>));
  if (e != cudaSuccess)
    return internal_fail(BBH_ERR_CUDA, std::string("bbh_dequantize_i8: ") + cudaGetErrorString(e));
  return BBH_OK;
}

}  // extern "C"
