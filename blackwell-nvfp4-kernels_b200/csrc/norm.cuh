// Residual addition, root-mean-square norm and quantised output, sm_100a:
//
//   h = rn(x + residual)                    (rounded to the residual's type; h = x without one)
//   r = rn(1 / sqrt(sum(h^2) / K + eps))    (the sum and the root in fp64, r in fp32)
//   y = rn(rn(h * r) * weight)              (fp32)
//
// and y as
//   kNormPlain  fp16, bf16 or fp32;
//   kNormFp8    e4m3 with one fp32 scale for each `group` columns (or the whole
//               row): s = amax / 448, q = e4m3_rne(y / s) (from h * weight: the rounding of
//               r does not move a code), all zero when s is 0;
//   kNormNvfp4  e2m1 + e4m3 scales per 16 in the layouts the GEMMs read, by the
//               rules of quantize.cuh.
//
// The sum is fp64 because it decides on which side of a rounding border a
// code falls: summed in fp32 the last bit of r depends on the order of the
// sum, and codes on a border move with it.  In fp64 two orders differ by
// about 2^-53, so that r, and with it every output bit, is the same for any
// number of threads (but for one row in about 2^28).
//
// A row is read once: each thread keeps its elements in registers from the
// load to the output.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>
#include "gemv.cuh"
#include "ptx.cuh"
#include "quantize.cuh"

namespace nvfp4 {

constexpr int kNormAnyType = -1;
constexpr int kNormPlain = 0, kNormFp8 = 1, kNormNvfp4 = 2;
constexpr int kNormFp8Row = 3;         // the kernel's fp8 with one scale for the row
constexpr int kNormMaxThreads = 1024;
constexpr int kNormMaxK = kNormMaxThreads * 8 * 4;
constexpr int kNormPadAtoms = 8;       // scale atoms whose padding rows one CTA clears

struct NormParams {
  const void *x, *residual, *weight;   // residual may be null
  void* h;                             // [rows][k], the residual's type; null without a residual
  int64_t ldx, ldr, ldh;
  double eps, inv_k;                   // inv_k = 1 / k
  int rows, k, x_dtype, r_dtype, w_dtype;
  void* y;                             // plain: [rows][k]; fp8: e4m3 bytes; nvfp4: packed [rows][k/2]
  int64_t ldy;                         // plain only
  int y_dtype;                         // plain only
  float* scales;                       // fp8: [rows][k / group]
  int group_bits;                      // fp8: 5, 6 or 7 for groups of 32, 64 or 128 columns
  uint8_t *sf_perm, *sf_plain;         // nvfp4
};

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The larger magnitude, with some sign; NaN if either is.
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float largest_of(const float (&v)[8]) {
  const float a = max_abs_nan(max_abs_nan(v[0], v[1]), max_abs_nan(v[2], v[3]));
  const float b = max_abs_nan(max_abs_nan(v[4], v[5]), max_abs_nan(v[6], v[7]));
  return fabsf(max_abs_nan(a, b));
}

template <bool kVec>
__device__ __forceinline__ Raw8 norm_load8(const void* base, int dtype, int64_t at, int left) {
  Raw8 r;
  r.a = r.b = make_uint4(0, 0, 0, 0);
  if (left <= 0) return r;
  if (dtype == kDtF32) {
    const uint32_t* q = static_cast<const uint32_t*>(base) + at;
    if constexpr (kVec) {
      r.a = *reinterpret_cast<const uint4*>(q), r.b = *reinterpret_cast<const uint4*>(q + 4);
    } else {
      uint32_t v[8];
      #pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? q[i] : 0u;
      r.a = make_uint4(v[0], v[1], v[2], v[3]), r.b = make_uint4(v[4], v[5], v[6], v[7]);
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(base) + at;
    if constexpr (kVec) {
      r.a = *reinterpret_cast<const uint4*>(q);
    } else {
      uint32_t v[4];
      #pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = (2 * i < left ? (uint32_t)q[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)q[2 * i + 1] << 16 : 0u);
      r.a = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
  return r;
}

// fp32 -> the type's bits; `f` becomes the rounded values.
__device__ __forceinline__ Raw8 norm_round(float (&f)[8], int dtype) {
  Raw8 r;
  uint32_t w[8];
  #pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
  if (dtype == kDtF32) {
    r.a = make_uint4(w[0], w[1], w[2], w[3]), r.b = make_uint4(w[4], w[5], w[6], w[7]);
    return r;
  }
  uint32_t h[4];
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == kDtBF16) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      h[i] = *reinterpret_cast<const uint32_t*>(&t);
    } else {
      const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      h[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  r.a = make_uint4(h[0], h[1], h[2], h[3]), r.b = make_uint4(0, 0, 0, 0);
  widen8(r, dtype, f);
  return r;
}

// Sums of fp16 or bf16 elements, rounded once: what the fp32 sum rounds to as
// well, since fp32 has two digits more than twice theirs (Figueroa's condition).
template <int kType>
__device__ __forceinline__ Raw8 norm_add16(const Raw8& a, const Raw8& b) {
  using T2 = std::conditional_t<kType == kDtBF16, __nv_bfloat162, __half2>;
  uint32_t x[4] = {a.a.x, a.a.y, a.a.z, a.a.w};
  const uint32_t y[4] = {b.a.x, b.a.y, b.a.z, b.a.w};
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T2 t = __hadd2_rn(*reinterpret_cast<const T2*>(&x[i]), *reinterpret_cast<const T2*>(&y[i]));
    x[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  Raw8 r;
  r.a = make_uint4(x[0], x[1], x[2], x[3]), r.b = make_uint4(0, 0, 0, 0);
  return r;
}

template <bool kVec>
__device__ __forceinline__ void norm_store8(void* base, int dtype, int64_t at, int left, const Raw8& r) {
  if (left <= 0) return;
  if (dtype == kDtF32) {
    uint32_t* q = static_cast<uint32_t*>(base) + at;
    if constexpr (kVec) {
      *reinterpret_cast<uint4*>(q) = r.a, *reinterpret_cast<uint4*>(q + 4) = r.b;
    } else {
      const uint32_t v[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
      #pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) q[i] = v[i];
    }
  } else {
    uint16_t* q = static_cast<uint16_t*>(base) + at;
    if constexpr (kVec) {
      *reinterpret_cast<uint4*>(q) = r.a;
    } else {
      const uint32_t v[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
      #pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) q[i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
    }
  }
}

// Two fp32 operations in one instruction (each rounded as by itself).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t fma2_down(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rm.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// v / s (IEEE): by the two fused multiply-adds of quantize.cuh's div_by_scale
// where Markstein's theorem holds (r = RN(1 / s), s's mantissa not all ones, nothing
// near under- or overflow: `fast`), else by the division itself.
__device__ __forceinline__ void norm_divide(float (&v)[8], float s, bool fast) {
  if (fast) {
    const float rs = __frcp_rn(s);
    const uint64_t s2 = pack2(-s, -s), r2 = pack2(rs, rs);
    #pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint64_t x = pack2(v[e], v[e + 1]), q = mul2(x, r2);
      unpack2(fma2(fma2_down(q, s2, x), r2, q), v[e], v[e + 1]);
    }
  } else {
    // hardly ever taken: one division in a loop that turns the values round (indexed by the
    // loop they would lie in local memory, also for the branch above)
    #pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const float q = __fdiv_rn(v[0], s);
      #pragma unroll
      for (int e = 0; e < 7; ++e) v[e] = v[e + 1];
      v[7] = q;
    }
  }
}

// One CTA for each row (chunks of 8 elements, chunk c = thread + i * threads,
// i < NV); kNormNvfp4: CTAs past the rows clear the padding rows of the last
// block's scale atoms.  kVec: every 8 elements of every tensor are 16-byte aligned
// and K % 8 == 0.
//
// Bound: 7 bytes an element at 16 bits (fp8), 63 us of 8192 x 7168 at the rate of a copy; the
// kernel takes 66.2 (6.2 TB/s), its instructions (28 an element) 67 % of the issue slots.  16-bit
// additions and fp32 products go two at a time (83 us before); the group's columns are a power of
// two and no register is indexed (75 us with integer divisions, 80 with values in local memory).
// h stays in registers in its own type, half the registers of fp32 for the 16-bit
// types: several CTAs fit on an SM, whose loads and arithmetic overlap.
// Four CTAs of 512 threads on an SM with the types known (32 registers): 8192 x
// 7168 bf16 to fp8 66.2 us; with three, and the codes by division, 74.0, four 67.7.
template <int NV, int kThreads, int kOut, bool kVec, int kType>
__global__ void __launch_bounds__(kThreads, kThreads == 512 && kType != kNormAnyType ? 4 : 1) norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ double s_sum[32];
  __shared__ float s_max[32], s_r;
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
  griddep_wait();
  griddep_launch_dependents();
  if constexpr (kOut == kNormNvfp4) {
    if ((int)blockIdx.x >= p.rows) {
      const int rest = p.rows % 128, atoms = p.k / 64;
      const int a0 = ((int)blockIdx.x - p.rows) * kNormPadAtoms, a1 = min(a0 + kNormPadAtoms, atoms);
      uint32_t* base = reinterpret_cast<uint32_t*>(p.sf_perm + (size_t)(p.rows / 128) * atoms * 512);
      for (int i = a0 * 128 + tid; i < a1 * 128; i += (int)blockDim.x) {
        const int w = i % 128;                            // word of the atom: row w/4 of quarter w%4
        if ((w % 4) * 32 + w / 4 >= rest) base[i] = 0u;
      }
      return;
    }
  }
  const int row = (int)blockIdx.x;
  auto col_of = [&](int i) { return (tid + i * (int)blockDim.x) * 8; };
  const bool add = p.residual != nullptr;
  const int x_dtype = kType == kNormAnyType ? p.x_dtype : kType, r_dtype = kType == kNormAnyType ? p.r_dtype : kType;
  const int w_dtype = kType == kNormAnyType ? p.w_dtype : kType, h_dtype = add ? r_dtype : x_dtype;
  Raw8 h[NV], wt;
  double sum = 0.0;
  {
    Raw8 rr[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      h[i] = norm_load8<kVec>(p.x, x_dtype, (int64_t)row * p.ldx + col_of(i), p.k - col_of(i));
    if (add) {
      #pragma unroll
      for (int i = 0; i < NV; ++i)
        rr[i] = norm_load8<kVec>(p.residual, r_dtype, (int64_t)row * p.ldr + col_of(i), p.k - col_of(i));
    }
    if constexpr (NV == 1) wt = norm_load8<kVec>(p.weight, w_dtype, col_of(0), p.k - col_of(0));
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8];
      if (kType != kNormAnyType && add) h[i] = norm_add16<kType>(h[i], rr[i]);
      widen8(h[i], x_dtype, f);
      if (kType != kNormAnyType && add) {
        norm_store8<kVec>(p.h, r_dtype, (int64_t)row * p.ldh + col_of(i), p.k - col_of(i), h[i]);
      } else if (add) {
        float g[8];
        widen8(rr[i], r_dtype, g);
        #pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __fadd_rn(f[e], g[e]);
        h[i] = norm_round(f, r_dtype);
        norm_store8<kVec>(p.h, r_dtype, (int64_t)row * p.ldh + col_of(i), p.k - col_of(i), h[i]);
      }
      #pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double d = (double)f[e];
        sum = fma(d, d, sum);
      }
    }
  }
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float r;
  if (warps > 1) {
    // one warp adds up and takes the root: its 50 instructions in every warp would cost
    // more than the second barrier
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = lane < warps ? s_sum[lane] : 0.0;
      #pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s_r = (float)rsqrt(fma(sum, p.inv_k, p.eps));
    }
    __syncthreads();
    r = s_r;
  } else {
    r = (float)rsqrt(fma(sum, p.inv_k, p.eps));
  }
  auto values = [&](int i, float (&v)[8], float r) {      // h r weight of chunk i
    float w[8];
    if constexpr (NV > 1) wt = norm_load8<kVec>(p.weight, w_dtype, col_of(i), p.k - col_of(i));
    widen8(wt, w_dtype, w);
    widen8(h[i], h_dtype, v);
    #pragma unroll
    for (int e = 0; e < 8; e += 2)
      unpack2(mul2(mul2(pack2(v[e], v[e + 1]), pack2(r, r)), pack2(w[e], w[e + 1])), v[e], v[e + 1]);
  };

  if constexpr (kOut == kNormPlain) {
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
      values(i, v, r);
      norm_store8<kVec>(p.y, p.y_dtype, (int64_t)row * p.ldy + col_of(i), p.k - col_of(i), norm_round(v, p.y_dtype));
    }
  } else if constexpr (kOut == kNormFp8 || kOut == kNormFp8Row) {
    // With r = r2 rho, r2 a power of two, v = h r2 weight is exact for 16-bit types and as far from
    // over- and underflow as y = v rho.  y / s = v (448 / largest v): two roundings, where y, its
    // largest, s and the quotient would have six, each of which can move a code that is near a border.
    // Chunks past the row's end hold 0 * r * 0: NaN when r is, as the whole row is then.
    const uint32_t r_bits = __float_as_uint(r);
    const bool r_normal = r >= 1.1754944e-38f && r <= 3.402823466e38f;
    const float r2 = r_normal ? __uint_as_float(r_bits & 0x7f800000u) : r;
    const float rho = r_normal ? __uint_as_float((r_bits & 0x7fffffu) | 0x3f800000u) : 1.f;
    float row_top = 0.f;
    if constexpr (kOut == kNormFp8Row) {
      #pragma unroll
      for (int i = 0; i < NV; ++i) {
        float v[8];
        values(i, v, r2);
        row_top = max_nan(row_top, largest_of(v));
      }
      #pragma unroll
      for (int o = 16; o > 0; o >>= 1) row_top = max_nan(row_top, __shfl_xor_sync(0xffffffffu, row_top, o));
      if (warps > 1) {
        if (lane == 0) s_max[warp] = row_top;
        __syncthreads();
        row_top = lane < warps ? s_max[lane] : 0.f;
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) row_top = max_nan(row_top, __shfl_xor_sync(0xffffffffu, row_top, o));
      }
    }
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
      values(i, v, r2);
      float top = row_top;
      if constexpr (kOut == kNormFp8) {
        top = largest_of(v);
        #pragma unroll
        for (int o = 1; o < 16; o <<= 1)                  // 4, 8 or 16 neighbouring lanes
          if (8 * o < 1 << p.group_bits) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      const int col = col_of(i), left = p.k - col;
      // Markstein's theorem (see div_by_scale) for / 448 = 1.75 * 2^8, a mantissa of the exhaustive
      // proof in quantize.cuh, and for 448 / top unless top's mantissa is all ones; numbers between 2^-90 and
      // 2^126 where it matters
      const float y_top = __fmul_rn(top, rho);
      const bool fast = top >= 3.308722e-24f /* 2^-78 */ && top <= 4.253530e37f /* 2^125 */ &&
                        (__float_as_uint(top) & 0x7fffffu) != 0x7fffffu;
      const float s = fast ? div_by_scale(y_top, 448.f, 1.f / 448.f) : __fdiv_rn(y_top, 448.f);
      uint32_t code[2] = {0u, 0u};
      if (s != 0.f) {
        if (fast) {
          const float c = div_by_scale(448.f, top, __frcp_rn(top));
          #pragma unroll
          for (int e = 0; e < 8; e += 2) unpack2(mul2(pack2(v[e], v[e + 1]), pack2(c, c)), v[e], v[e + 1]);
        } else {
          #pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __fmul_rn(v[e], rho);
          norm_divide(v, s, false);
        }
        #pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[e], v[e + 1]), __NV_SATFINITE, __NV_E4M3);
          code[e / 4] |= two << (8 * (e % 4));
        }
      }
      if (left > 0) {
        uint8_t* q = static_cast<uint8_t*>(p.y) + (int64_t)row * p.k + col;
        if constexpr (kVec) {
          *reinterpret_cast<uint2*>(q) = make_uint2(code[0], code[1]);
        } else {
          #pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) q[e] = (uint8_t)(code[e / 4] >> (8 * (e % 4)));
        }
        if constexpr (kOut == kNormFp8Row) {
          if (tid == 0 && i == 0) p.scales[row] = s;
        } else if ((col & ((1 << p.group_bits) - 1)) == 0) {
          p.scales[(int64_t)row * (p.k >> p.group_bits) + (col >> p.group_bits)] = s;
        }
      }
    }
  } else {
    const int sub = lane & 7;                             // chunk of the 64-column atom
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
      values(i, v, r);
      const int col = col_of(i);
      float amax = largest_of(v);
      amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      const bool finite = amax <= 3.402823466e38f;
      const float a6 = finite ? div_by_scale(amax, 6.0f, 1.0f / 6.0f) : amax;
      const __nv_fp8_storage_t s8 = __nv_cvt_float_to_fp8(a6, __NV_SATFINITE, __NV_E4M3);
      const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw(s8, __NV_E4M3)));
      uint32_t word = 0;
      if (s != 0.f) {
        norm_divide(v, s, finite);
        #pragma unroll
        for (int e = 0; e < 8; e += 2) word |= e2m1x2(v[e], v[e + 1]) << (4 * e);
      }
      const uint32_t pair = (uint32_t)s8 | (__shfl_down_sync(0xffffffffu, (uint32_t)s8, 2) << 8);
      const uint32_t sf_word = pair | (__shfl_down_sync(0xffffffffu, pair, 4) << 16);   // sub 0
      if (col < p.k) {
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.y) + (int64_t)row * (p.k / 2) + col / 2) = word;
        if (sub == 0) {
          const int atom = col / 64;
          *reinterpret_cast<uint32_t*>(p.sf_perm + ((size_t)(row / 128) * (p.k / 64) + atom) * 512 + (row % 32) * 16 +
                                       (row % 128 / 32) * 4) = sf_word;
          if (p.sf_plain != nullptr)
            *reinterpret_cast<uint32_t*>(p.sf_plain + (int64_t)row * (p.k / 16) + atom * 4) = sf_word;
        }
      }
    }
  }
}

}  // namespace nvfp4
