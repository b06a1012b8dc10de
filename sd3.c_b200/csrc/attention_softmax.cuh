// Pieces of an online softmax on rows of scores in registers, shared by the tcgen05 attention kernels: one thread owns a
// query row and sees it 64 keys at a time.
#pragma once
#include <math.h>

#include "kernels.h"
#include "ptx.cuh"

namespace sd3 {
namespace softmax_detail {

constexpr int POLY_EVERY = 4;  // of every 4 pairs of exponentials, one element goes to the FMA pipe

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// exp2 on the FMA pipe: x = n + f with n = round(x), f in [-0.5, 0.5]; 2^f by a
// degree-3 polynomial (relative error at most 8.5e-4, 2.2e-4 root mean square, below bf16 resolution: the minimax cubic,
// 7.5e-5, changes the error of the output by less than 0.3 %), exponent added as an integer.  Inputs below -125 give a
// denormal-sized result.
__device__ __forceinline__ float ex2_poly(float x) {
  x = fmaxf(x, -125.0f);
  const float t = x + 12582912.0f;  // 1.5 * 2^23: the low mantissa bits now hold round(x)
  const float f = x - (t - 12582912.0f);
  float p = fmaf(f, 0.0558011f, 0.2402265f);
  p = fmaf(p, f, 0.6931472f);
  p = fmaf(p, f, 1.0f);
  return __int_as_float(__float_as_int(p) + (__float_as_int(t) << 23));
}

// lane 0 arrives; a predicated instruction instead of a divergent branch
__device__ __forceinline__ void mbar_arrive_lane0(uint64_t* bar, int lane) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.eq.s32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
      "}\n" ::"r"(smem_u32(bar)), "r"(lane)
      : "memory");
}
// `pre` is the result of an earlier mbar_test_wait of the same phase by every lane
// (one broadcast read, warp-uniform result); blocks only if that test failed.
__device__ __forceinline__ bool mbar_wait_pre(uint32_t pre, uint64_t* bar, uint32_t parity, const WaitCtx& w,
                                              int code) {
  if (pre != 0) return true;
  return mbar_wait_warp(bar, parity, w, code);
}

// keys >= T of a ragged last tile do not exist: their scores become -inf
__device__ __forceinline__ void mask_cols(uint32_t (&r)[32], int key0, int T) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (key0 + i >= T) r[i] = 0xff800000u;
}

// maximum of 64 scores: eight independent chains of 3-input maxima, then a tree
__device__ __forceinline__ float max_of2(const uint32_t (&a)[32], const uint32_t (&b)[32]) {
  float m[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    m[q] = fmaxf(__uint_as_float(a[8 * q]), __uint_as_float(a[8 * q + 1]));
    m[4 + q] = fmaxf(__uint_as_float(b[8 * q]), __uint_as_float(b[8 * q + 1]));
#pragma unroll
    for (int i = 2; i < 8; i += 2) {
      m[q] = max3(m[q], __uint_as_float(a[8 * q + i]), __uint_as_float(a[8 * q + i + 1]));
      m[4 + q] = max3(m[4 + q], __uint_as_float(b[8 * q + i]), __uint_as_float(b[8 * q + i + 1]));
    }
  }
  return fmaxf(max3(m[0], m[1], m[2]), max3(max3(m[3], m[4], m[5]), m[6], m[7]));
}

// p *= alpha on 32 packed bf16 pairs (rare path: the maximum moved after these were formed)
__device__ __forceinline__ void scale_packed(uint32_t (&r)[32], float alpha) {
  const __nv_bfloat162 a2 = __float2bfloat162_rn(alpha);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    __nv_bfloat162 v = *reinterpret_cast<__nv_bfloat162*>(&r[i]);
    v = __hmul2(v, a2);
    r[i] = *reinterpret_cast<uint32_t*>(&v);
  }
}

// r[i] = bf16x2(exp2(r[2i] c + nmc), exp2(r[2i+1] c + nmc)) for i < 16, in place (word i
// is written after scores 2i and 2i+1 were read); the exponentials are added into acc.
template <bool POLY = true>  // without: every exponential on the MUFU unit, a score of -inf (a masked key) gives exactly 0
__device__ __forceinline__ void exp_pack(uint32_t (&r)[32], float c, float nmc, float2& acc) {
  const float2 c2 = make_float2(c, c), n2 = make_float2(nmc, nmc);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), c2, n2);
    float2 p;
    p.x = ex2_approx(x.x);
    p.y = (POLY && i % POLY_EVERY == 0) ? ex2_poly(x.y) : ex2_approx(x.y);
    acc = __fadd2_rn(acc, p);
    r[i] = pack_bf16x2(p.x, p.y);
  }
}

}  // namespace softmax_detail
}  // namespace sd3
