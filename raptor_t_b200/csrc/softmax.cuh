// The softmax of a row of scores held in registers: maxima, base-2 exponentials and sums of 64 columns at a time, in the packed
// fp32 arithmetic of sm_100.  Shared by the attention kernels whose score tiles are in TMEM.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rt {
namespace softmax {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed fp32x2 arithmetic and three-input max (sm_100): half the issue slots of the
// scalar forms in the softmax inner loops.
__device__ __forceinline__ unsigned long long f2_pack(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_unpack(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long f2_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long f2_add(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// Row maximum of 64 scores held in registers.
__device__ __forceinline__ float max64(const uint32_t* s) {
  float mx0 = __uint_as_float(s[0]), mx1 = __uint_as_float(s[1]);
  float mx2 = __uint_as_float(s[2]), mx3 = __uint_as_float(s[3]);
#pragma unroll
  for (int i = 4; i < 60; i += 8) {
    mx0 = max3(mx0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    mx1 = max3(mx1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
    mx2 = max3(mx2, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
    mx3 = max3(mx3, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
  }
  mx0 = max3(mx0, __uint_as_float(s[60]), __uint_as_float(s[61]));
  mx1 = max3(mx1, __uint_as_float(s[62]), __uint_as_float(s[63]));
  return fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
}

// 2^x for a pair of arguments on the FMA pipe (the exponential unit is the kernel's bottleneck, a part of
// the columns goes here instead): clamp, split x = n + f with |f| <= 0.5 by adding 1.5 * 2^23 (the integer
// lands in the low mantissa bits), 2^f by a cubic (relative error 7.5e-5, below the 16-bit rounding of the
// probabilities), n added to the exponent field.  NAN_STAYS: NaN gives NaN (otherwise a small number); 2^n is then a factor.
template <bool NAN_STAYS>
__device__ __forceinline__ void ex2_fma_pair(float x0, float x1, float& r0, float& r1) {
  if constexpr (NAN_STAYS) {
    x0 = max_nan(x0, -126.f);
    x1 = max_nan(x1, -126.f);
  } else {
    x0 = fmaxf(x0, -126.f);
    x1 = fmaxf(x1, -126.f);
  }
  const unsigned long long x = f2_pack(x0, x1);
  const unsigned long long xr = f2_add(x, f2_pack(12582912.f, 12582912.f));
  const unsigned long long n = f2_add(xr, f2_pack(-12582912.f, -12582912.f));
  const unsigned long long f = f2_fma(n, f2_pack(-1.f, -1.f), x);
  unsigned long long r = f2_fma(f, f2_pack(0.05517167f, 0.05517167f), f2_pack(0.24261112f, 0.24261112f));
  r = f2_fma(r, f, f2_pack(0.69326099f, 0.69326099f));
  r = f2_fma(r, f, f2_pack(0.99992807f, 0.99992807f));
  float a0, a1, b0, b1;
  f2_unpack(xr, b0, b1);
  if constexpr (NAN_STAYS) {
    f2_unpack(f2_mul(r, f2_pack(__int_as_float((__float_as_int(b0) << 23) + 0x3f800000), __int_as_float((__float_as_int(b1) << 23) + 0x3f800000))),
              r0, r1);
    return;
  }
  f2_unpack(r, a0, a1);
  r0 = __int_as_float(__float_as_int(a0) + (__float_as_int(b0) << 23));
  r1 = __int_as_float(__float_as_int(a1) + (__float_as_int(b1) << 23));
}

// p[i] = 2^(s[2i] * c - m), 2^(s[2i+1] * c - m) packed to 16 bits, for N scores; returns their sum.
// Every EVERY-th pair is computed on the FMA pipe.
constexpr int kPolyEvery = 4;  // measured: 3 and 4 are equal within noise, 2 is slower (issue slots)
template <bool BF16, int N, int EVERY = kPolyEvery, bool NAN_STAYS = false>
__device__ __forceinline__ float exp_columns(const uint32_t* s, uint32_t* p, float scale_log2, float m_ref) {
  static_assert(EVERY > 0, "every how many pairs");
  const unsigned long long c2 = f2_pack(scale_log2, scale_log2);
  const unsigned long long nm2 = f2_pack(-m_ref, -m_ref);
  unsigned long long acc0 = 0ull, acc1 = 0ull;  // two packed partial sums (+0.0f, +0.0f)
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const unsigned long long t = f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, nm2);
    float t0, t1;
    f2_unpack(t, t0, t1);
    float p0, p1;
    if (i % EVERY == EVERY - 1) {
      ex2_fma_pair<NAN_STAYS>(t0, t1, p0, p1);
    } else {
      p0 = ex2(t0);
      p1 = ex2(t1);
    }
    if (i & 1) acc1 = f2_add(acc1, f2_pack(p0, p1));
    else acc0 = f2_add(acc0, f2_pack(p0, p1));
    p[i] = pack2<BF16>(p0, p1);
  }
  float s0, s1;
  f2_unpack(f2_add(acc0, acc1), s0, s1);
  return s0 + s1;
}
template <bool BF16>
__device__ __forceinline__ float exp64(const uint32_t* s, uint32_t* p, float scale_log2, float m_ref) {
  return exp_columns<BF16, 64>(s, p, scale_log2, m_ref);
}

// setmaxnreg: executed by all four warps of a warpgroup at one place.
template <int N>
__device__ __forceinline__ void reg_dealloc() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_alloc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

}  // namespace softmax
}  // namespace rt
