// The 8-bit key/value cache: blocks of 64 tokens x 64 dimensions of one head, one code byte a value, one fp32 scale for each
// block and head (value = code * scale).  Shared by the kernels that write, read and attend over it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.h"

namespace rt {

struct KvView {  // rt_kv_cache by value
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int blocks;
  int heads;
};

// Checks of a cache argument that every entry point makes.
rt_status check_kv_cache(const char* what, const rt_kv_cache* cache, KvView* view);

namespace kv {

constexpr float kE4m3Max = 448.f, kInt8Max = 127.f;
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100: 1 / scale stays a normal number

__device__ __forceinline__ void index_error(int* err, int site) { atomicCAS(err, 0, site); }

// Which part of which sequence a CTA takes, where nobody knows the longest one: sequence s has the places
// (first[s] * group >> shift) + spare * s up to where those of s + 1 begin, at least (n * group >> shift) + spare for n tokens.  Each CTA looks for
// the sequence that has place `at`; none: seq = -1.  All threads call it; found and count are in shared memory.
struct Place {
  int seq, nth;
};
__device__ __forceinline__ Place find_place(int at, const int32_t* __restrict__ first, int n_seq, int group, int shift, int spare, int tokens,
                                            int most, Place* found, int* count, int* err, int site) {
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < n_seq; s += blockDim.x) {
    const int f0 = first[s], f1 = first[s + 1];
    if (f1 <= f0) continue;
    if (f0 < 0 || f1 > tokens || f1 - f0 > most) {
      index_error(err, site);
      continue;
    }
    const int64_t lo = (static_cast<int64_t>(f0) * group >> shift) + static_cast<int64_t>(spare) * s;
    const int64_t hi = (static_cast<int64_t>(f1) * group >> shift) + static_cast<int64_t>(spare) * (s + 1);
    if (lo <= at && at < hi) {
      if (atomicAdd(count, 1)) index_error(err, site);  // rows of two sequences
      *found = Place{s, static_cast<int>(at - lo)};
    }
  }
  __syncthreads();
  return *count == 1 ? *found : Place{-1, 0};
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// Codes as half2, exactly.
//   int8: the code with its sign bit flipped is an unsigned byte u = code + 128; the half with bits 0x6400 | u is 1024 + u.
//   e4m3: the hardware's conversion.  The writer never stores the code NaN; where it stands in a place that holds no token, the kernels
//     that would multiply it take a zero instead.
template <bool INT8>
struct Codes;

template <>
struct Codes<true> {
  static constexpr float kUnit = 1.f;
  static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w ^ 0x80808080u; }
  // bytes `LO` and `LO + 1` of prepared codes
  template <int LO>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t x = prmt(w, 0x64646464u, LO == 0 ? 0x4140u : 0x4342u);
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0xe480)));  // - 1152
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};

template <>
struct Codes<false> {
  static constexpr float kUnit = 1.f, kBias = 0.f;
  static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w; }
  template <int LO>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    uint32_t r;
    if constexpr (LO == 0) asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo;}" : "=r"(r) : "r"(w));
    else asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, hi;}" : "=r"(r) : "r"(w));
    return r;
  }
};

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

}  // namespace kv
}  // namespace rt
