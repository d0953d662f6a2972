// Scores of tokens from rows of logits z over a vocabulary, and their gradient.  With m = max z and S = sum e^(z - m):
//   logp = (z_t - m) - log S,   entropy H = log S - sum e^(z - m) (z - m) / S,   the k best tokens by (value, then lower index);
//   dz_v = -p_v (g_logp + sum_j g_top_j + g_H (log p_v + H)) + [v = t] g_logp + sum_j [v = id_j] g_top_j.
// Both read every logit once and are bound by that (the gradient writes as much).
//
// Forward: a CTA, or a cluster of CTAs where there are few rows, takes a row.  A thread keeps the running maximum, sum and weighted sum of its
// share.  The k best come without a second pass over the row: the k-th largest of the maxima of groups of four threads is a
// value that at least k logits reach; only threads whose own maximum reaches it look at their share again (a few dozen
// logits, still in L2) and list what does.  A list that does not fit (thousands of equal logits) is replaced by k
// searches over the row.
//
// Measured (50,358 logits a row, device time in a captured graph; 0.3 to 0.5 us more a call in a loop, and up to 4 % between GPUs): forward of 2,048 rows of fp16 with 8 alternatives 47.7 us, 4.3 TB/s (41 without alternatives: the list costs four
// barriers and a round trip to L2 a row); 4,096 rows 83, 5.0 TB/s; 19 rows 7.0, a launch and the chain of one row.  Gradient of 4,096 rows of bf16
// with 4 alternatives 135 to 137 us, 6.0 TB/s; with one value at a time instead of packed pairs 144.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "device_error.h"
#include "launch.h"
#include "launch_count.h"
#include "sm100_ptx.cuh"

namespace rt {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 4;  // threads of a group
constexpr int kGroups = kThreads / kGroup;
constexpr int kMaxTop = 32;
constexpr int kMaxRanks = 4;  // CTAs of a row
constexpr int kSms = 148;
constexpr int kListed = 1024;  // candidates that a CTA can list
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 5.5f;  // the reference follows a share's maximum when e^z has grown by more than 2^8

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ unsigned long long f2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_split(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long f2_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long f2_add(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int TYPE>
struct Logits;  // vectors of 16 bytes

template <>
struct Logits<RT_F32> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float one(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ T from(float f) { return f; }
  // the largest number of some vectors (NaN left out), and -inf replaced by a number far below every reference
  static constexpr float kFloor = -1e30f;
  template <int N>
  static __device__ __forceinline__ float largest(const uint4* v) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[4];
      unpack(v[i], x);
      m = fmaxf(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    }
    return m;
  }
  static __device__ __forceinline__ uint4 floored(const uint4& v) {
    float x[4];
    unpack(v, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = max_nan(x[j], kFloor);
    return pack(x);
  }
};

template <>
struct Logits<RT_F16> {
  using T = __half;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(const T* p) { return __half2float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint4 v;
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return v;
  }
  static __device__ __forceinline__ T from(float f) { return __float2half_rn(f); }
  static constexpr float kFloor = -65504.f;
  template <int N>
  static __device__ __forceinline__ float largest(const uint4* v) {
    const __half2* h = reinterpret_cast<const __half2*>(v);
    __half2 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = __hmax2(m, h[i]);
    const float a = __low2float(m), b = __high2float(m);
    return fmaxf(fmaxf(a, b), -INFINITY);
  }
  static __device__ __forceinline__ uint4 floored(const uint4& v) {
    uint4 r;
    const __half2 low = __float2half2_rn(kFloor);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<__half2*>(&r)[i] = __hmax2_nan(reinterpret_cast<const __half2*>(&v)[i], low);
    return r;
  }
};

template <>
struct Logits<RT_BF16> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(const T* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return v;
  }
  static __device__ __forceinline__ T from(float f) { return __float2bfloat16_rn(f); }
  static constexpr float kFloor = -1e30f;
  template <int N>
  static __device__ __forceinline__ float largest(const uint4* v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(v);
    __nv_bfloat162 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * N; ++i) m = __hmax2(m, h[i]);
    const float a = __low2float(m), b = __high2float(m);
    return fmaxf(fmaxf(a, b), -INFINITY);
  }
  static __device__ __forceinline__ uint4 floored(const uint4& v) {
    uint4 r;
    const __nv_bfloat162 low = __float2bfloat162_rn(kFloor);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<__nv_bfloat162*>(&r)[i] = __hmax2_nan(reinterpret_cast<const __nv_bfloat162*>(&v)[i], low);
    return r;
  }
};

// Running statistics of a share of a row relative to a reference r near the share's maximum: with t = (z - r) log2 e,
// s = sum 2^t and w = sum 2^t t.
struct Stats {
  float r = -INFINITY, s = 0.f, w = 0.f;
  // relative to another reference (at least r)
  __device__ __forceinline__ void raise(float to) {
    if (r == -INFINITY) {
      w = 0.f;  // s is 0, or NaN and stays
    } else {
      const float d = (r - to) * kLog2e, f = ex2(d);
      w = f > 0.f ? (w + s * d) * f : s * f;  // the product of 0 and an infinite d is left out; a NaN of s stays
      s *= f;
    }
    r = to;
  }
  __device__ __forceinline__ void add(float z) {
    const float t = max_nan((z - r) * kLog2e, -2000.f);  // -inf: 2^t is 0 and so is its product with t
    const float e = ex2(t);
    s += e;
    w = fmaf(e, t, w);
  }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The statistics of a warp's shares, in every lane: one change of reference each, then plain sums.
__device__ __forceinline__ void join_warp(Stats& x) {
  const float to = warp_max(x.r);
  if (to != x.r) x.raise(to);
  x.s = warp_sum(x.s);
  x.w = warp_sum(x.w);
}

// A share of `nv` vectors and the elements before and behind them.  Vectors [lo, hi) belong to this CTA.
template <int TYPE>
struct Share {
  using L = Logits<TYPE>;
  const typename L::T* row;
  int head, nv, vocab;  // elements before the first aligned vector; vectors
  int lo, hi;
  bool edge;  // this CTA takes the elements outside the vectors
  __device__ __forceinline__ Share(const typename L::T* p, int v, int rank, int ranks) : row(p), vocab(v) {
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u) / static_cast<int>(sizeof(typename L::T));
    head = min(v, (L::kVec - mis) % L::kVec);
    nv = (v - head) / L::kVec;
    const int each = (nv + ranks - 1) / ranks;
    lo = min(nv, rank * each);
    hi = min(nv, lo + each);
    edge = rank == 0;
  }
  __device__ __forceinline__ const uint4* vectors() const { return reinterpret_cast<const uint4*>(row + head); }
  // the index of the `i`-th element outside the vectors, -1 behind the last one
  __device__ __forceinline__ int outside(int i) const {
    if (!edge) return -1;
    if (i < head) return i;
    const int j = head + nv * L::kVec + (i - head);
    return j < vocab ? j : -1;
  }
  // every element of the calling thread's share
  template <typename F>
  __device__ __forceinline__ void each_of_mine(F f) const {
    for (int i = lo + static_cast<int>(threadIdx.x); i < hi; i += kThreads) {
      float x[L::kVec];
      L::unpack(__ldg(vectors() + i), x);
#pragma unroll
      for (int j = 0; j < L::kVec; ++j) f(x[j], head + i * L::kVec + j);
    }
    if (threadIdx.x < 2 * L::kVec) {
      const int i = outside(threadIdx.x);
      if (i >= 0) f(L::one(row + i), i);
    }
  }
};

// Order of candidates as unsigned numbers: by value (NaN not among them), then lower index first.
__device__ __forceinline__ unsigned long long key_of(float z, int index) {
  uint32_t u = __float_as_uint(z == 0.f ? 0.f : z);  // -0 equals 0
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(u) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  uint32_t u = static_cast<uint32_t>(key >> 32);
  u = u & 0x80000000u ? u & 0x7fffffffu : ~u;
  return __uint_as_float(u);
}
__device__ __forceinline__ int index_of(unsigned long long key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

__device__ __forceinline__ unsigned long long max_u64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// How many of n keys are better; eight loads at a time.
__device__ __forceinline__ int better(const unsigned long long* keys, int n, unsigned long long key) {
  int before = 0, i = 0;
  for (; i + 8 <= n; i += 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) before += keys[i + k] > key;
  }
  for (; i < n; ++i) before += keys[i] > key;
  return before;
}

struct ScoreArgs {
  const void* logits;
  int64_t pitch;
  const int32_t* targets;
  int rows, vocab, top, ranks;
  float* logp;
  float* entropy;
  float2* stats;
  int32_t* top_ids;
  float* top_logp;
  int* err;
};

// CTAS: how many an SM holds at once; the registers of a thread follow from it.
template <int TYPE, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) token_logprobs_kernel(const ScoreArgs a) {
  using L = Logits<TYPE>;
  constexpr int kRowWarps = kMaxRanks * kThreads / 32;
  // of the row's first CTA: what every warp of the row has found, written by them, and what comes of it
  __shared__ Stats s_warp[kRowWarps];
  __shared__ float s_warp_max[kRowWarps];
  __shared__ unsigned long long s_all[kMaxRanks * kMaxTop];  // the best of each CTA, in order; 0: none
  __shared__ unsigned long long s_best[kMaxTop];
  __shared__ Stats s_row;
  __shared__ float s_max;
  // of each CTA
  __shared__ __align__(16) float s_group[kGroups];
  __shared__ int s_flagged[kThreads], s_flags;  // threads whose share holds candidates
  __shared__ float s_bar;                       // what a candidate reaches
  __shared__ int s_count;
  __shared__ unsigned long long s_list[kListed];
  RT_PDL_WAIT();
  RT_PDL_LAUNCH_DEPENDENTS();
  const int rank = blockIdx.x % a.ranks, row = blockIdx.x / a.ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Share<TYPE> share(static_cast<const typename L::T*>(a.logits) + row * a.pitch, a.vocab, rank, a.ranks);
  static_assert(kMaxRanks * kMaxTop <= kThreads && kRowWarps <= 32, "one warp joins what the row's warps have found");
  if (tid < kMaxRanks * kMaxTop) s_all[tid] = 0;
  if (tid == 0) s_count = s_flags = 0;
  if (a.ranks > 1) ptx::cluster_arrive();  // waited for before another CTA's shared memory is written
  int target = -1;
  float z_target = 0.f;
  if (tid == 0 && rank == 0 && a.logp) {  // on its way with the row
    target = a.targets[row];
    if (target >= 0 && target < a.vocab) z_target = L::one(share.row + target);
  }

  Stats mine;
  float my_most = -INFINITY;
  // N vectors: one look at their maximum, then five instructions a value in packed fp32
  auto take = [&](auto count, const uint4* v) {
    constexpr int N = decltype(count)::value;
    const float most = L::template largest<N>(v);
    my_most = fmaxf(my_most, most);
    if (most == -INFINITY) {  // nothing but -inf or NaN
#pragma unroll
      for (int u = 0; u < N; ++u) {
        float x[L::kVec];
        L::unpack(v[u], x);
#pragma unroll
        for (int j = 0; j < L::kVec; ++j) mine.s += x[j] == x[j] ? 0.f : x[j];
      }
      return;
    }
    if (!(most <= mine.r + kSlack)) mine.raise(most);
    if (!(mine.r > 0.5f * L::kFloor && mine.r < 1e30f)) {  // logits near the value that stands for -inf, or near overflow
#pragma unroll
      for (int u = 0; u < N; ++u) {
        float x[L::kVec];
        L::unpack(v[u], x);
#pragma unroll
        for (int j = 0; j < L::kVec; ++j) mine.add(x[j]);
      }
      return;
    }
    const unsigned long long k = f2(kLog2e, kLog2e), r = f2(-mine.r, -mine.r);
    unsigned long long s2 = 0ull, w2 = 0ull;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[L::kVec];
      L::unpack(L::floored(v[u]), x);
#pragma unroll
      for (int j = 0; j < L::kVec; j += 2) {
        const unsigned long long t = f2_mul(f2_add(f2(x[j], x[j + 1]), r), k);
        const float2 q = f2_split(t);
        const unsigned long long e = f2(ex2(q.x), ex2(q.y));
        s2 = f2_add(s2, e);
        w2 = f2_fma(e, t, w2);
      }
    }
    const float2 s = f2_split(s2), w = f2_split(w2);
    mine.s += s.x + s.y;
    mine.w += w.x + w.y;
  };
  {
    const uint4* p = share.vectors();
    int i = share.lo + tid;
    for (; i + 3 * kThreads < share.hi; i += 4 * kThreads) {
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = __ldg(p + i + u * kThreads);
      take(std::integral_constant<int, 4>(), v);
    }
    for (; i < share.hi; i += kThreads) {
      const uint4 v = __ldg(p + i);
      take(std::integral_constant<int, 1>(), &v);
    }
    if (tid < 2 * L::kVec) {
      const int at = share.outside(tid);
      if (at >= 0) {
        const float z = L::one(share.row + at);
        my_most = fmaxf(my_most, z);
        if (z > mine.r) mine.raise(z);
        if (mine.r == -INFINITY) mine.s += z == z ? 0.f : z;
        else mine.add(z);
      }
    }
  }
  if (a.top > 0) {
    float most = my_most;
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane % kGroup == 0) s_group[tid / kGroup] = most;
  }
  join_warp(mine);
  const float warp_most = warp_max(my_most);
  // the address of a variable in the row's first CTA
  auto home = [&](const void* p) {
    uint32_t at = ptx::smem_u32(p);
    if (a.ranks > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(at));
    return at;
  };
  auto put = [](uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); };
  auto put_key = [&](int place, unsigned long long key) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(home(&s_all[rank * a.top + place])), "l"(key) : "memory");
  };
  if (a.ranks > 1) ptx::cluster_wait();
  if (lane == 0) {
    const int w = rank * (kThreads / 32) + warp;
    const uint32_t at = home(&s_warp[w]);
    put(at, mine.r);
    put(at + 4, mine.s);
    put(at + 8, mine.w);
    put(home(&s_warp_max[w]), warp_most);
  }
  __syncthreads();
  if (a.top > 0) {
    if (tid < kGroups) {  // the top-th largest of the groups' maxima: equal ones by place
      const float x = s_group[tid];
      int before = 0;
#pragma unroll
      for (int i = 0; i < kGroups; i += 4) {
        const float4 y = *reinterpret_cast<const float4*>(&s_group[i]);
        before += y.x > x || (y.x == x && i < tid);
        before += y.y > x || (y.y == x && i + 1 < tid);
        before += y.z > x || (y.z == x && i + 2 < tid);
        before += y.w > x || (y.w == x && i + 3 < tid);
      }
      if (before == a.top - 1) s_bar = x;
    }
    __syncthreads();
    const float bar = s_bar;
    auto list = [&](float z, int index) {
      if (z >= bar) {
        const int at = atomicAdd(&s_count, 1);
        if (at < kListed) s_list[at] = key_of(z, index);
      }
    };
    if (tid < 2 * L::kVec) {
      const int at = share.outside(tid);
      if (at >= 0) list(L::one(share.row + at), at);
    }
    auto look = [&](int i) {
      float x[L::kVec];
      L::unpack(__ldg(share.vectors() + i), x);
#pragma unroll
      for (int j = 0; j < L::kVec; ++j) list(x[j], share.head + i * L::kVec + j);
    };
    const int per = (share.hi - share.lo + kThreads - 1) / kThreads;
    if (per <= 4) {
      if (my_most >= bar)
        for (int i = share.lo + tid; i < share.hi; i += kThreads) look(i);
    } else {  // the vectors of all these threads, one a thread and turn
      if (my_most >= bar) s_flagged[atomicAdd(&s_flags, 1)] = tid;
      __syncthreads();
      const int n = s_flags * per;
      for (int q = tid; q < n; q += kThreads) {
        const int i = share.lo + s_flagged[q / per] + q % per * kThreads;
        if (i < share.hi) look(i);
      }
    }
    __syncthreads();
    const int count = s_count;
    if (count <= kListed) {
      for (int c = tid; c < count; c += kThreads) {
        const unsigned long long key = s_list[c];
        const int before = better(s_list, count, key);
        if (before < a.top) put_key(before, key);
      }
    } else {  // too many: one search for each place, for the best below the one before
      unsigned long long last = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        unsigned long long best = 0;
        if (my_most >= bar)
          share.each_of_mine([&](float z, int index) {
            if (z >= bar) {
              const unsigned long long key = key_of(z, index);
              if (key < last) best = max_u64(best, key);
            }
          });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max_u64(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) s_list[warp] = best;
        __syncthreads();
        best = s_list[0];
        for (int w = 1; w < kThreads / 32; ++w) best = max_u64(best, s_list[w]);
        if (tid == 0) put_key(k, best);
        last = best;
        __syncthreads();
      }
    }
  }
  // ---- the row's first CTA has everything
  __syncwarp();
  if (a.ranks > 1) {
    ptx::cluster_arrive();
    if (rank != 0) return;
    ptx::cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == kThreads / 32 - 1) {
    const int n = a.ranks * (kThreads / 32);
    Stats x;
    float most = -INFINITY;
    if (lane < n) {
      x = s_warp[lane];
      most = s_warp_max[lane];
    }
    join_warp(x);
    most = warp_max(most);
    if (lane == 0) {
      s_row = x;
      s_max = most;
    }
  } else if (a.ranks > 1 && tid < a.top) {
    s_best[tid] = 0;
  }
  const unsigned long long* best = s_all;
  __syncthreads();
  if (a.ranks > 1 && a.top > 0) {
    const int n = a.ranks * a.top;
    if (tid < n) {
      const unsigned long long key = s_all[tid];
      const int before = better(s_all, n, key);
      if (key != 0 && before < a.top) s_best[before] = key;
    }
    best = s_best;
    __syncthreads();
  }
  const Stats all = s_row;
  const float m = s_max;
  const bool nothing = m == -INFINITY && all.s == 0.f;  // a row of -inf
  const float log2_s = log2f(all.s);
  const float log_s = nothing ? 0.f : m == -INFINITY ? all.s : fmaf(kLn2, log2_s, all.r - m);
  if (tid == 0) {
    a.stats[row] = make_float2(m, log_s);
    if (a.entropy) a.entropy[row] = nothing ? 0.f : kLn2 * (log2_s - all.w / all.s);
    if (a.logp) {
      float r = 0.f;
      if (target >= a.vocab) {
        atomicCAS(a.err, 0, kSiteToken);
        r = NAN;
      } else if (target >= 0) {
        r = nothing ? -INFINITY : (z_target - m) - log_s;
      }
      a.logp[row] = r;
    }
  }
  if (tid < a.top) {
    const unsigned long long key = best[tid];
    const bool none = key == 0;  // fewer logits than places that are numbers
    a.top_ids[static_cast<int64_t>(row) * a.top + tid] = none ? -1 : index_of(key);
    a.top_logp[static_cast<int64_t>(row) * a.top + tid] =
        none ? NAN : nothing ? -INFINITY : (value_of(key) - m) - log_s;
  }
}

struct GradArgs {
  void* out;
  int64_t out_pitch;
  const void* logits;
  int64_t pitch;
  const int32_t* targets;
  const float2* stats;
  const float* entropy;
  const float* g_logp;
  const float* g_entropy;
  const int32_t* top_ids;
  const float* g_top;
  int vocab, top, chunks;
  int* err;
};

constexpr int kGradVecs = 4;  // vectors of a thread

template <int TYPE>
__global__ void __launch_bounds__(256) token_logprobs_grad_kernel(const GradArgs a) {
  using L = Logits<TYPE>;
  using T = typename L::T;
  RT_PDL_WAIT();
  RT_PDL_LAUNCH_DEPENDENTS();
  const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks;
  const int tid = threadIdx.x;
  const Share<TYPE> share(static_cast<const T*>(a.logits) + row * a.pitch, a.vocab, 0, 1);
  T* out = static_cast<T*>(a.out) + row * a.out_pitch;
  // the logits are on their way while the row's terms are read
  const uint4* src = share.vectors();
  const int v0 = chunk * 256 * kGradVecs + tid;
  uint4 v[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    v[u] = make_uint4(0, 0, 0, 0);
    if (v0 + u * 256 < share.nv) v[u] = src[v0 + u * 256];
  }
  const float2 st = a.stats[row];
  const int target = a.g_logp ? a.targets[row] : -1;
  const bool given = target >= 0 && target < a.vocab;
  if (target >= a.vocab && chunk == 0 && tid == 0) atomicCAS(a.err, 0, kSiteToken);
  const float g_t = given ? a.g_logp[row] : 0.f;
  // every warp reads the alternatives, one a lane
  const int lane = tid & 31, warp = tid >> 5;
  const int64_t alt = static_cast<int64_t>(row) * a.top + lane;
  const float g_alt = lane < a.top ? a.g_top[alt] : 0.f;
  const int id = lane < a.top ? a.top_ids[alt] : -1;
  const float pull = g_t + (a.top > 0 ? warp_sum(g_alt) : 0.f);
  const float g_h = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float h = a.g_entropy ? a.entropy[row] : 0.f;
  const bool nothing = st.x == -INFINITY && st.y == 0.f;  // a row of -inf; with a NaN among them its gradient is NaN
  constexpr float kLeast = -1e4f;  // of log p: p = 0 leaves nothing there, and with -inf it would be 0 * inf
  auto grad = [&](float z) {
    const float lp = max_nan((z - st.x) - st.y, kLeast);
    return nothing ? 0.f : -ex2(lp * kLog2e) * fmaf(g_h, lp + h, pull);
  };
  // columns with a term of their own, before anything is overwritten (out may be the logits)
  int column = -1;
  float special = 0.f;
  const int first = share.head + chunk * 256 * kGradVecs * L::kVec;
  const int behind = min(share.head + share.nv * L::kVec, first + 256 * kGradVecs * L::kVec);
  if (warp < 2) {  // warp 0: the alternatives, lane 0 of warp 1: the target
    column = warp == 0 ? id : lane == 0 && given ? target : -1;
    if (column >= a.vocab) {
      if (chunk == 0) atomicCAS(a.err, 0, kSiteToken);
      column = -1;
    }
    const bool in_vectors = column >= share.head && column < share.head + share.nv * L::kVec;
    if (!(in_vectors ? column >= first && column < behind : chunk == 0)) column = -1;
    if (__any_sync(0xffffffffu, column >= 0)) {
      float own = given && column == target ? g_t : 0.f;
      for (int j = 0; j < a.top; ++j) {
        const float g = __shfl_sync(0xffffffffu, g_alt, j);
        if (__shfl_sync(0xffffffffu, id, j) == column) own += g;
      }
      if (column >= 0) special = grad(L::one(share.row + column)) + (nothing ? 0.f : own);
    }
  }
  __syncthreads();
  const bool aligned = (reinterpret_cast<uintptr_t>(out + share.head) & 15u) == 0;
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int i = v0 + u * 256;
    if (i >= share.nv) break;
    float x[L::kVec];
    L::unpack(v[u], x);
#pragma unroll
    for (int j = 0; j < L::kVec; j += 2) {  // as `grad`, two at a time
      const unsigned long long full = f2_add(f2_add(f2(x[j], x[j + 1]), f2(-st.x, -st.x)), f2(-st.y, -st.y));
      const float2 cut = f2_split(full);
      const unsigned long long lp = f2(max_nan(cut.x, kLeast), max_nan(cut.y, kLeast));
      const float2 t = f2_split(f2_mul(lp, f2(kLog2e, kLog2e)));
      const unsigned long long c = f2_fma(f2(-g_h, -g_h), f2_add(lp, f2(h, h)), f2(-pull, -pull));
      const float2 d = f2_split(f2_mul(f2(ex2(t.x), ex2(t.y)), c));
      x[j] = nothing ? 0.f : d.x;
      x[j + 1] = nothing ? 0.f : d.y;
    }
    T* dst = out + share.head + static_cast<int64_t>(i) * L::kVec;
    if (aligned) {
      *reinterpret_cast<uint4*>(dst) = L::pack(x);
    } else {
#pragma unroll
      for (int j = 0; j < L::kVec; ++j) dst[j] = L::from(x[j]);
    }
  }
  if (chunk == 0 && tid < 2 * L::kVec) {
    const int at = share.outside(tid);
    if (at >= 0) out[at] = L::from(grad(L::one(share.row + at)));
  }
  __syncthreads();
  if (column >= 0) out[column] = L::from(special);
}

int type_size(int dtype) { return dtype == RT_F32 ? 4 : 2; }

rt_status check_logits(const char* what, const void* logits, int64_t pitch, int rows, int vocab, int dtype) {
  RT_REQUIRE(dtype == RT_F16 || dtype == RT_BF16 || dtype == RT_F32, RT_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  RT_REQUIRE(rows >= 0 && vocab > 0 && pitch >= vocab, RT_ERR_INVALID, "%s: need rows >= 0, vocab > 0 and a row pitch of at least that",
             what);
  RT_REQUIRE(vocab <= (1 << 30), RT_ERR_UNSUPPORTED, "%s: vocabulary of %d", what, vocab);
  RT_REQUIRE(rows == 0 || logits, RT_ERR_INVALID, "%s: null pointer", what);
  RT_REQUIRE(reinterpret_cast<uintptr_t>(logits) % type_size(dtype) == 0, RT_ERR_INVALID, "%s: misaligned logits", what);
  return RT_OK;
}

}  // namespace
}  // namespace rt

using namespace rt;

namespace {

// A row takes about as long as all others, so the CTAs come in rounds, and the last round is as long as a full one.  More CTAs on an SM have
// fewer registers for loads in flight and take longer for a round (592 rows of 50,358 fp16 logits: 4 CTAs an SM 16.3 us, 5: 18.5, 6: 20.7), in
// the ratio CTAs + 3.5, but there may be fewer rounds: 2,048 rows 53.2, 48.1, 48.0 us, 4,096 rows 95.8, 87.9, 83.4, 700 rows 25.4, 19.1, 21.1.
int ctas_of_an_sm(int64_t ctas) {
  int best = 4;
  double least = 0;
  for (int n = 4; n <= 6; ++n) {
    const double cost = static_cast<double>((ctas + kSms * n - 1) / (kSms * n)) * (n + 3.5);
    if (n == 4 || cost < least) {
      best = n;
      least = cost;
    }
  }
  return best;
}

template <int TYPE>
void (*kernel_of(int ctas))(const ScoreArgs) {
  return ctas == 4 ? token_logprobs_kernel<TYPE, 4> : ctas == 5 ? token_logprobs_kernel<TYPE, 5> : token_logprobs_kernel<TYPE, 6>;
}

}  // namespace

extern "C" rt_status rt_token_logprobs(const void* logits, int64_t pitch, const int32_t* targets, int rows, int vocab, int top,
                                       float* logp, float* entropy, float* stats, int32_t* top_ids, float* top_logp, int dtype,
                                       void* stream) {
  RT_TRY(check_logits("token_logprobs", logits, pitch, rows, vocab, dtype));
  RT_REQUIRE(top >= 0 && top <= kMaxTop && top <= vocab, RT_ERR_UNSUPPORTED,
             "token_logprobs: %d alternatives (0 to 32, at most the vocabulary)", top);
  if (rows == 0) return RT_OK;
  RT_REQUIRE(stats && (!logp || targets) && (top == 0 || (top_ids && top_logp)), RT_ERR_INVALID, "token_logprobs: null pointer");
  RT_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7u) == 0, RT_ERR_INVALID, "token_logprobs: stats must be 8-byte aligned");
  ScoreArgs a{logits, pitch, targets, rows, vocab, top, 1, logp, entropy, reinterpret_cast<float2*>(stats), top_ids, top_logp,
              device_error_word()};
  RT_REQUIRE(a.err != nullptr, RT_ERR_CUDA, "token_logprobs: cannot allocate the device error word");
  // few rows: several CTAs for each, as long as every thread has four vectors
  const int vectors = vocab / (16 / type_size(dtype));
  while (a.ranks < kMaxRanks && static_cast<int64_t>(rows) * a.ranks * 2 <= kSms && vectors >= 4 * kThreads * a.ranks) a.ranks *= 2;
  RT_REQUIRE(static_cast<int64_t>(rows) * a.ranks < (int64_t{1} << 31), RT_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  const int held = ctas_of_an_sm(static_cast<int64_t>(rows) * a.ranks);
  auto kern = dtype == RT_F32 ? kernel_of<RT_F32>(held) : dtype == RT_BF16 ? kernel_of<RT_BF16>(held) : kernel_of<RT_F16>(held);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * a.ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.ranks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.ranks > 1 ? 2 : 1;
  RT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  count_launch();
  RT_CHECK_CUDA(cudaGetLastError());
  return RT_OK;
}

extern "C" rt_status rt_token_logprobs_backward(void* dlogits, int64_t out_pitch, const void* logits, int64_t pitch,
                                                const int32_t* targets, const float* stats, const float* entropy, int rows, int vocab,
                                                const float* g_logp, const float* g_entropy, int top, const int32_t* top_ids,
                                                const float* g_top, int dtype, void* stream) {
  RT_TRY(check_logits("token_logprobs_backward", logits, pitch, rows, vocab, dtype));
  RT_REQUIRE(top >= 0 && top <= kMaxTop && top <= vocab, RT_ERR_UNSUPPORTED,
             "token_logprobs_backward: %d alternatives (0 to 32, at most the vocabulary)", top);
  RT_REQUIRE(out_pitch >= vocab, RT_ERR_INVALID, "token_logprobs_backward: the output's row pitch is below the vocabulary");
  if (rows == 0) return RT_OK;
  RT_REQUIRE(dlogits && stats && (!g_logp || targets) && (!g_entropy || entropy) && (top == 0 || (top_ids && g_top)), RT_ERR_INVALID,
             "token_logprobs_backward: null pointer");
  RT_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7u) == 0 && reinterpret_cast<uintptr_t>(dlogits) % type_size(dtype) == 0, RT_ERR_INVALID,
             "token_logprobs_backward: misaligned stats or output");
  RT_REQUIRE(dlogits != logits || out_pitch == pitch, RT_ERR_INVALID,
             "token_logprobs_backward: in place, the output has the logits' row pitch");
  GradArgs a{dlogits, out_pitch, logits, pitch, targets, reinterpret_cast<const float2*>(stats), entropy, g_logp, g_entropy, top_ids,
             g_top, vocab, top, 1, device_error_word()};
  RT_REQUIRE(a.err != nullptr, RT_ERR_CUDA, "token_logprobs_backward: cannot allocate the device error word");
  const int vec = 16 / type_size(dtype);
  a.chunks = std::max(1, (vocab / vec + 256 * kGradVecs - 1) / (256 * kGradVecs));
  RT_REQUIRE(static_cast<int64_t>(rows) * a.chunks < (int64_t{1} << 31), RT_ERR_UNSUPPORTED, "token_logprobs_backward: too many rows");
  auto kern = dtype == RT_F32   ? token_logprobs_grad_kernel<RT_F32>
              : dtype == RT_BF16 ? token_logprobs_grad_kernel<RT_BF16>
                                 : token_logprobs_grad_kernel<RT_F16>;
  RT_CHECK_CUDA(launch_kernel(kern, dim3(static_cast<unsigned>(rows * a.chunks)), dim3(256), 0, static_cast<cudaStream_t>(stream), a));
  count_launch();
  RT_CHECK_CUDA(cudaGetLastError());
  return RT_OK;
}
