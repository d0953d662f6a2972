// Writing keys and values of new tokens into the 8-bit cache, and reading them back (layout: kv_cache.cuh).
//
// A block's scale follows its tokens.  With a = the largest finite |value| that a call adds to the block,
//   need = e4m3: the smallest power of two >= a / 448;  int8: a / 127 rounded up to eight significant bits;  at least 2^-100.
// A block that holds earlier tokens keeps its scale if it is >= need; otherwise the scale becomes `need` and the earlier codes c
// become round(c * old / need).  New codes are round(x / scale), ties to even.
// The scale's few bits cost int8 at most 1/128 of its range and e4m3 none of its precision (a power of two moves the
// exponent), and they make every code exact: x has at most 11 significant bits and the scale 8, so a quotient that is not itself on a border
// between two codes is at least 2^-17 away from it, more than a correctly rounded fp32 division moves it (2^-18 at 127).  So every
// implementation of the definition gets the same codes.  Scales made elsewhere may have all 24 bits: there a code is that of the quotient as fp32 has
// it.
//
// Both kernels move bytes: 2 in and 1 out a value, or the reverse.  Two warps take one block of one head, keys or values: its
// 64 rows of 128 bytes stay in registers between the maximum and the rounding, one pass over the data.
#include "kv_cache.cuh"

#include <algorithm>
#include <type_traits>

#include "device_error.h"
#include "launch.h"
#include "launch_count.h"

namespace rt {

rt_status check_kv_cache(const char* what, const rt_kv_cache* c, KvView* view) {
  RT_REQUIRE(c != nullptr, RT_ERR_INVALID, "%s: null cache", what);
  RT_REQUIRE(c->k_dev && c->v_dev && c->k_scale_dev && c->v_scale_dev, RT_ERR_INVALID, "%s: null pointer in the cache", what);
  RT_REQUIRE(c->blocks > 0 && c->kv_heads > 0 && c->kv_heads <= 1024, RT_ERR_INVALID,
             "%s: a cache needs blocks > 0 and 1 to 1024 heads (got %d, %d)", what, c->blocks, c->kv_heads);
  RT_REQUIRE(c->format == RT_KV_E4M3 || c->format == RT_KV_INT8, RT_ERR_INVALID, "%s: unknown cache format %d", what, c->format);
  RT_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_dev) | reinterpret_cast<uintptr_t>(c->v_dev)) & 15u) == 0, RT_ERR_INVALID,
             "%s: cache buffers must be 16-byte aligned", what);
  RT_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_scale_dev) | reinterpret_cast<uintptr_t>(c->v_scale_dev)) & 3u) == 0, RT_ERR_INVALID,
             "%s: scales must be 4-byte aligned", what);
  *view = KvView{static_cast<uint8_t*>(c->k_dev), static_cast<uint8_t*>(c->v_dev), c->k_scale_dev, c->v_scale_dev, c->blocks,
                 c->kv_heads};
  return RT_OK;
}

namespace {

// What one warp works on: tokens [lo, hi) (positions in the sequence) of one block.
struct Span {
  int page;          // block of the cache, < 0: nothing to do
  int64_t base, lo, hi;
  int64_t row0;      // packed row of position 0 (may be negative: only positions >= start are used)
  int first, len;    // of the sequence in the packed rows
};

__device__ __forceinline__ Span span_of(int seq, int nth, const int32_t* __restrict__ table, int table_stride,
                                        const int32_t* __restrict__ start, const int32_t* __restrict__ first, int tokens, int max_tokens,
                                        int blocks, int* err, int site) {
  Span s;
  s.page = -1;
  const int f0 = first[seq], f1 = first[seq + 1], p0 = start[seq];
  if (f1 <= f0) return s;
  if (f0 < 0 || f1 > tokens || p0 < 0 || f1 - f0 > max_tokens) {
    kv::index_error(err, site);
    return s;
  }
  s.first = f0;
  s.len = f1 - f0;
  s.row0 = static_cast<int64_t>(f0) - p0;
  const int64_t b = p0 / 64 + nth, end = static_cast<int64_t>(p0) + s.len;
  s.base = b * 64;
  s.lo = s.base > p0 ? s.base : p0;
  s.hi = s.base + 64 < end ? s.base + 64 : end;
  if (s.lo >= s.hi) return s;
  const int page = b < table_stride ? table[static_cast<int64_t>(seq) * table_stride + b] : -1;
  if (page < 0 || page >= blocks) {
    kv::index_error(err, site);
    return s;
  }
  s.page = page;
  return s;
}

// Which sequence and which of its blocks a CTA takes.  Direct: every sequence has `spans` places, as many as its longest one may need.  From a list
// (kv::find_place): a sequence of n tokens touches at most (n + 62) / 64 + 1 blocks, never more than n / 64 + 2.
template <bool LISTED>
__device__ __forceinline__ kv::Place place_of(int at, int spans, const int32_t* __restrict__ first, int n_seq, int tokens, int max_tokens, int* err,
                                              int site) {
  if constexpr (!LISTED) return kv::Place{at / spans, at % spans};
  __shared__ kv::Place found;
  __shared__ int count;
  return kv::find_place(at, first, n_seq, 1, 6, 2, tokens, max_tokens, &found, &count, err, site);
}

// The packed row of 64 values of token `t` (row of the batch): token-major with strides, or head-major per sequence
// (rt_qkv_bias_transpose).
__device__ __forceinline__ int64_t value_offset(const Span& s, int64_t t, int head, int heads, int64_t token_stride,
                                                int64_t head_stride) {
  if (token_stride == 0) return (static_cast<int64_t>(s.first) * heads + static_cast<int64_t>(head) * s.len + (t - s.first)) * 64;
  return t * token_stride + head * head_stride;
}

template <bool INT8>
__device__ __forceinline__ float scale_for(float most) {
  const uint32_t low = INT8 ? 0xffffu : 0x7fffffu;  // mantissa bits that a scale does not have
  const uint32_t bits = __float_as_uint(most / (INT8 ? kv::kInt8Max : kv::kE4m3Max));
  return fmaxf(__uint_as_float((bits + low) & ~low), kv::kMinScale);
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
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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

// Codes of x / scale: the quotient from the correctly rounded reciprocal y by Markstein's correction, q = x y,
// q + (x - q s) y, which is the correctly rounded one (P. Markstein, IBM J. Res. Dev. 34, 1990), also for scales that were not made here.  int8: rounded to
// a whole number by adding 1.5 * 2^23, whose last byte is the code.
template <bool INT8>
struct Coder {
  unsigned long long inv, neg;
  __device__ __forceinline__ explicit Coder(float scale) {
    const float y = __frcp_rn(scale);
    inv = f2(y, y);
    neg = f2(-scale, -scale);
  }
  // what infinities become
  static __device__ __forceinline__ uint32_t largest(bool negative) { return INT8 ? (negative ? 0x81u : 0x7fu) : (negative ? 0xfeu : 0x7eu); }
  __device__ __forceinline__ uint32_t four(const float* x) const {
    const unsigned long long a = f2(x[0], x[1]), b = f2(x[2], x[3]);
    unsigned long long p = f2_mul(a, inv), q = f2_mul(b, inv);
    p = f2_fma(f2_fma(p, neg, a), inv, p);
    q = f2_fma(f2_fma(q, neg, b), inv, q);
    if constexpr (INT8) {
      const unsigned long long magic = f2(12582912.f, 12582912.f);
      const float2 u = f2_split(f2_add(p, magic)), v = f2_split(f2_add(q, magic));
      const uint32_t lo = kv::prmt(__float_as_uint(u.x), __float_as_uint(u.y), 0x0040u);
      return kv::prmt(lo, kv::prmt(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040u), 0x5410u);
    } else {
      const float2 u = f2_split(p), v = f2_split(q);
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(u, __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
      return lo | (hi << 16);
    }
  }
};

// values of four codes, times `scale`
template <bool INT8>
__device__ __forceinline__ void values4(uint32_t w, float scale, float* x) {
  using C = kv::Codes<INT8>;
  const uint32_t p = C::prepare(w);
  const float2 a = kv::unpack16<false>(C::template pair<0>(p)), b = kv::unpack16<false>(C::template pair<2>(p));
  x[0] = a.x * scale;
  x[1] = a.y * scale;
  x[2] = b.x * scale;
  x[3] = b.y * scale;
}

// grid: (block of the sequence, head) pairs of every sequence; warps 0 and 1 take the keys, 2 and 3 the values, 32 tokens each.
// A tile is read once, and its largest value is known before the first code is: it stays in registers.  Two warps for a tile keep 36
// warps an SM at that (32: 19.9 us, 40: 21.3, they spill).  8 sequences of 1024 to 4096 tokens, 12 heads, f16 to int8 (95 MB): 19.5 us of device time, 20.1 a call, 4.9 TB/s,
// bound by HBM and a CTA's chain of index, load, maximum, store; one warp a tile, quotients by division and maxima in fp32 took 67.7.  A step's tokens (32 sequences, 12 heads) are that
// chain alone, 2.8 us.
constexpr int kWriteThreads = 128;
template <bool BF16, bool INT8, bool LISTED>
__global__ void __launch_bounds__(kWriteThreads, 9)
kv_write_kernel(KvView c, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int64_t token_stride, int64_t head_stride,
                const int32_t* __restrict__ table, int table_stride, const int32_t* __restrict__ start,
                const int32_t* __restrict__ first, int n_seq, int tokens, int max_tokens, int spans, int* err) {
  __shared__ uint32_t s_most[kWriteThreads / 32];
  RT_PDL_WAIT();
  RT_PDL_LAUNCH_DEPENDENTS();  // not before the wait: launches would queue up on the SMs
  const int head = blockIdx.x % c.heads;
  const kv::Place place = place_of<LISTED>(blockIdx.x / c.heads, spans, first, n_seq, tokens, max_tokens, err, kSiteCacheWrite);
  if (place.seq < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool values = warp >= 2;
  const Span s = span_of(place.seq, place.nth, table, table_stride, start, first, tokens, max_tokens, c.blocks, err, kSiteCacheWrite);
  if (s.page < 0) return;
  const int64_t slot = static_cast<int64_t>(s.page) * c.heads + head;
  uint8_t* dst = (values ? c.v : c.k) + slot * 4096;
  float* scale_at = (values ? c.v_scale : c.k_scale) + slot;
  const bool older = s.lo > s.base;
  const float was = older ? *scale_at : 0.f;

  // eight lanes a row, four rows an instruction
  const int row0 = (warp & 1) * 32 + (lane >> 3), col = (lane & 7) * 8;
  const int lo = static_cast<int>(s.lo - s.base), hi = static_cast<int>(s.hi - s.base);
  uint4 w[8];
  {
    const int64_t t = s.row0 + s.base + row0;
    const uint16_t* x = (values ? v : k) + value_offset(s, t, head, c.heads, token_stride, head_stride) + col;
    const int64_t step = 4 * (token_stride == 0 ? 64 : token_stride);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (row0 + 4 * i >= lo && row0 + 4 * i < hi) w[i] = __ldg(reinterpret_cast<const uint4*>(x + i * step));
    }
  }
  // the largest magnitude: without their signs the bits order as the numbers do, infinity and NaN on top
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(&w[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __vmaxu2(top, p[j] & 0x7fff7fffu);
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  const bool strange = top >= kInf;  // of the whole warp
  if (strange) {                     // the largest finite one then
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(&w[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = p[j] & 0x7fffu, b = (p[j] >> 16) & 0x7fffu;
        top = max(top, max(a < kInf ? a : 0u, b < kInf ? b : 0u));
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  if (lane == 0) s_most[warp] = top;
  __syncthreads();  // also: both warps of the tile have read the old scale
  top = max(top, s_most[warp ^ 1]);
  const float need = scale_for<INT8>(kv::unpack16<BF16>(top).x);
  const bool keep = older && need <= was;
  const float scale = keep ? was : need;
  const Coder<INT8> code(scale);
  if (older && !keep) {  // the earlier tokens' codes, four lanes a row
    for (int r = (warp & 1) * 8 + (lane >> 2); r < lo; r += 16) {
      uint4* at = reinterpret_cast<uint4*>(dst + r * 64 + (lane & 3) * 16);
      uint4 old = *at;
      uint32_t* p = reinterpret_cast<uint32_t*>(&old);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[4];
        values4<INT8>(p[j], was, f);
        p[j] = code.four(f);
      }
      *at = old;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = row0 + 4 * i;
    if (r < lo || r >= hi) continue;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(&w[i]);
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = kv::unpack16<BF16>(p[j]);
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
    uint32_t infinite[2] = {0u, 0u};  // the codes of the infinities among them, whose quotients are 0 here
    if (strange) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (fabsf(f[j]) < INFINITY) continue;
        if (f[j] == f[j]) infinite[j >> 2] |= code.largest(f[j] < 0.f) << (8 * (j & 3));
        f[j] = 0.f;
      }
    }
    *reinterpret_cast<uint2*>(dst + r * 64 + col) = make_uint2(code.four(f) | infinite[0], code.four(f + 4) | infinite[1]);
  }
  if ((warp & 1) == 0 && lane == 0 && !keep) *scale_at = scale;
}

// The same grid and warps; out_k / out_v are token-major [tokens][heads * 64].  Bound by HBM: 249 MB in 42.4 us, 5.9 TB/s.
template <bool BF16, bool INT8, bool LISTED>
__global__ void __launch_bounds__(kWriteThreads, 9)
kv_read_kernel(KvView c, uint16_t* __restrict__ out_k, uint16_t* __restrict__ out_v, const int32_t* __restrict__ table,
               int table_stride, const int32_t* __restrict__ start, const int32_t* __restrict__ first, int n_seq, int tokens, int max_tokens, int spans,
               int* err) {
  RT_PDL_WAIT();
  RT_PDL_LAUNCH_DEPENDENTS();
  const int head = blockIdx.x % c.heads;
  const kv::Place place = place_of<LISTED>(blockIdx.x / c.heads, spans, first, n_seq, tokens, max_tokens, err, kSiteCacheRead);
  if (place.seq < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool values = warp >= 2;
  const Span s = span_of(place.seq, place.nth, table, table_stride, start, first, tokens, max_tokens, c.blocks, err, kSiteCacheRead);
  if (s.page < 0) return;
  const int64_t slot = static_cast<int64_t>(s.page) * c.heads + head;
  const int row0 = (warp & 1) * 32 + (lane >> 3), col = (lane & 7) * 8;
  const int lo = static_cast<int>(s.lo - s.base), hi = static_cast<int>(s.hi - s.base);
  const uint8_t* src = (values ? c.v : c.k) + slot * 4096 + row0 * 64 + col;
  const float scale = (values ? c.v_scale : c.k_scale)[slot];
  uint16_t* out = (values ? out_v : out_k) + ((s.row0 + s.base + row0) * c.heads + head) * 64 + col;
  uint2 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = make_uint2(0, 0);
    if (row0 + 4 * i >= lo && row0 + 4 * i < hi) w[i] = __ldg(reinterpret_cast<const uint2*>(src + 256 * i));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (row0 + 4 * i < lo || row0 + 4 * i >= hi) continue;
    float f[8];
    values4<INT8>(w[i].x, scale, f);
    values4<INT8>(w[i].y, scale, f + 4);
    uint4 o;
    o.x = kv::pack16<BF16>(f[0], f[1]);
    o.y = kv::pack16<BF16>(f[2], f[3]);
    o.z = kv::pack16<BF16>(f[4], f[5]);
    o.w = kv::pack16<BF16>(f[6], f[7]);
    *reinterpret_cast<uint4*>(out + static_cast<int64_t>(i) * 4 * c.heads * 64) = o;
  }
}

// Blocks that `max_tokens` new tokens of a sequence touch at most, wherever they start.
int spans_of(int max_tokens) { return static_cast<int>((static_cast<int64_t>(max_tokens) + 62) / 64 + 1); }

// How a call's CTAs find their work, and how many there are.
struct Plan {
  int64_t grid;
  bool listed;
};

rt_status check_ragged(const char* what, const int32_t* table, int table_stride, const int32_t* start, const int32_t* first, int n_seq,
                       int tokens, int max_tokens, int kv_heads, int dtype, Plan* plan) {
  RT_REQUIRE(table && start && first, RT_ERR_INVALID, "%s: null pointer", what);
  RT_REQUIRE(dtype == RT_F16 || dtype == RT_BF16, RT_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  RT_REQUIRE(n_seq >= 0 && tokens >= 0 && table_stride > 0 && max_tokens >= 0, RT_ERR_INVALID, "%s: bad sizes", what);
  *plan = Plan{0, false};
  if (n_seq == 0 || tokens == 0 || max_tokens == 0) return RT_OK;
  const int64_t direct = static_cast<int64_t>(n_seq) * spans_of(std::min(max_tokens, tokens)), places = tokens / 64 + int64_t{2} * n_seq;  // under 2^57
  // A CTA without work costs 10 to 15 ns of a call, a CTA that looks for its sequence 7 % more and as much again for each 1000 sequences.  12 heads, int8,
  // us direct and listed: 8 x 4096 tokens with 1.0 CTAs for each place 24.8 and 26.6, with 2.0 27.2 and 26.6, with 7.8 (any of them may bring all) 55.8 and
  // 26.6; 64 x 2048, 60: 1632 and 96; 300 x 40, 2.3: 25.0 and 21.6; 1000 x 65, 2.0: 98 and 127, 11: 424 and 127; 5000 x 1, 1.0: 152 and 948.
  plan->listed = static_cast<double>(direct) > static_cast<double>(places) * (2.0 + n_seq * 1e-3);
  const int64_t ctas = plan->listed ? places : direct;
  RT_REQUIRE(ctas < (int64_t{1} << 31) && ctas * kv_heads < (int64_t{1} << 31), RT_ERR_UNSUPPORTED,
             "%s: %d sequences of up to %d tokens are too many for one call", what, n_seq, max_tokens);
  plan->grid = ctas * kv_heads;
  return RT_OK;
}

// The kernel for the 16-bit type, the cache's format and the plan.
template <typename F>
auto choose(bool bf16, bool int8, bool listed, F kernel) {
  using T = std::true_type;
  using N = std::false_type;
  auto with = [&](auto b, auto i) { return listed ? kernel(b, i, T()) : kernel(b, i, N()); };
  return bf16 ? (int8 ? with(T(), T()) : with(T(), N())) : (int8 ? with(N(), T()) : with(N(), N()));
}

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" rt_status rt_kv_cache_write(const rt_kv_cache* cache, const void* k, const void* v, int64_t token_stride,
                                       int64_t head_stride, const int32_t* table, int table_stride, const int32_t* start,
                                       const int32_t* first, int n_seq, int tokens, int max_tokens, int dtype, void* stream) {
  KvView c;
  Plan plan;
  RT_TRY(check_kv_cache("kv_cache_write", cache, &c));
  RT_TRY(check_ragged("kv_cache_write", table, table_stride, start, first, n_seq, tokens, max_tokens, c.heads, dtype, &plan));
  if (plan.grid == 0) return RT_OK;
  RT_REQUIRE(k && v, RT_ERR_INVALID, "kv_cache_write: null pointer");
  RT_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 && token_stride % 8 == 0 &&
                 head_stride % 8 == 0 && token_stride >= 0 && head_stride >= 0,
             RT_ERR_INVALID, "kv_cache_write: keys and values must be 16-byte aligned, with strides that are multiples of 8 values");
  int* err = device_error_word();
  RT_REQUIRE(err != nullptr, RT_ERR_CUDA, "kv_cache_write: cannot allocate the device error word");
  auto kern = choose(dtype == RT_BF16, cache->format == RT_KV_INT8, plan.listed, [](auto bf16, auto int8, auto listed) {
    return kv_write_kernel<decltype(bf16)::value, decltype(int8)::value, decltype(listed)::value>;
  });
  RT_CHECK_CUDA(launch_kernel(kern, dim3(static_cast<unsigned>(plan.grid)), dim3(kWriteThreads), 0, static_cast<cudaStream_t>(stream), c,
                              static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), token_stride, head_stride, table,
                              table_stride, start, first, n_seq, tokens, max_tokens, spans_of(std::min(max_tokens, tokens)), err));
  count_launch();
  RT_CHECK_CUDA(cudaGetLastError());
  return RT_OK;
}

extern "C" rt_status rt_kv_cache_read(const rt_kv_cache* cache, void* out_k, void* out_v, const int32_t* table, int table_stride,
                                      const int32_t* start, const int32_t* first, int n_seq, int tokens, int max_tokens, int dtype,
                                      void* stream) {
  KvView c;
  Plan plan;
  RT_TRY(check_kv_cache("kv_cache_read", cache, &c));
  max_tokens += max_tokens == 0;
  RT_TRY(check_ragged("kv_cache_read", table, table_stride, start, first, n_seq, tokens, max_tokens, c.heads, dtype, &plan));
  if (plan.grid == 0) return RT_OK;
  RT_REQUIRE(out_k && out_v, RT_ERR_INVALID, "kv_cache_read: null pointer");
  RT_REQUIRE(((reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) & 15u) == 0, RT_ERR_INVALID,
             "kv_cache_read: outputs must be 16-byte aligned");
  int* err = device_error_word();
  RT_REQUIRE(err != nullptr, RT_ERR_CUDA, "kv_cache_read: cannot allocate the device error word");
  auto kern = choose(dtype == RT_BF16, cache->format == RT_KV_INT8, plan.listed, [](auto bf16, auto int8, auto listed) {
    return kv_read_kernel<decltype(bf16)::value, decltype(int8)::value, decltype(listed)::value>;
  });
  RT_CHECK_CUDA(launch_kernel(kern, dim3(static_cast<unsigned>(plan.grid)), dim3(kWriteThreads), 0, static_cast<cudaStream_t>(stream), c,
                              static_cast<uint16_t*>(out_k), static_cast<uint16_t*>(out_v), table, table_stride, start, first, n_seq,
                              tokens, max_tokens, spans_of(std::min(max_tokens, tokens)), err));
  count_launch();
  RT_CHECK_CUDA(cudaGetLastError());
  return RT_OK;
}
