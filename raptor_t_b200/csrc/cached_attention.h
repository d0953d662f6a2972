// Arguments of the kernels behind rt_cached_attention (cached_attention.cu: few query rows, cached_attention_sm100.cu: many).
#pragma once
#include <limits.h>

#include "device_error.h"
#include "kv_cache.cuh"

namespace rt {

struct CachedAttentionArgs {
  uint16_t* out;
  const uint16_t* q;
  int64_t q_stride;
  KvView cache;
  const int32_t* table;
  int table_stride;
  const int32_t* context;
  const int32_t* first;
  int n_seq, tokens, max_q, heads, group;  // group: query heads of a key head
  int tile_rows, tiles;                    // rows of a tile, tiles of the longest sequence
  int splits;                              // CTAs of a cluster that share a tile's keys
  int sorted;                              // long sequences first
  int listed;                              // many rows: tiles by kv::find_place, at most `tiles` of a sequence otherwise
  float scale_log2;
  int causal;
  int* err;
};

// What one sequence of a call is: its query rows and how many keys each of them sees.
struct CachedRows {
  int f0, n, ctx, rows;
  bool ok;
  __device__ __forceinline__ CachedRows(const CachedAttentionArgs& a, int seq) {
    f0 = a.first[seq];
    const int f1 = a.first[seq + 1];
    ctx = a.context[seq];
    ok = f1 > f0;
    n = rows = 0;
    if (!ok) return;
    if (f0 < 0 || f1 > a.tokens || f1 - f0 > a.max_q || ctx < 0 || ctx > static_cast<int64_t>(a.table_stride) * 64) {
      kv::index_error(a.err, kSiteCachedAttention);
      ok = false;
      return;
    }
    n = f1 - f0;
    rows = n * a.group;
  }
  __device__ __forceinline__ int limit(const CachedAttentionArgs& a, int row) const {
    return a.causal ? max(0, ctx - n + row / a.group + 1) : ctx;
  }
  __device__ __forceinline__ const uint16_t* query(const CachedAttentionArgs& a, int head, int row) const {
    return a.q + (f0 + row / a.group) * a.q_stride + (head * a.group + row % a.group) * 64;
  }
  __device__ __forceinline__ uint16_t* output(const CachedAttentionArgs& a, int head, int row) const {
    return a.out + (static_cast<int64_t>(f0 + row / a.group) * a.heads + head * a.group + row % a.group) * 64;
  }
};

// The `place`-th largest of `n` costs (in keys; by whole blocks, equal ones in order of their index), n at most kRanked and at most the CTA's
// threads; key[] in shared memory, kRanked + 4 ints, 16-byte aligned.  All threads of the CTA call it; `mine` is the cost of the calling
// thread's index.  CTAs start in order of their index: with the longest work first the last ones to end are short.
constexpr int kRanked = 256;
__device__ __forceinline__ int index_by_cost(int* key, int n, int mine, int place) {
  const int tid = threadIdx.x;
  const int own = max(-1, min(mine >> 6, (1 << 23) - 1)) * kRanked + (kRanked - 1 - tid);  // no two are equal
  if (tid < n) key[tid] = own;
  if (tid < 4) key[n + tid] = INT_MIN;
  __syncthreads();
  int before = 0;
  if (tid < n) {
    for (int i = 0; i < n; i += 4) {
      const int4 k = *reinterpret_cast<const int4*>(key + i);
      before += k.x > own;
      before += k.y > own;
      before += k.z > own;
      before += k.w > own;
    }
  }
  __syncthreads();
  if (tid < n && before == place) key[0] = tid;
  __syncthreads();
  return key[0];
}

namespace kv {

// Codes as operands of the products, two codes a register, to be multiplied with kUnit after kBias has been taken off.
//   int8: the code with its sign bit flipped is an unsigned byte u = code + 128; the half with the bits u is the subnormal number
//     u 2^-24, so a byte move does it.  128 of each code is taken off the sums: 128 sum q is the same for every key, and 128 sum p
//     comes from the product that sums the probabilities anyway.  fp32 sums keep 2^-17 of a code that way.
//   e4m3: as everywhere (kv_cache.cuh).
template <bool INT8>
struct Operand : Codes<false> {};
template <>
struct Operand<true> {
  static constexpr float kUnit = 16777216.f, kBias = 128.f;
  static __device__ __forceinline__ uint32_t prepare(uint32_t w) { return w ^ 0x80808080u; }
  template <int LO>
  static __device__ __forceinline__ uint32_t pair(uint32_t w) { return prmt(w, 0u, LO == 0 ? 0x4140u : 0x4342u); }
};

// 2^up that brings a row's largest magnitude (its bf16 or fp32 bits, sign removed) into [2^14, 2^15), so that the row can be
// held in halves; infinities and NaN pass as they are.
__device__ __forceinline__ int query_shift(uint32_t most) {
  const int e = static_cast<int>(most >> 23);  // biased exponent
  return e == 255 ? 0 : max(-126, min(126, 127 + 14 - e));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st_cluster_f4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void st_cluster_f2(uint32_t addr, const float2& v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
// The address of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

}  // namespace kv

// Tiles that the kernel of many rows has a place for.
inline int64_t many_rows_items(const CachedAttentionArgs& a) {
  return a.listed ? (static_cast<int64_t>(a.tokens) * a.group >> 8) + a.n_seq : static_cast<int64_t>(a.n_seq) * a.tiles;
}
rt_status launch_cached_attention_many_rows(const CachedAttentionArgs& a, bool bf16, bool int8, cudaStream_t st);

}  // namespace rt
