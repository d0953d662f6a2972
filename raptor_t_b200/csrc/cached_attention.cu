// Attention of few query rows over the 8-bit key/value cache (layout: kv_cache.cuh): single tokens of running answers, short
// questions.
//
// The rows of one sequence that share a key head (token x query heads of the group) form tiles of 16.  A warp takes every n-th
// 64-token block of the tile's sequence and keeps the tile's running maximum, sum and output for its blocks alone; the
// warps of a CTA, and the CTAs of a cluster through distributed shared memory, are joined at the end:
//   out = sum_w O_w 2^(m_w - M) / sum_w l_w 2^(m_w - M),  M = max_w m_w.
// Splitting the keys and not the rows is what fills the chip with a handful of rows, and one launch does it.
//
// A warp's blocks come by bulk copies of 4 KB into a ring of its own, two blocks ahead, so that HBM sees 192 KB of requests per SM
// and no register waits for them.  The products run on mma.sync (m16n8k16, 16-bit operands, fp32 sums): the work is the bytes of the cache, and a 16-row tile costs
// about a fifth of the tensor pipe at the rate HBM delivers codes.  Codes become halves exactly (kv_cache.cuh), a block's
// scale multiplies its scores and its output in fp32.  Codes go from shared memory straight into the operand registers:
// the order of the 64 dimensions inside Q K^T and of the keys and dimensions inside P V is free, so it is chosen such that a thread's
// operands are 16 consecutive bytes of a key and 8 of a value.
// bf16 queries are turned into halves scaled by a power of two per row (largest entry in [2^14, 2^15)): exact but for
// entries 2^-28 below the row's largest.  Probabilities are rounded to halves (2^-11 relative) for the second product; their
// sum is taken in fp32 before.
#include "cached_attention.h"

#include <algorithm>

#include "device_error.h"
#include "launch.h"
#include "launch_count.h"
#include "sm100_ptx.cuh"

namespace rt {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxSplits = 16;
constexpr int kFewRows = 64;  // rows of a sequence and key head up to which this kernel is taken

using Args = CachedAttentionArgs;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 dimensions [16 t, 16 t + 16) of one query row as eight half2, and the power of two that they were multiplied with.
template <bool BF16>
__device__ __forceinline__ float load_query(const uint16_t* row, int t, uint32_t* h) {
  uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (row) {
    w[0] = __ldg(reinterpret_cast<const uint4*>(row + 16 * t));
    w[1] = __ldg(reinterpret_cast<const uint4*>(row + 16 * t + 8));
  }
  const uint32_t* p = reinterpret_cast<const uint32_t*>(w);
  if constexpr (!BF16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = p[i];
    return 1.f;
  } else {
    uint32_t most = 0;  // bits of the largest magnitude: integers order as the magnitudes do
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, max((p[i] << 16) & 0x7fffffffu, p[i] & 0x7fff0000u));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int up = kv::query_shift(most);
    const float f = kv::pow2(up);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = kv::unpack16<true>(p[i]);
      h[i] = kv::pack16<false>(x.x * f, x.y * f);
    }
    return kv::pow2(-up);
  }
}

constexpr int kStages = 2;
struct Smem {
  uint8_t ring[kWarps][kStages][2][4096];  // keys, values; afterwards the first 4 KB of a warp's ring are its output, fp32 [16][64]
  float sum[16][64];                       // of the CTA
  float2 sum_ml[16];
  float2 ml[kWarps][16];
  uint64_t full[kWarps][kStages];
  int abort_flag;
};
static_assert(3 * (sizeof(Smem) + 1024) <= 228 * 1024, "three CTAs share an SM");

// Contiguous copy global -> shared (16-byte aligned), completion on an mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ptx::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}

template <bool BF16, bool INT8>
__global__ void __launch_bounds__(kWarps * 32, 3) few_rows_kernel(const Args a) {
  using C = kv::Codes<INT8>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  RT_PDL_LAUNCH_DEPENDENTS();
  RT_PDL_WAIT();
  const int rank = blockIdx.x % a.splits;
  int rest = blockIdx.x / a.splits;
  const int tile = rest % a.tiles;
  rest /= a.tiles;
  const int head = rest % a.cache.heads, seq = rest / a.cache.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  const CachedRows seq_rows(a, seq);
  if (!seq_rows.ok) return;
  const int rows = seq_rows.rows, row0 = tile * 16;
  if (row0 >= rows) return;
  auto limit_of = [&](int row) { return row < rows ? seq_rows.limit(a, row) : 0; };  // keys that a row sees
  const int least = limit_of(row0), most = limit_of(min(row0 + 16, rows) - 1);
  const int lim0 = limit_of(row0 + g), lim1 = limit_of(row0 + g + 8);
  const bool two = row0 + 8 < rows;  // the tile's upper eight rows are in use

  uint32_t q[4][4];
  float unit0, unit1;
  {
    uint32_t lo[8], hi[8];
    unit0 = load_query<BF16>(row0 + g < rows ? seq_rows.query(a, head, row0 + g) : nullptr, t, lo);
    unit1 = load_query<BF16>(row0 + g + 8 < rows ? seq_rows.query(a, head, row0 + g + 8) : nullptr, t, hi);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      q[s][0] = lo[2 * s];
      q[s][1] = hi[2 * s];
      q[s][2] = lo[2 * s + 1];
      q[s][3] = hi[2 * s + 1];
    }
  }
  unit0 *= a.scale_log2 * C::kUnit;
  unit1 *= a.scale_log2 * C::kUnit;

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float o[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  const int n_blocks = (most + 63) / 64, step = a.splits * kWarps;
  const int32_t* table = a.table + static_cast<int64_t>(seq) * a.table_stride;
  const int b0 = rank * kWarps + warp;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kStages; ++s) ptx::mbar_init(&sm.full[w][s], 1);
    sm.abort_flag = 0;
    ptx::fence_barrier_init();
  }
  __syncthreads();
  ptx::AbortCtx ab{&sm.abort_flag, a.err};
  // A block on its way: its scales, negative where the table has no such block.
  float ks[kStages], vs[kStages];
  int page[kStages];  // of the blocks to be requested next
  auto look = [&](int s, int b) { page[s] = b < n_blocks ? __ldg(table + b) : -1; };
  auto request = [&](int s, int b) {
    if (b >= n_blocks) return;
    const bool bad = page[s] < 0 || page[s] >= a.cache.blocks;
    if (bad && lane == 0) kv::index_error(a.err, kSiteCachedAttention);
    const int64_t slot = static_cast<int64_t>(bad ? 0 : page[s]) * a.cache.heads + head;
    if (lane == 0) {
      ptx::mbar_arrive_expect_tx(&sm.full[warp][s], 8192);
      bulk_load(sm.ring[warp][s][0], a.cache.k + slot * 4096, 4096, &sm.full[warp][s]);
      bulk_load(sm.ring[warp][s][1], a.cache.v + slot * 4096, 4096, &sm.full[warp][s]);
    }
    ks[s] = bad ? -1.f : __ldg(a.cache.k_scale + slot);
    vs[s] = __ldg(a.cache.v_scale + slot);
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) look(s, b0 + s * step);
#pragma unroll
  for (int s = 0; s < kStages; ++s) request(s, b0 + s * step);
#pragma unroll
  for (int s = 0; s < kStages; ++s) look(s, b0 + (kStages + s) * step);

  // Thread (g, t) takes key row g ^ (t's lowest bit) of every eight, so that the rows that four threads read at once are even and odd:
  // rows are 64 bytes, banks repeat after 128.
  const int kg = g ^ ((g >> 1) & 1), odd = t & 1;
  bool ok = true;
  uint32_t phase = 0;
  for (int bb = b0; bb < n_blocks && ok; bb += kStages * step, phase ^= 1) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      const int b = bb + st * step;
      if (b >= n_blocks) break;
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&sm.full[warp][st], phase, ab, 330))) {
        // gives up: copies in flight land before the ring is used again
        const long long t0 = clock64();
        for (int s = 0; lane == 0 && s < kStages; ++s) {
          const bool next = s < st;  // the slot has been requested again
          if (bb + (next ? kStages + s : s) * step >= n_blocks) continue;
          while (!ptx::mbar_try_wait(&sm.full[warp][s], next ? phase ^ 1 : phase) && clock64() - t0 < ptx::kWaitCycles) {
          }
        }
        __syncwarp();
        ok = false;
        break;
      }
      const uint8_t* kp = sm.ring[warp][st][0];
      const uint8_t* vp = sm.ring[warp][st][1];
      const float k_scale = ks[st], v_scale = vs[st] * C::kUnit;
      uint4 kw[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) kw[j] = *reinterpret_cast<const uint4*>(kp + (8 * j + kg) * 64 + 16 * t);

      // scores; step s of the product covers dimensions 16 t + 4 s .. + 3 of every thread's share
      float sc[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
        const uint32_t w[4] = {kw[j].x, kw[j].y, kw[j].z, kw[j].w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t p = C::prepare(w[s]);
          mma16816(sc[j], q[s], C::template pair<0>(p), C::template pair<2>(p));
        }
      }
      const float u0 = unit0 * k_scale, u1 = unit1 * k_scale;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sc[j][0] *= u0;
        sc[j][1] *= u0;
        sc[j][2] *= u1;
        sc[j][3] *= u1;
      }
      if (b * 64 + 64 > least || k_scale < 0.f) {  // keys that some row of the tile does not see
        const int l0 = k_scale < 0.f ? 0 : lim0, l1 = k_scale < 0.f ? 0 : lim1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = b * 64 + 8 * j + 2 * t;
          if (key + odd >= l0) sc[j][0] = -INFINITY;
          if (key + 1 - odd >= l0) sc[j][1] = -INFINITY;
          if (key + odd >= l1) sc[j][2] = -INFINITY;
          if (key + 1 - odd >= l1) sc[j][3] = -INFINITY;
        }
      }
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x0 = fmaxf(x0, fmaxf(sc[j][0], sc[j][1]));
        x1 = fmaxf(x1, fmaxf(sc[j][2], sc[j][3]));
      }
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
      x0 = fmaxf(x0, m0);
      x1 = fmaxf(x1, m1);
      // a row that has seen nothing yet: every exponential below is 2^(-inf)
      const float r0 = x0 == -INFINITY ? 0.f : x0, r1 = x1 == -INFINITY ? 0.f : x1;
      const float c0 = ex2(m0 - r0), c1 = ex2(m1 - r1);
      m0 = x0;
      m1 = x1;
      l0 *= c0;
      l1 *= c1;
      uint32_t p[4][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e0 = ex2(sc[j][0] - r0), e1 = ex2(sc[j][1] - r0);
        l0 += e0 + e1;
        p[j >> 1][(j & 1) * 2] = kv::pack16<false>(e0, e1);
        p[j >> 1][(j & 1) * 2 + 1] = 0u;
      }
      if (two) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float e0 = ex2(sc[j][2] - r1), e1 = ex2(sc[j][3] - r1);
          l1 += e0 + e1;
          p[j >> 1][(j & 1) * 2 + 1] = kv::pack16<false>(e0, e1);
        }
      }
      uint2 vw[16];  // keys 16 s + 2 t, + 1, + 8, + 9 of every step s of 16 keys, dimensions 8 g .. 8 g + 7
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          vw[4 * s + i] = *reinterpret_cast<const uint2*>(vp + (16 * s + 2 * t + ((i & 1) ^ odd) + 4 * (i & 2)) * 64 + 8 * g);
      __syncwarp();  // the slot has been read
      request(st, b + kStages * step);
      look(st, b + 2 * kStages * step);
      // output: column c of 8-column tile j is dimension 8 c + j
      float acc[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint2* w = vw + 4 * s;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // dimensions 8 g + 4 half .. + 3
          const uint32_t ka = half ? w[0].y : w[0].x, kb = half ? w[1].y : w[1].x;
          const uint32_t kc = half ? w[2].y : w[2].x, kd = half ? w[3].y : w[3].x;
          const uint32_t ab0 = C::prepare(kv::prmt(ka, kb, 0x5140u)), ab1 = C::prepare(kv::prmt(ka, kb, 0x7362u));
          const uint32_t cd0 = C::prepare(kv::prmt(kc, kd, 0x5140u)), cd1 = C::prepare(kv::prmt(kc, kd, 0x7362u));
          mma16816(acc[4 * half], p[s], C::template pair<0>(ab0), C::template pair<0>(cd0));
          mma16816(acc[4 * half + 1], p[s], C::template pair<2>(ab0), C::template pair<2>(cd0));
          mma16816(acc[4 * half + 2], p[s], C::template pair<0>(ab1), C::template pair<0>(cd1));
          mma16816(acc[4 * half + 3], p[s], C::template pair<2>(ab1), C::template pair<2>(cd1));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j][0] = fmaf(acc[j][0], v_scale, o[j][0] * c0);
        o[j][1] = fmaf(acc[j][1], v_scale, o[j][1] * c0);
      }
      if (two) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j][2] = fmaf(acc[j][2], v_scale, o[j][2] * c1);
          o[j][3] = fmaf(acc[j][3], v_scale, o[j][3] * c1);
        }
      }
    }
  }
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

  // ---- the warps of the CTA.  Thread (g, t) holds dimensions 16 t .. 16 t + 15 of rows g and g + 8.
  auto out_of = [&](int w) { return reinterpret_cast<float(*)[64]>(sm.ring[w][0][0]); };
  if (t == 0) {
    sm.ml[warp][g] = make_float2(m0, l0);
    sm.ml[warp][g + 8] = make_float2(m1, l1);
  }
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      *reinterpret_cast<float4*>(&out_of(warp)[g][16 * t + 8 * c + j]) = make_float4(o[j][c], o[j + 1][c], o[j + 2][c], o[j + 3][c]);
      if (two)
        *reinterpret_cast<float4*>(&out_of(warp)[g + 8][16 * t + 8 * c + j]) =
            make_float4(o[j][2 + c], o[j + 1][2 + c], o[j + 2][2 + c], o[j + 3][2 + c]);
    }
  __syncthreads();
  auto store = [&](int r, int d, float4 v, float l) {
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // NaN stays
    uint2 w;
    w.x = kv::pack16<BF16>(v.x * inv, v.y * inv);
    w.y = kv::pack16<BF16>(v.z * inv, v.w * inv);
    *reinterpret_cast<uint2*>(seq_rows.output(a, head, row0 + r) + d) = w;
  };
  const int valid = min(16, rows - row0);
  for (int i = threadIdx.x; i < valid * 16; i += kWarps * 32) {
    const int r = i >> 4, d = (i & 15) * 4;
    float M = -INFINITY, L = 0.f;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.ml[w][r].x);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = sm.ml[w][r];
      const float f = ex2(ml.x - ref);
      const float4 x = *reinterpret_cast<const float4*>(&out_of(w)[r][d]);
      L = fmaf(ml.y, f, L);
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
      v.z = fmaf(x.z, f, v.z);
      v.w = fmaf(x.w, f, v.w);
    }
    if (a.splits == 1) {
      store(r, d, v, L);
    } else {
      *reinterpret_cast<float4*>(&sm.sum[r][d]) = v;
      if (d == 0) sm.sum_ml[r] = make_float2(M, L);
    }
  }
  if (a.splits == 1) return;
  // ---- the CTAs of the cluster: each finishes its share of the tile's quads of dimensions
  ptx::cluster_arrive();
  ptx::cluster_wait();
  for (int i = rank + a.splits * static_cast<int>(threadIdx.x); i < valid * 16; i += a.splits * kWarps * 32) {
    const int r = i >> 4, d = (i & 15) * 4;
    const uint32_t ml_at = ptx::smem_u32(&sm.sum_ml[r]), o_at = ptx::smem_u32(&sm.sum[r][d]);
    float M = -INFINITY, L = 0.f;
    float4 v = make_float4(0, 0, 0, 0);
    for (int w = 0; w < a.splits; ++w) M = fmaxf(M, kv::ld_cluster_f2(kv::peer_address(ml_at, w)).x);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll 4
    for (int w = 0; w < a.splits; ++w) {
      const float2 ml = kv::ld_cluster_f2(kv::peer_address(ml_at, w));
      const float4 x = kv::ld_cluster_f4(kv::peer_address(o_at, w));
      const float f = ex2(ml.x - ref);
      L = fmaf(ml.y, f, L);
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
      v.z = fmaf(x.z, f, v.z);
      v.w = fmaf(x.w, f, v.w);
    }
    store(r, d, v, L);
  }
  ptx::cluster_arrive();  // no CTA leaves while another one reads its shared memory
  ptx::cluster_wait();
}

rt_status launch_few_rows(const Args& a, bool bf16, bool int8, cudaStream_t st) {
  auto kern = bf16 ? (int8 ? few_rows_kernel<true, true> : few_rows_kernel<true, false>)
                   : (int8 ? few_rows_kernel<false, true> : few_rows_kernel<false, false>);
  const int64_t grid = static_cast<int64_t>(a.n_seq) * a.cache.heads * a.tiles * a.splits;
  RT_TRY(ensure_kernel_smem(reinterpret_cast<const void*>(kern), sizeof(Smem), true));
  if (a.splits > 8) RT_TRY(ensure_large_clusters(reinterpret_cast<const void*>(kern)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = sizeof(Smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.splits > 1 ? 2 : 1;
  RT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  count_launch();
  RT_CHECK_CUDA(cudaGetLastError());
  return RT_OK;
}

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" rt_status rt_cached_attention(void* out, const void* q, int64_t q_stride, const rt_kv_cache* cache, const int32_t* table,
                                         int table_stride, const int32_t* context, const int32_t* first, int n_seq, int tokens,
                                         int max_q, int max_context, int heads, float scale, int causal, int dtype, void* stream) {
  Args a{};
  RT_TRY(check_kv_cache("cached_attention", cache, &a.cache));
  RT_REQUIRE(table && context && first, RT_ERR_INVALID, "cached_attention: null pointer");
  RT_REQUIRE(dtype == RT_F16 || dtype == RT_BF16, RT_ERR_INVALID, "cached_attention: unknown dtype %d", dtype);
  RT_REQUIRE(n_seq >= 0 && tokens >= 0 && table_stride > 0 && max_q >= 0 && max_context >= 0 && heads > 0, RT_ERR_INVALID,
             "cached_attention: bad sizes");
  RT_REQUIRE(heads % a.cache.heads == 0 && heads <= 4096, RT_ERR_UNSUPPORTED,
             "cached_attention: %d query heads over %d key heads (a multiple, at most 4096)", heads, a.cache.heads);
  if (n_seq == 0 || tokens == 0 || max_q == 0) return RT_OK;
  RT_REQUIRE(out && q, RT_ERR_INVALID, "cached_attention: null pointer");
  RT_REQUIRE(((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0 && q_stride % 8 == 0 && q_stride >= 0,
             RT_ERR_INVALID, "cached_attention: queries and output must be 16-byte aligned, the query stride a multiple of 8 values");
  max_q = std::min(max_q, tokens);
  a.out = static_cast<uint16_t*>(out);
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride;
  a.table = table;
  a.table_stride = table_stride;
  a.context = context;
  a.first = first;
  a.n_seq = n_seq;
  a.tokens = tokens;
  a.max_q = max_q;
  a.heads = heads;
  a.group = heads / a.cache.heads;
  RT_REQUIRE(static_cast<int64_t>(max_q) * a.group < (int64_t{1} << 30), RT_ERR_UNSUPPORTED, "cached_attention: too many query rows");
  const int rows = max_q * a.group;
  const bool many = rows > kFewRows;
  a.tiles = many ? (rows + 255) / 256 : (rows + 15) / 16;
  const int64_t heads_of_all = static_cast<int64_t>(n_seq) * a.cache.heads;  // under 2^41
  RT_REQUIRE(heads_of_all < (int64_t{1} << 28) && heads_of_all * a.tiles < (int64_t{1} << 28), RT_ERR_UNSUPPORTED,
             "cached_attention: %d sequences of up to %d query tokens are too many for one call", n_seq, max_q);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  a.err = device_error_word();
  RT_REQUIRE(a.err != nullptr, RT_ERR_CUDA, "cached_attention: cannot allocate the device error word");
  const int64_t widest = static_cast<int64_t>(table_stride) * 64;
  const int64_t keys = max_context > 0 ? std::min<int64_t>(max_context, widest) : widest;
  a.splits = 1;
  if (many) {
    // tiles of up to 256 rows see very different numbers of keys under the causal rule: four CTAs per SM over the call balance them
    while (a.splits < 8 && heads_of_all * a.tiles * a.splits < 4 * 148 && keys > 512 * a.splits) a.splits *= 2;
  } else {
    // 16 blocks a CTA, four a warp; fewer, down to one a warp, until the chip is full
    while (a.splits < kMaxSplits && (keys > 1024 * a.splits || (heads_of_all * a.tiles * a.splits < 4 * 148 && keys > 256 * a.splits)))
      a.splits *= 2;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == RT_BF16, int8 = cache->format == RT_KV_INT8;
  return many ? launch_cached_attention_many_rows(a, bf16, int8, st) : launch_few_rows(a, bf16, int8, st);
}
