// Attention of many query rows over the 8-bit key/value cache (layout: kv_cache.cuh) on tcgen05: whole questions and
// continuations.
//
// A CTA owns up to 256 rows (token x query head of the group) of one sequence and key head, as two streams of 128: rows 0-127 and rows
// 128-255 over the same keys, or, where the tile has at most 128 rows, the same rows over the even and the odd steps.  A step is 128 keys
// (two blocks of the cache).  Two streams keep the exponential unit busy: one computes while the other loads, stores and waits.
//
//   warps 0-3, 4-7   softmax of stream 0, 1: thread r owns row r (TMEM lane r), as in attention_sm100.cu: score row from TMEM, running
//                    maximum and sum in fp32, 16-bit probabilities back to TMEM, output rescaled only when the maximum has grown by
//                    more than 2^8.
//   warps 8-11       bring the codes: bulk copies of whole blocks (4 KB) a few steps ahead into a ring, from there exact conversion to
//                    halves and stores into the 128-byte-swizzled operand tiles (keys K-major, values MN-major).  The tile that 256
//                    rows share is converted once.
//   warps 12-15      issue the MMAs: scores and outputs of stream 0, scores and outputs of stream 1.
// A block's key scale multiplies its scores.  Its value scale goes into the probabilities, relative to the largest one of the keys that the CTA
// visits: p' = p * scale / largest * 2^7 (2^7: halves keep all their bits down to p = 2^-21 of the row's maximum; p' <= 2^15).
//
// Bound by the exponentials (16 a clock and SM) and the softmax warps' issue slots.
// Few tiles over many keys are split over the CTAs of a cluster; partial results, of streams and of CTAs, meet in (distributed) shared memory.
#include "cached_attention.h"

#include <algorithm>

#include "device_error.h"
#include "launch.h"
#include "launch_count.h"
#include "sm100_ptx.cuh"
#include "softmax.cuh"

namespace rt {
namespace {

using namespace ptx;
using namespace softmax;
using Args = CachedAttentionArgs;

constexpr int kThreads = 512;
constexpr int kStages = 3;               // of keys, and of values
constexpr int kRaw = 4;                  // steps of codes on their way
constexpr int kBlock = 4096;             // codes of a block
constexpr int kRing = 16;                // scales of a step, read up to two steps after its keys' slot is free
constexpr int kHalfTile = 64 * 128;      // 64 rows of 64 halves
constexpr int kTile = 2 * kHalfTile;
constexpr int kTmemCols = 512;
constexpr int kColS = 0, kColO = 256, kColP = 384;  // 2 x 128 scores, 2 x 64 outputs, 2 x 64 packed probabilities
constexpr float kRescaleThreshold = 8.0f;
constexpr float kShift = 7.0f;           // p' is 2^7 times larger than p * scale / largest scale
// 8 x 200 + 4 x 72 + 4 x 40 = 16 x 128 registers a lane, what the launch has
constexpr int kRegsSoftmax = 200, kRegsBring = 72, kRegsIssue = 40;

struct Smem {
  uint8_t q[2][kTile];
  uint8_t k[kStages][kTile];
  uint8_t v[kStages][kTile];
  uint8_t raw[kRaw][4 * kBlock];  // keys of block 0, 1, values of block 0, 1; afterwards: partial results, [2][128 rows][64] fp32
  uint64_t raw_full[kRaw], raw_empty[kRaw];
  uint64_t q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2];
  float4 scales[kRing];  // {key scale of block 0, 1, value scale of block 0, 1}
  float2 ml[2][128];
  float vmax[8];
  uint32_t tmem_slot;
  int abort_flag;
};
static_assert(kRaw * 4 * kBlock >= 2 * 128 * 64 * 4, "partial results fit the ring of codes");
static_assert(sizeof(Smem) <= 227 * 1024, "one CTA per SM");

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void softmax_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Contiguous copy global -> shared (16-byte aligned), completion on an mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 16 bytes of codes (16 dimensions of row `row`, chunk `c` of four) as 32 bytes of halves into a swizzled tile.
template <bool INT8>
__device__ __forceinline__ void put_codes(uint8_t* tile, int row, int c, const uint4& w) {
  using C = kv::Codes<INT8>;
  const uint32_t in[4] = {w.x, w.y, w.z, w.w};
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p = C::prepare(in[i]);
    h[2 * i] = C::template pair<0>(p);
    h[2 * i + 1] = C::template pair<2>(p);
  }
  uint8_t* at = tile + row * 128;
  *reinterpret_cast<uint4*>(at + (((2 * c) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
  *reinterpret_cast<uint4*>(at + (((2 * c + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
}

template <bool BF16, bool INT8>
__global__ void __launch_bounds__(kThreads, 1) many_rows_kernel(const Args a) {
  using C = kv::Codes<INT8>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  RT_PDL_LAUNCH_DEPENDENTS();
  RT_PDL_WAIT();
  // ---- what this CTA works on; the same for all CTAs of a cluster but for the keys.  The last tiles, which see most
  // under the causal rule, start first.
  const int rank = blockIdx.x % a.splits;
  const int item = blockIdx.x / a.splits;
  const int per_tile = a.n_seq * a.cache.heads;
  const int tile = a.tiles - 1 - item / per_tile;
  const int head = item % per_tile % a.cache.heads, seq = item % per_tile / a.cache.heads;
  const CachedRows sr(a, seq);
  if (!sr.ok) return;
  const int row0 = tile * 256, here = min(256, sr.rows - row0);
  if (here <= 0) return;
  const bool two = here > 128;  // two row tiles; otherwise one whose steps the streams share
  const int most = sr.limit(a, row0 + here - 1);
  const int n_blocks = (most + 63) / 64;
  const int all_steps = (n_blocks + 1) / 2, each = (all_steps + a.splits - 1) / a.splits;
  const int j0 = min(rank * each, all_steps);
  const int n_steps = min(j0 + each, all_steps) - j0;
  // steps of stream x: the first steps_of(0) of a first row tile that sees less, or every second one
  const int steps0 = two ? min(n_steps, max(0, (sr.limit(a, row0 + 127) + 127) / 128 - j0)) : (n_steps + 1) / 2;
  auto steps_of = [&](int x) { return x == 0 ? steps0 : two ? n_steps : n_steps / 2; };
  auto uses = [&](int x, int j) { return two ? (x == 1 || j < steps0) : (j & 1) == x; };
  const bool combine = !two || a.splits > 1;

  if ((smem_u32(smem_raw) & 1023u) != 0) {  // the swizzled tiles need 1024-byte alignment
    if (tid == 0) atomicCAS(a.err, 0, 399);
    return;
  }
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sm.q_full[x], 4);
      mbar_init(&sm.s_full[x], 1);
      mbar_init(&sm.s_free[x], 4);
      mbar_init(&sm.p_full[x][0], 4);
      mbar_init(&sm.p_full[x][1], 4);
      mbar_init(&sm.pv_done[x], 1);
    }
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(&sm.raw_full[s], 1);
      mbar_init(&sm.raw_empty[s], 4);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.k_full[s], 4);
      mbar_init(&sm.k_empty[s], 2);  // both streams, whether they use the step or not
      mbar_init(&sm.v_full[s], 4);
      mbar_init(&sm.v_empty[s], 2);
    }
    sm.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(&sm.tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sm.tmem_slot;
  AbortCtx ab{&sm.abort_flag, a.err};
  // bounded, and the same answer for the whole warp
  auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, ab, site)) != 0;
  };
  const int32_t* table = a.table + static_cast<int64_t>(seq) * a.table_stride;
  const int64_t slots = static_cast<int64_t>(a.cache.heads);

  if (warp >= 12) {
    // ---------------------------------------------------------------- MMA issuers
    reg_dealloc<kRegsIssue>();
    const int x = (warp - 12) >> 1;
    const bool leader = elect_one();
    int c = 0;  // steps of this stream so far
    if (((warp - 12) & 1) == 0) {
      constexpr uint32_t idesc128 = make_idesc_f16(128, 128, 0, false), idesc64 = make_idesc_f16(128, 64, 0, false);
      const uint64_t dq = make_smem_desc_sw128(smem_u32(sm.q[x]));
      const uint32_t d = tmem + kColS + x * 128;
      if (steps_of(x) > 0 && wait(&sm.q_full[x], 0, 310)) {
        for (int j = 0; j < n_steps; ++j) {
          const int s = j % kStages;
          const bool mine = uses(x, j);
          if (mine && c > 0 && !wait(&sm.s_free[x], (c - 1) & 1, 311)) break;
          if (!wait(&sm.k_full[s], (j / kStages) & 1, 312)) break;
          if (mine) {
            tc_fence_after_sync();
            const uint64_t dk = make_smem_desc_sw128(smem_u32(sm.k[s]));
            if (leader) {
              const uint32_t idesc = 2 * (j0 + j) + 1 < n_blocks ? idesc128 : idesc64;
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_ss(d, dq + (k * 32 >> 4), dk + (k * 32 >> 4), idesc, k ? 1u : 0u);
              tc_commit(&sm.k_empty[s]);
              tc_commit(&sm.s_full[x]);
            }
            ++c;
          } else if (leader) {
            mbar_arrive(&sm.k_empty[s]);
          }
          __syncwarp();
        }
      } else if (steps_of(x) == 0) {
        for (int j = 0; j < n_steps; ++j) {
          if (!wait(&sm.k_full[j % kStages], (j / kStages) & 1, 313)) break;
          if (leader) mbar_arrive(&sm.k_empty[j % kStages]);
          __syncwarp();
        }
      }
    } else {
      constexpr uint32_t idesc = make_idesc_f16(128, 64, 0, true);
      const uint32_t d = tmem + kColO + x * 64, p = tmem + kColP + x * 64;
      for (int j = 0; j < n_steps; ++j) {
        const int s = j % kStages;
        if (!wait(&sm.v_full[s], (j / kStages) & 1, 314)) break;
        if (uses(x, j)) {
          const uint64_t dv = make_smem_desc_sw128(smem_u32(sm.v[s]));
          if (!wait(&sm.p_full[x][0], c & 1, 315)) break;
          tc_fence_after_sync();
          if (leader) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_ts(d, p + k * 8, dv + (k * 2048 >> 4), idesc, c > 0 || k ? 1u : 0u);
          }
          if (!wait(&sm.p_full[x][1], c & 1, 316)) break;
          tc_fence_after_sync();
          if (leader) {
            if (2 * (j0 + j) + 1 < n_blocks) {
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_ts(d, p + 32 + k * 8, dv + ((kHalfTile + k * 2048) >> 4), idesc, 1u);
            }
            tc_commit(&sm.v_empty[s]);
            tc_commit(&sm.pv_done[x]);
          }
          ++c;
        } else if (leader) {
          mbar_arrive(&sm.v_empty[s]);
        }
        __syncwarp();
      }
    }
    __syncwarp();
    if (a.splits > 1) {
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- codes to operand tiles
    reg_dealloc<kRegsBring>();
    const int p = tid - 256;
    auto page_of = [&](int b) { return b < n_blocks ? __ldg(table + b) : 0; };
    // the first code of a block, and its key scale: negative where the table has no such block, whose keys nobody sees then
    auto place_of = [&](int page, float* scale) {
      const bool bad = page < 0 || page >= a.cache.blocks;
      if (bad) kv::index_error(a.err, kSiteCachedAttention);
      const int64_t slot = (bad ? 0 : page) * slots + head;
      *scale = bad ? -1.f : a.cache.k_scale[slot];
      return slot;
    };
    // thread 0 requests step j: pages and scales were read a step earlier
    int pa = 0, pb = 0;
    auto look = [&](int j) {
      pa = page_of(2 * (j0 + j));
      pb = page_of(2 * (j0 + j) + 1);
    };
    auto request = [&](int j) {
      const int s = j % kRaw;
      const bool pair = 2 * (j0 + j) + 1 < n_blocks;
      float ka, kb;
      const int64_t sa = place_of(pa, &ka), sb = place_of(pb, &kb);
      const int64_t oa = sa * kBlock, ob = sb * kBlock;
      mbar_arrive_expect_tx(&sm.raw_full[s], pair ? 4 * kBlock : 2 * kBlock);
      bulk_load(sm.raw[s], a.cache.k + oa, kBlock, &sm.raw_full[s]);
      if (pair) bulk_load(sm.raw[s] + kBlock, a.cache.k + ob, kBlock, &sm.raw_full[s]);
      bulk_load(sm.raw[s] + 2 * kBlock, a.cache.v + oa, kBlock, &sm.raw_full[s]);
      if (pair) bulk_load(sm.raw[s] + 3 * kBlock, a.cache.v + ob, kBlock, &sm.raw_full[s]);
      sm.scales[j % kRing] = make_float4(ka, kb, a.cache.v_scale[sa], a.cache.v_scale[sb]);
    };
    // two of a block's 256 chunks of 16 codes a thread, of both blocks; a second block that a step does not have is what was there before
    auto convert = [&](uint8_t* dst, const uint8_t* src) {
      const uint4* w = reinterpret_cast<const uint4*>(src) + p;
      const uint4 w0 = w[0], w1 = w[128], w2 = w[256], w3 = w[384];
      put_codes<INT8>(dst, p >> 2, p & 3, w0);
      put_codes<INT8>(dst, (p >> 2) + 32, p & 3, w1);
      put_codes<INT8>(dst + kHalfTile, p >> 2, p & 3, w2);
      put_codes<INT8>(dst + kHalfTile, (p >> 2) + 32, p & 3, w3);
    };
    int asked = 0;
    if (p == 0) {
      for (; asked < min(kRaw, n_steps); ++asked) {
        look(asked);
        request(asked);
      }
      if (asked < n_steps) look(asked);
    }
    for (int j = 0; j < n_steps; ++j) {
      const int s = j % kStages, rs = j % kRaw;
      if (!wait(&sm.raw_full[rs], (j / kRaw) & 1, 322)) break;
      if (!wait(&sm.k_empty[s], ((j / kStages) & 1) ^ 1, 317)) break;
      convert(sm.k[s], sm.raw[rs]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.k_full[s]);
      if (!wait(&sm.v_empty[s], ((j / kStages) & 1) ^ 1, 318)) break;
      convert(sm.v[s], sm.raw[rs] + 2 * kBlock);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.v_full[s]);
        mbar_arrive(&sm.raw_empty[rs]);
      }
      if (j + kRaw < n_steps && warp == 8) {  // into the slot that this step has just left
        if (!wait(&sm.raw_empty[rs], (j / kRaw) & 1, 323)) break;
        if (p == 0) {
          request(asked++);
          if (asked < n_steps) look(asked);
        }
        __syncwarp();
      }
    }
    if (p == 0 && *ab.cta_flag) {  // gave up: copies in flight land before the CTA ends
      const long long t0 = clock64();
      for (int j = max(0, asked - kRaw); j < asked; ++j)
        while (!mbar_try_wait(&sm.raw_full[j % kRaw], (j / kRaw) & 1) && clock64() - t0 < kWaitCycles) {
        }
    }
    __syncwarp();
    if (a.splits > 1) {
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else {
    // ---------------------------------------------------------------- softmax
    reg_alloc<kRegsSoftmax>();
    const int x = warp >> 2, r = tid & 127;
    const int row = row0 + (two ? x * 128 : 0) + r;
    const int row_c = min(row, row0 + here - 1);  // rows behind the last one do as it does and are not stored
    const int lim = sr.limit(a, row_c);
    const bool live = row0 + (two ? x * 128 : 0) + (r & ~31) < row0 + here;  // the warp has a row
    const int wmin = __reduce_min_sync(0xffffffffu, lim), wmax = __reduce_max_sync(0xffffffffu, lim);
    const int steps = steps_of(x);
    // ---- the query row, as halves
    float unit;
    {
      const uint4* src = reinterpret_cast<const uint4*>(sr.query(a, head, row_c));
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 t = __ldg(src + i);
        w[4 * i] = t.x;
        w[4 * i + 1] = t.y;
        w[4 * i + 2] = t.z;
        w[4 * i + 3] = t.w;
      }
      // a negative scale turns the scores around, and with it the queries; with a scale of 0 they are 0
      const float sign = a.scale_log2 > 0.f ? 1.f : a.scale_log2 < 0.f ? -1.f : 0.f;
      int up = 0;
      if constexpr (BF16) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
        up = kv::query_shift(top);
      }
      const float f = kv::pow2(up) * sign;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 t = kv::unpack16<BF16>(w[i]);
        w[i] = kv::pack16<false>(t.x * f, t.y * f);
      }
      uint8_t* at = sm.q[x] + r * 128;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(at + ((i ^ (r & 7)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[x]);
      unit = kv::pow2(-up) * (sign == 0.f ? 1.f : fabsf(a.scale_log2)) * C::kUnit;
    }
    // ---- the largest value scale of the keys visited here
    float vref = 0.f;
    for (int b = 2 * j0 + tid; b < min(2 * (j0 + n_steps), n_blocks); b += 256) {
      const int page = table[b];
      if (page >= 0 && page < a.cache.blocks) vref = fmaxf(vref, a.cache.v_scale[page * slots + head]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) vref = fmaxf(vref, __shfl_xor_sync(0xffffffffu, vref, o));
    if (lane == 0) sm.vmax[warp] = vref;
    softmax_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) vref = fmaxf(vref, sm.vmax[i]);
    if (!(vref > 0.f)) vref = 1.f;
    const float inv_vref = 1.f / vref;

    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + kColS + x * 128, to = tmem + lanes + kColO + x * 64, tp = tmem + lanes + kColP + x * 64;
    float m_ref = -INFINITY, l = 0.f;
    bool pzero0 = false, pzero1 = false;
    bool ok = true;
    for (int c = 0; c < steps; ++c) {
      const int j = two ? c : 2 * c + x;
      const int key0 = (j0 + j) * 128;
      const bool pair = 2 * (j0 + j) + 1 < n_blocks;
      if (!wait(&sm.s_full[x], c & 1, 319)) { ok = false; break; }
      tc_fence_after_sync();
      const float4 sc = sm.scales[j % kRing];
      const bool act0 = live && key0 < wmax && sc.x >= 0.f, act1 = live && pair && key0 + 64 < wmax && sc.y >= 0.f;
      uint32_t s[128];
      tmem_ld32(ts, s);
      tmem_ld32(ts + 32, s + 32);
      tmem_ld32(ts + 64, s + 64);
      tmem_ld32(ts + 96, s + 96);
      tc_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.s_free[x]);

      if (key0 + 128 > wmin) {  // keys that some row of the warp does not see
        const int left = lim - key0;
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= left) s[i] = 0xff800000u;
      }
      // at least the smallest normal number: -inf * 0 would be NaN
      const float c0 = fmaxf(unit * sc.x, 1.17549435e-38f), c1 = fmaxf(unit * sc.y, 1.17549435e-38f);
      float alpha = 1.f;
      bool fix = false;
      if (act0 || act1) {
        float m_new = act0 ? max64(s) * c0 : -INFINITY;
        if (act1) m_new = fmaxf(m_new, max64(s + 64) * c1);
        if (m_ref == -INFINITY) {
          m_ref = m_new;
        } else if (m_new > m_ref + kRescaleThreshold) {
          alpha = ex2(m_ref - m_new);
          m_ref = m_new;
          fix = true;
        }
      }
      const float ref = m_ref == -INFINITY ? 0.f : m_ref;
      const float e0 = __log2f(fmaxf(sc.z * inv_vref, 8.7e-19f)) + kShift, e1 = __log2f(fmaxf(sc.w * inv_vref, 8.7e-19f)) + kShift;
      uint32_t p[32];
      l *= alpha;
      if (act0) l = fmaf(exp64<false>(s, p, c0, ref - e0), ex2(-e0), l);
      if (c > 0) {
        if (!wait(&sm.pv_done[x], (c - 1) & 1, 320)) { ok = false; break; }
        tc_fence_after_sync();
      }
      if (__any_sync(0xffffffffu, fix) && c > 0) {
#pragma unroll 1
        for (int i = 0; i < 64; i += 16) {
          uint32_t o[16];
          tmem_ld16(to + i, o);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tmem_st16(to + i, o);
        }
      }
      if (act0) {
        tmem_st32(tp, p);
        pzero0 = false;
      } else if (!pzero0) {
#pragma unroll
        for (int i = 0; i < 32; ++i) p[i] = 0u;
        tmem_st32(tp, p);
        pzero0 = true;
      }
      tc_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[x][0]);
      if (pair) {
        if (act1) {
          l = fmaf(exp64<false>(s + 64, p, c1, ref - e1), ex2(-e1), l);
          tmem_st32(tp + 32, p);
          pzero1 = false;
        } else if (!pzero1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) p[i] = 0u;
          tmem_st32(tp + 32, p);
          pzero1 = true;
        }
        tc_wait_st();
        tc_fence_before_sync();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&sm.p_full[x][1]);
    }
    ok = __all_sync(0xffffffffu, ok);
    if (ok && steps > 0) {
      ok = wait(&sm.pv_done[x], (steps - 1) & 1, 321);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after_sync();
    }
    const bool any = ok && steps > 0 && live;  // there is an output tile to read; the same for the whole warp
    const float unit_o = vref * C::kUnit * 0.0078125f;  // 2^-kShift
    if (!combine) {
      if (any) {  // warp-uniform: TMEM loads are for whole warps
        const float inv = lim > 0 ? unit_o / l : 0.f;
        uint16_t* dst = sr.output(a, head, row_c);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          tmem_ld32(to + 32 * h, o);
          tc_wait_ld();
          if (row < row0 + here) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float lo = __uint_as_float(o[8 * q + 2 * e]), hi = __uint_as_float(o[8 * q + 2 * e + 1]);
                w[e] = lim > 0 ? pack2<BF16>(lo * inv, hi * inv) : 0u;
              }
              *reinterpret_cast<uint4*>(dst + 32 * h + 8 * q) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      } else if (row < row0 + here) {  // no key at all
#pragma unroll
        for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(sr.output(a, head, row) + 8 * q) = make_uint4(0, 0, 0, 0);
      }
    } else {
      softmax_barrier();  // both streams have seen the last step: its codes have been converted, the ring is free
      float* part = reinterpret_cast<float*>(sm.raw) + x * 128 * 64 + r * 64;
      sm.ml[x][r] = make_float2(any && lim > 0 ? m_ref : -INFINITY, any && m_ref != -INFINITY ? l : 0.f);
      const bool keep = any;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t o[16];
        if (keep) {
          tmem_ld16(to + 16 * h, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0u;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 f = make_float4(__uint_as_float(o[4 * q]) * unit_o, __uint_as_float(o[4 * q + 1]) * unit_o,
                                       __uint_as_float(o[4 * q + 2]) * unit_o, __uint_as_float(o[4 * q + 3]) * unit_o);
          *reinterpret_cast<float4*>(part + (((4 * h + q) ^ (r & 15)) << 2)) = f;
        }
      }
      if (a.splits > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
      } else {
        softmax_barrier();
      }
      // a quarter of a row (16 dimensions) a thread, over all threads of the cluster
      for (int i = rank * 256 + tid; i < here * 4; i += a.splits * 256) {
        const int rr = i >> 2, quarter = i & 3;
        const int x0 = two ? rr >> 7 : 0, xs = two ? 1 : 2, pr = rr & 127;
        const uint32_t ml_at = smem_u32(&sm.ml[x0][pr]), o_at = smem_u32(reinterpret_cast<float*>(sm.raw) + (x0 * 128 + pr) * 64);
        float M = -INFINITY, L = 0.f;
        for (int w = 0; w < a.splits; ++w)
          for (int y = 0; y < xs; ++y) M = max_nan(M, kv::ld_cluster_f2(kv::peer_address(ml_at + y * 1024, w)).x);
        float acc[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[k] = 0.f;
        if (M != -INFINITY) {
          for (int w = 0; w < a.splits; ++w)
            for (int y = 0; y < xs; ++y) {
              const float2 ml = kv::ld_cluster_f2(kv::peer_address(ml_at + y * 1024, w));
              if (ml.x == -INFINITY) continue;
              const float f = ex2(ml.x - M);
              L = fmaf(ml.y, f, L);
              const uint32_t at = kv::peer_address(o_at + y * 32768, w);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float4 v = kv::ld_cluster_f4(at + (((4 * quarter + q) ^ (pr & 15)) << 4));
                acc[4 * q] = fmaf(v.x, f, acc[4 * q]);
                acc[4 * q + 1] = fmaf(v.y, f, acc[4 * q + 1]);
                acc[4 * q + 2] = fmaf(v.z, f, acc[4 * q + 2]);
                acc[4 * q + 3] = fmaf(v.w, f, acc[4 * q + 3]);
              }
            }
        }
        const float inv = M != -INFINITY ? 1.f / L : 0.f;
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = pack2<BF16>(acc[2 * k] * inv, acc[2 * k + 1] * inv);
        uint4* dst = reinterpret_cast<uint4*>(sr.output(a, head, row0 + rr) + 16 * quarter);
        dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
        dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
      if (a.splits > 1) {
        __syncwarp();
        cluster_arrive();  // no CTA leaves while another one reads its shared memory
        cluster_wait();
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace

rt_status launch_cached_attention_many_rows(const Args& a, bool bf16, bool int8, cudaStream_t st) {
  auto kern = bf16 ? (int8 ? many_rows_kernel<true, true> : many_rows_kernel<true, false>)
                   : (int8 ? many_rows_kernel<false, true> : many_rows_kernel<false, false>);
  RT_TRY(ensure_kernel_smem(reinterpret_cast<const void*>(kern), sizeof(Smem), true));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(a.n_seq) * a.cache.heads * a.tiles * a.splits));
  cfg.blockDim = dim3(kThreads);
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

}  // namespace rt
