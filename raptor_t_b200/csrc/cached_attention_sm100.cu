// Attention of many query rows over the 8-bit key/value cache (layout: kv_cache.cuh) on tcgen05: whole questions and
// continuations.
//
// A CTA owns up to 256 rows (token x query head of the group) of one sequence and key head.  Its work is four streams of 128 rows that know
// nothing of one another until the end: two row tiles times even and odd blocks of 64 keys, or, where there are at most 128 rows, one row tile
// times every fourth block.  A stream's step is one block: scores, softmax, output, one after the other; the four streams fill each other's waits.
//
//   warps 0-15       softmax, four warps a stream: thread r owns row r (TMEM lane r).  Score row from TMEM, running maximum and sum in fp32
//                    (base-2 exponentials, every eighth pair on the FMA pipe), probabilities as halves into an operand tile of shared memory, output
//                    rescaled only when the maximum has grown by more than 2^8.  A row's scores are in registers at once, so the next block's are
//                    computed meanwhile.
//   warps 16-19      bring the codes: bulk copies of whole blocks a few blocks ahead into a ring, from there exact conversion to
//                    halves and stores into the 128-byte-swizzled operand tiles (keys K-major, values MN-major).  The block that two row
//                    tiles share is converted once.
//   warps 20-23      issue the MMAs, one warp a stream: the next block's S = Q K^T (M 128, N 64, K 64) as soon as this one's scores have been read, and
//                    O += P V when the probabilities are there.
// A block's key scale multiplies its scores.  Its value scale goes into the probabilities as an exponent, p' = 2^(score + log2 scale - R + 7), with
// R the row's own running maximum of score + log2 scale (raised when that has grown by more than 8): halves keep all their bits down to 2^-21 of
// what counts most in the row's output, whatever scales other rows see (2^7; p' <= 2^15).  The sum of the probabilities has a running maximum M of
// the scores as its reference and is taken from the same exponentials, times 2^(R - M - log2 scale - 7); out = O 2^(R - M - 7) / sum.
//
// No unit is full: the issue slots are 60 % used, the exponentials (16 a clock and SM) 49 %.  What bounds a stream is the chain of its step: scores, maximum,
// the wait for the product before, exponentials, store, fence, product; four streams overlap it as far as the registers of their softmax warps go.  0.86 us for
// 256 rows and a block of keys, 720 TFLOP/s of the chip, after 10 to 12 us for the start, the queries, the join and the end of a CTA.  256 rows x 64 blocks x 144
// heads, device time in a captured graph: 65.7 us (int8), 64.2 (e4m3).  Before: two streams of 128 keys a step, eight softmax warps an SM, 2.0 us for 256
// rows x 128 keys; probabilities over the scores' TMEM columns, which the next scores wait for,
// 77.8 us for the whole.
// Few tiles over many keys are split over the CTAs of a cluster; partial results, of streams and of CTAs, meet in (distributed) shared memory.
#include "cached_attention.h"

#include <algorithm>
#include <type_traits>

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

constexpr int kThreads = 768;
constexpr int kSoftmaxThreads = 512;
constexpr int kStreams = 4;
constexpr int kMaxSplits = 8;            // CTAs of a cluster
constexpr int kSms = 148;
constexpr int kStages = 4;               // operand tiles of keys, and of values: one for each warp that fills them
constexpr int kRaw = 4;                  // blocks of codes on their way, one for each of these warps
constexpr int kBlock = 4096;             // codes of a block's keys, or values
constexpr int kRing = 32;                // scales of a block, read after its operand slots are free again
constexpr int kTile = 64 * 128;          // 64 rows of 64 halves
constexpr int kTmemCols = 512;
constexpr int kColS = 0, kColO = 256;    // 4 x 64 scores, 4 x 64 outputs
constexpr float kRescaleThreshold = 8.0f;
constexpr int kPolyEvery = 8;            // pairs; 256 rows, 64 blocks: 73.4 us, with 4 78.6, 6 74.3, 16 76.2
constexpr float kShift = 7.0f;           // p' is 2^7 times larger than its share of the output
constexpr float kApart = 64.0f;          // p' of a block from which its sum is taken by itself
// 16 x 96 + 4 x 56 + 4 x 40 = 24 x 80 registers a lane, what the launch has
constexpr int kRegsSoftmax = 96, kRegsBring = 56, kRegsIssue = 40;

struct Smem {
  uint8_t q[2][2 * kTile];
  // afterwards k, v, raw and p hold partial results, [4 streams][128 rows][64] fp32
  uint8_t k[kStages][kTile];
  uint8_t v[kStages][kTile];
  uint8_t raw[kRaw][2 * kBlock];  // keys, values
  uint8_t p[kStreams][2 * kTile];  // probabilities
  uint64_t raw_k[kRaw], raw_v[kRaw];
  uint64_t q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[kStreams], s_free[kStreams], p_full[kStreams], o_full[kStreams];
  float2 scales[kRing];  // of a block: key scale, base-2 logarithm of the value scale; a negative key scale: nobody sees its keys
  float2 ml[kStreams][128];  // M and sum of a row
  float ref[kStreams][128];  // R
  float2 ml_cta[256];
  float ref_cta[256];
  alignas(16) int cost[kRanked + 4];
  uint32_t tmem_slot;
  int abort_flag;
  kv::Place place;
  int places;
};
static_assert(kStages * 2 * kTile + kRaw * 2 * kBlock + kStreams * 2 * kTile >= kStreams * 128 * 64 * 4, "partial results fit");
static_assert(sizeof(Smem) <= 227 * 1024, "one CTA per SM");

__device__ __forceinline__ void softmax_barrier() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// Contiguous copy global -> shared (16-byte aligned), completion on an mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 16 bytes of codes (16 dimensions of row `row`, chunk `c` of four) as 32 bytes of halves into a swizzled tile.
template <typename C>
__device__ __forceinline__ void put_codes(uint8_t* tile, int row, int c, const uint4& w) {
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

// Token and query head of the group of a row that goes up in equal steps: two divisions, not two for each row.
struct RowWalk {
  int token, member, tokens, members, group;
  __device__ __forceinline__ RowWalk(int row, int step, int group_size)
      : token(row / group_size), member(row % group_size), tokens(step / group_size), members(step % group_size), group(group_size) {}
  __device__ __forceinline__ void next() {
    token += tokens;
    member += members;
    if (member >= group) {
      member -= group;
      ++token;
    }
  }
};

template <bool BF16, bool INT8>
__global__ void __launch_bounds__(kThreads, 1) many_rows_kernel(const Args a) {
  using Keys = kv::Operand<INT8>;
  using Values = kv::Codes<INT8>;  // the sum of the rounded probabilities, which kv::Operand's values need, is not at hand here
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  RT_PDL_WAIT();
  RT_PDL_LAUNCH_DEPENDENTS();
  // ---- what this CTA works on; the same for all CTAs of a cluster but for the keys.  Tiles that see most start first.
  const int rank = blockIdx.x % a.splits;
  const int head = blockIdx.x / a.splits % a.cache.heads;
  int item = blockIdx.x / a.splits / a.cache.heads;  // (sequence, tile), the last tiles first
  kv::Place place{-1, 0};
  if (a.listed) {
    place = kv::find_place(item, a.first, a.n_seq, a.group, 8, 1, a.tokens, a.max_q, &sm.place, &sm.places, a.err, kSiteCachedAttention);
    if (place.seq < 0) return;
  } else if (a.sorted) {
    const int items = a.n_seq * a.tiles;
    int cost = -1;
    if (tid < items) {
      const int s = tid % a.n_seq, first_row = (a.tiles - 1 - tid / a.n_seq) * 256;
      const int rows = (a.first[s + 1] - a.first[s]) * a.group, last = min(first_row + 256, rows) - 1;
      if (last >= first_row) cost = a.causal ? a.context[s] - (rows - 1 - last) / a.group : a.context[s];
    }
    item = index_by_cost(sm.cost, items, cost, item);
  }
  const int seq = a.listed ? place.seq : item % a.n_seq;
  const CachedRows sr(a, seq);
  if (!sr.ok) return;
  const int tile = a.listed ? (sr.rows - 1) / 256 - place.nth : a.tiles - 1 - item / a.n_seq;
  const int row0 = tile * 256, here = min(256, sr.rows - row0);
  if (tile < 0 || here <= 0) return;
  const bool two = here > 128;  // two row tiles, each with two streams; otherwise one with four
  const int most = sr.limit(a, row0 + here - 1);
  const int all_blocks = (most + 63) / 64, each = (all_blocks + a.splits - 1) / a.splits;
  const int j0 = min(rank * each, all_blocks);
  const int n_blocks = min(j0 + each, all_blocks) - j0;
  // Stream x takes blocks first_of(x), + stride, ... below end_of(x): a first row tile may see less.
  const int stride = two ? 2 : 4;
  const int end0 = two ? min(n_blocks, max(0, (sr.limit(a, row0 + 127) + 63) / 64 - j0)) : n_blocks;
  auto first_of = [&](int x) { return two ? x & 1 : x; };
  auto end_of = [&](int x) { return two && x < 2 ? end0 : n_blocks; };

  if ((smem_u32(smem_raw) & 1023u) != 0) {  // the swizzled tiles need 1024-byte alignment
    if (tid == 0) atomicCAS(a.err, 0, 399);
    return;
  }
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) mbar_init(&sm.q_full[x], two ? 8 : 16);  // the warps of its streams
    for (int x = 0; x < kStreams; ++x) {
      mbar_init(&sm.s_full[x], 1);
      mbar_init(&sm.s_free[x], 4);
      mbar_init(&sm.p_full[x], 4);
      mbar_init(&sm.o_full[x], 1);
    }
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(&sm.raw_k[s], 1);
      mbar_init(&sm.raw_v[s], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], two ? 2 : 1);  // the streams that take the block
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_empty[s], two ? 2 : 1);
    }
    sm.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 20) {
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
  const int32_t* table = a.table + static_cast<int64_t>(seq) * a.table_stride + j0;

  if (warp >= 20) {
    // ---------------------------------------------------------------- MMA issuers
    reg_dealloc<kRegsIssue>();
    const int x = warp - 20;
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = make_idesc_f16(128, 64, 0, false), idesc_o = make_idesc_f16(128, 64, 0, true);
    const uint64_t dq = make_smem_desc_sw128(smem_u32(sm.q[two ? x >> 1 : 0]));
    const uint32_t d_s = tmem + kColS + x * 64, d_o = tmem + kColO + x * 64;
    const int end = end_of(x);
    const uint64_t dp = make_smem_desc_sw128(smem_u32(sm.p[x]));
    bool ok = true;
    uint32_t c = 0;  // steps so far
    auto round_of = [](int j) { return static_cast<uint32_t>(j / kStages) & 1; };
    auto scores = [&](int j) {
      const int s = j % kStages;
      tc_fence_after_sync();
      if (leader) {
        const uint64_t dk = make_smem_desc_sw128(smem_u32(sm.k[s]));
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_ss(d_s, dq + (k * 32 >> 4), dk + (k * 32 >> 4), idesc_s, k ? 1u : 0u);
        tc_commit(&sm.s_full[x]);
        tc_commit(&sm.k_empty[s]);
      }
      __syncwarp();
    };
    int j = first_of(x);
    if (j < end) {
      ok = wait(&sm.q_full[two ? x >> 1 : 0], 0, 310) && wait(&sm.k_full[j % kStages], round_of(j), 311);
      if (ok) scores(j);
    }
    for (; ok && j < end; j += stride, ++c) {
      const int next = j + stride, s = j % kStages;
      if (next < end) {  // as soon as the softmax warps have read this step's scores
        ok = wait(&sm.k_full[next % kStages], round_of(next), 316) && wait(&sm.s_free[x], c & 1, 315);
        if (!ok) break;
        scores(next);
      }
      ok = wait(&sm.v_full[s], round_of(j), 313) && wait(&sm.p_full[x], c & 1, 314);
      if (!ok) break;
      tc_fence_after_sync();
      if (leader) {
        const uint64_t dv = make_smem_desc_sw128(smem_u32(sm.v[s]));
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_ss(d_o, dp + (k * 32 >> 4), dv + (k * 2048 >> 4), idesc_o, c > 0 || k ? 1u : 0u);
        tc_commit(&sm.o_full[x]);
        tc_commit(&sm.v_empty[s]);
      }
      __syncwarp();
    }
    for (; ok && j < n_blocks; j += stride) {  // keys that this row tile does not see
      const int s = j % kStages;
      ok = wait(&sm.k_full[s], round_of(j), 320);
      if (leader && ok) mbar_arrive(&sm.k_empty[s]);
      ok = ok && wait(&sm.v_full[s], round_of(j), 312);
      if (leader && ok) mbar_arrive(&sm.v_empty[s]);
      __syncwarp();
    }
    __syncwarp();
    if (a.splits > 1) {
      cluster_arrive();
      cluster_wait();
      cluster_arrive();
      cluster_wait();
    }
  } else if (warp >= 16) {
    // ---------------------------------------------------------------- codes to operand tiles
    reg_dealloc<kRegsBring>();
    // Every fourth block a warp: a block is one chain of waits, copies and a fence, and four chains run side by side.  Lane 0 requests the
    // warp's blocks; their table entries were read a block earlier.
    const int own = warp - 16;
    // A slot that two warps filled in turn would need an order between them: one of them ahead by two rounds reads the parity of the
    // round before last as the last one's.
    static_assert(kRaw == 4 && kStages % 4 == 0, "a warp's blocks keep to its own slots");
    uint8_t* raw = sm.raw[own];
    int64_t slot_k = 0, slot_v = 0;  // of the blocks whose keys and values are requested next
    auto find = [&](int page, int j) {
      const bool there = page >= 0 && page < a.cache.blocks;
      const int64_t slot = static_cast<int64_t>(there ? page : 0) * a.cache.heads + head;
      const float ks = there ? a.cache.k_scale[slot] : -1.f, vs = a.cache.v_scale[slot];
      const bool bad = ks < 0.f || vs < 0.f;
      if (bad) kv::index_error(a.err, kSiteCachedAttention);
      sm.scales[j % kRing] = make_float2(bad ? -1.f : ks, __log2f(vs));
      return slot;
    };
    auto request = [&](uint8_t* dst, const uint8_t* base, int64_t slot, uint64_t* bar) {
      mbar_arrive_expect_tx(bar, kBlock);
      bulk_load(dst, base + slot * kBlock, kBlock, bar);
    };
    int page = 0;
    if (lane == 0 && own < n_blocks) {
      slot_k = slot_v = find(__ldg(table + own), own);
      request(raw, a.cache.k, slot_k, &sm.raw_k[own]);
      request(raw + kBlock, a.cache.v, slot_v, &sm.raw_v[own]);
      if (own + 4 < n_blocks) page = __ldg(table + own + 4);
    }
    // 256 chunks of 16 codes, eight a lane; rows from `rows` on hold no token: zeros, so that no code NaN meets a probability of 0
    auto convert = [&](auto codes, uint8_t* dst, const uint8_t* src, int rows) {
      const uint4* w = reinterpret_cast<const uint4*>(src) + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 in[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) in[i] = w[128 * h + 32 * i];
        if (rows < 64) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (32 * h + 8 * i + (lane >> 2) >= rows) in[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) put_codes<decltype(codes)>(dst, 32 * h + 8 * i + (lane >> 2), lane & 3, in[i]);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    // The keys go a block ahead of the values: a slot of keys is free once the scores are there, a slot of values a step later.
    uint32_t nk = 0, nv = 0;  // blocks done
    auto keys = [&](int j) {
      const int s = j % kStages;
      if (!wait(&sm.raw_k[own], nk & 1, 322) || !wait(&sm.k_empty[s], ((j / kStages) & 1) ^ 1, 317)) return false;
      convert(Keys(), sm.k[s], raw, 64);
      ++nk;
      if (lane == 0) {
        mbar_arrive(&sm.k_full[s]);
        if (j + 4 < n_blocks) {
          slot_k = find(page, j + 4);
          request(raw, a.cache.k, slot_k, &sm.raw_k[own]);
          if (j + 8 < n_blocks) page = __ldg(table + j + 8);
        }
      }
      __syncwarp();
      return true;
    };
    auto values = [&](int j) {
      const int s = j % kStages;
      if (!wait(&sm.raw_v[own], nv & 1, 324) || !wait(&sm.v_empty[s], ((j / kStages) & 1) ^ 1, 318)) return false;
      convert(Values(), sm.v[s], raw + kBlock, INT8 ? 64 : sm.scales[j % kRing].x < 0.f ? 0 : sr.ctx - (j0 + j) * 64);
      ++nv;
      if (lane == 0) {
        mbar_arrive(&sm.v_full[s]);
        if (j + 4 < n_blocks) request(raw + kBlock, a.cache.v, slot_v, &sm.raw_v[own]);
      }
      __syncwarp();
      return true;
    };
    bool ok = own >= n_blocks || keys(own);
    for (int j = own; ok && j < n_blocks; j += 4) {
      slot_v = slot_k;  // of block j + 4, if there is one
      ok = (j + 4 >= n_blocks || keys(j + 4)) && values(j);
    }
    if (lane == 0 && !ok) {  // gave up: copies in flight land before the CTA ends
      const long long t0 = clock64();
      auto land = [&](uint64_t* bar, uint32_t parity) {
        while (!mbar_try_wait(bar, parity) && clock64() - t0 < kWaitCycles) {
        }
      };
      const uint32_t blocks = (n_blocks - own + 3) / 4;  // of this warp; the next one's copies have been requested
      if (nk < blocks) land(&sm.raw_k[own], nk & 1);
      if (nv < blocks) land(&sm.raw_v[own], nv & 1);
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
    // With 64 rows or less the operand tile holds them twice or four times, and each stream has the softmax of another copy: a warp reaches
    // the TMEM lanes of its own scheduler only, and with one copy the same scheduler would do all streams' rows (12 x 4096 keys, 12 heads,
    // 64 rows: 57 us, now 38.5).
    const int x = warp >> 2, r = tid & 127, span = here > 64 ? 128 : here > 32 ? 64 : 32, own_r = r & (span - 1);
    const bool owner = two || r / span == x * 32 / span;
    const int row = row0 + (two ? (x >> 1) * 128 : 0) + own_r;
    const int row_c = min(row, row0 + here - 1);  // rows behind the last one are 0 and are not stored
    const int lim = sr.limit(a, row_c) - j0 * 64;   // keys that it sees, from this CTA's first on
    const bool live = owner && row - lane < row0 + here;  // the warp has a row
    const int wmin = __reduce_min_sync(0xffffffffu, lim), wmax = __reduce_max_sync(0xffffffffu, lim);
    // ---- the query rows, as halves.  Eight lanes a row, so that a load covers whole lines (a row a lane took 4 us).  The streams of a row tile share
    // its operand tile; each brings its part of the rows and leaves a row's unit and bias for the others.
    float2* found = sm.ml_cta + (two ? (x >> 1) * 128 : 0);
    {
      // a negative scale turns the scores around, and with it the queries; with a scale of 0 they are 0
      const float sign = a.scale_log2 > 0.f ? 1.f : a.scale_log2 < 0.f ? -1.f : 0.f;
      const float size = sign == 0.f ? 1.f : fabsf(a.scale_log2);
      const int chunk = lane & 7, parts = two ? 2 : 4, steps = 8 / parts, from = 4 * first_of(x) + (lane >> 3);
      const int left = row0 + here - (row - lane + from);  // rows from this lane's first one on
      RowWalk at(row - lane + from, 4 * parts, a.group);
      uint4 t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        t[i] = make_uint4(0, 0, 0, 0);
        if (i < steps && 4 * parts * i < left)
          t[i] = __ldg(reinterpret_cast<const uint4*>(a.q + (sr.f0 + at.token) * a.q_stride + (head * a.group + at.member) * 64) + chunk);
        at.next();
      }
      uint8_t* tile_q = sm.q[two ? x >> 1 : 0];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= steps) break;
        const uint32_t w[4] = {t[i].x, t[i].y, t[i].z, t[i].w};
        int up = 0;
        if constexpr (BF16) {
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max((w[k] << 16) & 0x7fffffffu, w[k] & 0x7fff0000u));
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          up = kv::query_shift(top);
        }
        const float f = kv::pow2(up) * sign;
        uint32_t h[4];
        float sum = 0.f;  // the keys' bias times the sum of the row, as the product sees it
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = kv::unpack16<BF16>(w[k]);
          h[k] = kv::pack16<false>(v.x * f, v.y * f);
          if constexpr (INT8) {
            const float2 y = kv::unpack16<false>(h[k]);
            sum += y.x + y.y;
          }
        }
        if constexpr (INT8) {
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        const int rr = (warp & 3) * 32 + 4 * parts * i + from;
        *reinterpret_cast<uint4*>(tile_q + rr * 128 + ((chunk ^ (rr & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        if (chunk == 0) found[rr] = make_float2(kv::pow2(-up) * size * Keys::kUnit, sum * (Keys::kBias / Keys::kUnit));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full[two ? x >> 1 : 0]);
    }
    softmax_barrier();
    const float unit = found[r].x, bias = found[r].y;  // a score in base 2 is (product - bias) * unit * key scale

    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + kColS + x * 64, to = tmem + lanes + kColO + x * 64;
    uint8_t* p_row = sm.p[x] + r * 128;
    float m = -INFINITY, ref = 0.f, gap = 0.f, l = 0.f;  // M, R, R - M - 7, sum
    bool ok = true;
    uint32_t c = 0;
    const int end = end_of(x);
    for (int j = first_of(x); j < end; j += stride, ++c) {
      const int key0 = j * 64;
      ok = wait(&sm.s_full[x], c & 1, 319);
      if (!ok) break;
      tc_fence_after_sync();
      const float2 sc = sm.scales[j % kRing];
      const bool act = live && key0 < wmax && !(sc.x < 0.f);
      uint32_t s[64];
      tmem_ld32(ts, s);
      tmem_ld32(ts + 32, s + 32);
      tc_wait_ld();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.s_free[x]);  // the next block's scores may come
      if (act) {
        float c0 = max_nan(unit * sc.x, 1.17549435e-38f);  // at least the smallest normal number: -inf * 0 would be NaN
        float off = bias * c0, log_v = sc.y;
        if (key0 + 64 > wmin) {  // keys that some row of the warp does not see
          const int left = lim - key0;
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (i >= left) s[i] = 0xff800000u;
          if (left <= 0) {  // no key of the block: neither its scales nor the row's own query touch the row
            c0 = 1.f;
            off = log_v = 0.f;
          }
        }
        const float m_new = max64(s) * c0 - off, most = m_new + log_v;
        float alpha = 1.f;
        bool fixes = false, apart = false;
        const bool grown = !(m_new <= m + kRescaleThreshold), more = !(most <= ref + kRescaleThreshold);
        if (__any_sync(0xffffffffu, grown || more || gap - log_v > kApart)) {
          const bool none = m == -INFINITY;  // no output yet
          if (grown) {
            l *= none ? 0.f : ex2(m - m_new);
            m = m_new;
          }
          if (none || more) {
            // with value scales of 0 there is an output, but nothing in it: any other scale raises R
            const float to = m == -INFINITY ? 0.f : most == -INFINITY ? m - 1000.f : most;
            if (!none) alpha = ex2(ref - to);
            ref = to;
          }
          gap = m == -INFINITY ? 0.f : ref - m - kShift;
          // Where the block's values are that much smaller than what the row has seen, its probabilities still count in the sum: they are taken
          // relative to M, and what they do to the output, nothing, is written over them.
          apart = m != -INFINITY && gap - log_v > kApart;
          fixes = __any_sync(0xffffffffu, !none && more);
        }
        // the product of the step before is done: its probabilities may be written over, and the output tile is at rest
        if (c > 0) ok = wait(&sm.o_full[x], (c - 1) & 1, 321);
        if (!ok) break;
        if (fixes) {
          tc_fence_after_sync();
#pragma unroll 1
          for (int i = 0; i < 64; i += 16) {
            uint32_t o[16];
            tmem_ld16(to + i, o);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st16(to + i, o);
          }
          tc_wait_st();
          tc_fence_before_sync();
        }
        // half a row at a time: the registers hold 64 scores and 32 packed probabilities at once no more than barely
        // (not from `rel`, which may be rounded: what that does to the probabilities goes into sum and output alike)
        const float rel = apart ? m : ref - kShift - log_v, back = ex2(apart ? 0.f : gap - log_v);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[16];
          l = fmaf(exp_columns<false, 32, kPolyEvery, true>(s + 32 * h, p, c0, rel + off), back, l);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(p_row + (((4 * h + i) ^ (r & 7)) << 4)) = make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
        }
        if (apart) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(p_row + 16 * i) = make_uint4(0, 0, 0, 0);
        }
      } else {
        if (c > 0) ok = wait(&sm.o_full[x], (c - 1) & 1, 323);
        if (!ok) break;
        if (live || c == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(p_row + 16 * i) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.p_full[x]);
    }
    if (ok && c > 0) {
      ok = wait(&sm.o_full[x], (c - 1) & 1, 325);
      tc_fence_after_sync();
    }
    const bool any = ok && c > 0 && live;  // there is an output tile to read; the same for the whole warp
    softmax_barrier();  // all streams have seen their last block: operand tiles and ring are free
    // ---- the streams of a row tile: each finishes its share of the dimensions, and leaves the others' in shared memory for them
    auto part_of = [&](int stream) { return reinterpret_cast<float*>(sm.k) + (stream * 128 + own_r) * 64; };
    auto quad_at = [&](int quad) { return (quad ^ (own_r & 15)) << 2; };
    // of a partial result with reference x among results whose largest reference is `most`
    auto weight = [](float x, float most) { return x == -INFINITY ? 0.f : ex2(x - most); };
    // of the outputs with reference R; 2^(R - M) in two steps, since it may be as large as a value
    auto factor = [](float R, float M, float L) {
      const float half = ex2(0.5f * (R - M));
      return L == 0.f ? 0.f : Values::kUnit * 0.0078125f / L * half * half;  // 2^-kShift
    };
    auto join = [&](auto count) {
      constexpr int N = decltype(count)::value, D = 64 / N, Q = D / 4;  // streams, dimensions of a share, their quads
      const int y = first_of(x), x0 = x - y;
      auto load = [&](int share, uint32_t* o) {
        if (any) {
          if constexpr (D == 32) tmem_ld32(to + share * D, o);
          else tmem_ld16(to + share * D, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < D; ++k) o[k] = 0u;
        }
      };
      if (owner) {
        sm.ml[x][own_r] = make_float2(any ? m : -INFINITY, any ? l : 0.f);
        sm.ref[x][own_r] = any && m != -INFINITY ? ref : -INFINITY;
#pragma unroll
        for (int s = 1; s < N; ++s) {
          const int share = (y + s) % N;
          uint32_t o[D];
          load(share, o);
#pragma unroll
          for (int q = 0; q < Q; ++q)
            *reinterpret_cast<uint4*>(part_of(x) + quad_at(share * Q + q)) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
      }
      softmax_barrier();
      if (!owner) return;
      uint32_t o[D];
      load(y, o);
      float M = -INFINITY, R = -INFINITY, L = 0.f, f[N];
#pragma unroll
      for (int s = 0; s < N; ++s) {
        M = max_nan(M, sm.ml[x0 + s][own_r].x);
        R = max_nan(R, sm.ref[x0 + s][own_r]);
      }
#pragma unroll
      for (int s = 0; s < N; ++s) {
        const float2 ml = sm.ml[x0 + s][own_r];
        L = fmaf(ml.y, weight(ml.x, M), L);
        f[s] = weight(sm.ref[x0 + s][own_r], R);
      }
      const float w = a.splits > 1 ? 1.f : factor(R, M, L);
      float v[D];
      float own = 0.f;
#pragma unroll
      for (int s = 0; s < N; ++s) {
        f[s] *= w;
        if (s == y) own = f[s];
      }
#pragma unroll
      for (int k = 0; k < D; ++k) v[k] = __uint_as_float(o[k]) * own;
#pragma unroll
      for (int s = 0; s < N; ++s) {
        if (s == y) continue;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const float4 t = *reinterpret_cast<const float4*>(part_of(x0 + s) + quad_at(y * Q + q));
          v[4 * q] = fmaf(t.x, f[s], v[4 * q]);
          v[4 * q + 1] = fmaf(t.y, f[s], v[4 * q + 1]);
          v[4 * q + 2] = fmaf(t.z, f[s], v[4 * q + 2]);
          v[4 * q + 3] = fmaf(t.w, f[s], v[4 * q + 3]);
        }
      }
      if (a.splits > 1) {
        if (y == 0) {
          sm.ml_cta[(two ? (x >> 1) * 128 : 0) + own_r] = make_float2(M, L);
          sm.ref_cta[(two ? (x >> 1) * 128 : 0) + own_r] = R;
        }
#pragma unroll
        for (int q = 0; q < Q; ++q)  // over what this thread has read
          *reinterpret_cast<float4*>(part_of(x0) + quad_at(y * Q + q)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      } else {  // through the same places, so that a store covers whole sectors of few lines
        constexpr int C = D / 8;
#pragma unroll
        for (int q = 0; q < C; ++q)
          *reinterpret_cast<uint4*>(part_of(x0) + quad_at(y * Q + q)) = make_uint4(pack2<BF16>(v[8 * q], v[8 * q + 1]), pack2<BF16>(v[8 * q + 2], v[8 * q + 3]),
                                                                                 pack2<BF16>(v[8 * q + 4], v[8 * q + 5]), pack2<BF16>(v[8 * q + 6], v[8 * q + 7]));
        __syncwarp();
        const int from = lane / C, q = lane % C;
        RowWalk at(row - lane + from, 32 / C, a.group);
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int rr = own_r - lane + from + 32 / C * i;
          const uint4 t = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(sm.k) + (x0 * 128 + rr) * 64 + (((y * Q + q) ^ (rr & 15)) << 2));
          if (row - lane + from + 32 / C * i < row0 + here)
            reinterpret_cast<uint4*>(a.out + (static_cast<int64_t>(sr.f0 + at.token) * a.heads + head * a.group + at.member) * 64 + y * D)[q] = t;
          at.next();
        }
      }
    };
    if (two) join(std::integral_constant<int, 2>());
    else join(std::integral_constant<int, 4>());
    auto store = [&](const RowWalk& to, int d, const float4& v) {
      *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(sr.f0 + to.token) * a.heads + head * a.group + to.member) * 64 + d) =
          make_uint2(pack2<BF16>(v.x, v.y), pack2<BF16>(v.z, v.w));
    };
    // ... then the CTAs of the cluster, each of which finishes its share of the tile; all parts are requested before one is used
    if (a.splits > 1) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      RowWalk to(row0 + ((rank * kSoftmaxThreads + tid) >> 4), a.splits * kSoftmaxThreads / 16, a.group);
      for (int i = rank * kSoftmaxThreads + tid; i < here * 16; i += a.splits * kSoftmaxThreads, to.next()) {
        const int rr = i >> 4, quad = i & 15, x0 = two ? (rr >> 7) * 2 : 0, pr = rr & 127;
        const uint32_t ml_at = smem_u32(&sm.ml_cta[rr]), ref_at = smem_u32(&sm.ref_cta[rr]);
        const uint32_t o_at = smem_u32(reinterpret_cast<float*>(sm.k) + (x0 * 128 + pr) * 64 + ((quad ^ (pr & 15)) << 2));
        float2 ml[kMaxSplits];
        float ref[kMaxSplits];
        float4 o[kMaxSplits];
#pragma unroll
        for (int w = 0; w < kMaxSplits; ++w) {
          ml[w] = make_float2(-INFINITY, 0.f);
          ref[w] = -INFINITY;
          o[w] = make_float4(0, 0, 0, 0);
          if (w < a.splits) {
            ml[w] = kv::ld_cluster_f2(kv::peer_address(ml_at, w));
            ref[w] = kv::ld_cluster_f1(kv::peer_address(ref_at, w));
            o[w] = kv::ld_cluster_f4(kv::peer_address(o_at, w));
          }
        }
        float M = -INFINITY, R = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kMaxSplits; ++w) {
          M = max_nan(M, ml[w].x);
          R = max_nan(R, ref[w]);
        }
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kMaxSplits; ++w) {
          const float f = weight(ref[w], R);
          L = fmaf(ml[w].y, weight(ml[w].x, M), L);
          v.x = fmaf(o[w].x, f, v.x);
          v.y = fmaf(o[w].y, f, v.y);
          v.z = fmaf(o[w].z, f, v.z);
          v.w = fmaf(o[w].w, f, v.w);
        }
        const float w = factor(R, M, L);
        store(to, 4 * quad, make_float4(v.x * w, v.y * w, v.z * w, v.w * w));
      }
    }
    if (a.splits > 1) {
      __syncwarp();
      cluster_arrive();  // no CTA leaves while another one reads its shared memory
      cluster_wait();
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 20) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace

rt_status launch_cached_attention_many_rows(const Args& args, bool bf16, bool int8, cudaStream_t st) {
  Args a = args;
  // Longest tiles first where there are more CTAs than run at once, but not so many that the last round hardly counts or that ranking them, which
  // every CTA does for itself, costs more than it saves.  Sequences of 65 to 256 rows over 64 to 4096 keys, us in order and ranked: 200 with one key head
  // (200 CTAs) 70.6 and 54.9, 128 with four (512) 95.5 and 73.7, 200 with four (800) 137.7 and 113.3, 256 with four (1024) 157.4 and 152.4, 256 with
  // twelve 414 and 456; equal lengths lose 3 to 6 %.  Ranking 768 of them took 110 us of a call of 160.
  const int64_t items = many_rows_items(a), ctas = items * a.cache.heads * a.splits;
  RT_REQUIRE(ctas < (int64_t{1} << 31), RT_ERR_UNSUPPORTED, "cached_attention: %d sequences of up to %d query tokens are too many for one call", a.n_seq,
             a.max_q);
  a.sorted = !a.listed && items <= kRanked && ctas > kSms && ctas <= 6 * kSms;
  auto kern = bf16 ? (int8 ? many_rows_kernel<true, true> : many_rows_kernel<true, false>)
                   : (int8 ? many_rows_kernel<false, true> : many_rows_kernel<false, false>);
  RT_TRY(ensure_kernel_smem(reinterpret_cast<const void*>(kern), sizeof(Smem), true));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
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
