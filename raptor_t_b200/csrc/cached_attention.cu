// Attention of few query rows over the 8-bit key/value cache (layout: kv_cache.cuh): single tokens of running answers, short
// questions.
//
// The rows of one sequence that share a key head (token x query heads of the group) form tiles of 8 or 16.  A warp works on one
// 64-token block of one tile at a time and keeps a running maximum, sum and output for the blocks it has seen; partial results are joined by
//   out = sum_w O_w 2^(m_w - M) / sum_w l_w 2^(m_w - M),  M = max_w m_w.
// Splitting the keys and not the rows is what fills the chip with a handful of rows: the warps of a CTA take every n-th block of a tile, and
// the CTAs of a cluster share it, too; results meet in (distributed) shared memory.  One launch.
//
// A warp's blocks come by bulk copies of 4 KB into a ring of its own, 12 KB ahead, so that HBM sees 192 KB of requests per SM
// and no register waits for them.  The products run on mma.sync (m16n8k16, 16-bit operands, fp32 sums): the work is the bytes of the cache.
// Codes become halves exactly, a block's scale multiplies its scores and its output in fp32.  Codes go from shared memory
// straight into the operand registers: the order of the 64 dimensions inside Q K^T and of the keys and dimensions inside P V is free, so it is chosen
// such that a thread's operands are 16 consecutive bytes of a key and 8 of a value.
// bf16 queries are turned into halves scaled by a power of two per row (largest entry in [2^14, 2^15)): exact but for
// entries 2^-28 below the row's largest.  Probabilities are rounded to halves (2^-11 relative) for the second product; their
// sum is that of the rounded ones, in fp32.
//
// Measured (int8, 12 heads): one token over 4,096 cached ones 6.6 us, of which 2 are a launch and the rest the chain context, block table, codes,
// products, join; 64 x 4096 tokens 78.6 us, 5.1 TB/s of codes; ragged calls lose the last CTAs' time.  From 16 rows on the warps' instructions count:
// 1.65 ns a tile of 16 rows and block of keys on the full chip.  Tiles of 32 rows (255 registers, two CTAs an SM) run slower: 16 x 4096 keys, 32 rows
// 53.4 us, 43.4 with two tiles of 16.
#include "cached_attention.h"

#include <algorithm>
#include <cmath>

#include "device_error.h"
#include "launch.h"
#include "launch_count.h"
#include "sm100_ptx.cuh"

namespace rt {
namespace {

using Args = CachedAttentionArgs;

constexpr int kWarps = 4;       // of a CTA
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 4 : 3; }  // as the registers allow
constexpr int kSlots = 3;       // pieces of 4 KB of a warp on their way
constexpr int kMaxSplits = 8;   // CTAs of a cluster
constexpr int kFewRows = 64;    // rows of a sequence and key head up to which these kernels are taken
constexpr int kBlock = 4096;    // bytes of a block's keys, or values
constexpr float kSlack = 8.f, kShift = 7.f;  // probabilities are at most 2^15

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Contiguous copy global -> shared (16-byte aligned), completion on an mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ptx::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}

// 8 x 8 halves: thread (g, t) gives row g, columns 2 t and 2 t + 1, and gets them of the transposed matrix.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// 16 dimensions [16 t, 16 t + 16) of one query row, times `sign`, as eight half2, and the power of two that they were multiplied with.
template <bool BF16>
__device__ __forceinline__ float load_query(const uint16_t* row, int t, float sign, uint32_t* h) {
  uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (row) {
    w[0] = __ldg(reinterpret_cast<const uint4*>(row + 16 * t));
    w[1] = __ldg(reinterpret_cast<const uint4*>(row + 16 * t + 8));
  }
  const uint32_t* p = reinterpret_cast<const uint32_t*>(w);
  int up = 0;
  if constexpr (BF16) {
    uint32_t most = 0;  // bits of the largest magnitude: integers order as the magnitudes do
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, max((p[i] << 16) & 0x7fffffffu, p[i] & 0x7fff0000u));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    up = kv::query_shift(most);
  }
  const float f = kv::pow2(up) * sign;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 x = kv::unpack16<BF16>(p[i]);
    h[i] = kv::pack16<false>(x.x * f, x.y * f);
  }
  return kv::pow2(-up);
}

// One warp's state for a tile of 8 NT rows.  The products are taken transposed, S^T = K Q^T and O^T = V^T P^T: keys and dimensions fill the
// 16-row side of m16n8k16, query rows the 8-column side, so a conversion serves all rows and nothing is computed for rows that a tile does
// not have.  Thread (g, t) = (lane / 4, lane % 4) has columns (rows of the tile) 8 n + 2 t, + 1.
template <bool BF16, bool INT8, int NT>
struct RowTile {
  using C = kv::Operand<INT8>;
  static constexpr int kRows = 8 * NT;
  int g, t;
  int ctx, least;         // keys of the sequence, and of those what the tile's first row sees
  int* err;
  int lim[NT][2];         // and what this thread's rows see
  uint32_t q[NT][4][2];
  float unit[NT][2], bias[NT][2];  // a score in base 2 is (product * unit - bias) * key scale
  float m[NT][2], l[NT][2];        // reference of the exponentials, sum of the rounded probabilities
  float o[NT][4][4];               // dimensions 8 g + 2 j (first two), 8 g + 2 j + 1 (last two)

  __device__ __forceinline__ void begin(const Args& a, const CachedRows& sr, int head, int row0) {
    ctx = sr.ctx;
    err = a.err;
    least = sr.limit(a, row0);
    // a negative scale turns the scores around, and with it the queries; with a scale of 0 they are 0
    const float sign = a.scale_log2 > 0.f ? 1.f : a.scale_log2 < 0.f ? -1.f : 0.f;
    const float size = (sign == 0.f ? 1.f : fabsf(a.scale_log2));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int mine = row0 + 8 * n + g;
      uint32_t h[8];
      const float back = load_query<BF16>(mine < sr.rows ? sr.query(a, head, mine) : nullptr, t, sign, h) * size;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      constexpr uint32_t kOnes[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        q[n][s][0] = h[2 * s];
        q[n][s][1] = h[2 * s + 1];
        if constexpr (INT8) mma16816(sum, kOnes, h[2 * s], h[2 * s + 1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + 8 * n + 2 * t + e;
        lim[n][e] = row < sr.rows ? sr.limit(a, row) : 0;
        const float u = __shfl_sync(0xffffffffu, back, (2 * t + e) * 4);  // of the thread that loaded the row
        unit[n][e] = u * C::kUnit;
        bias[n][e] = C::kBias * sum[e] * u;
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
    }
  }

  // Block b of the sequence; a negative scale: no such block, nobody sees its keys.  keys_read(): the keys' codes are in registers;
  // values(): where the values' codes are, once they are there; values_read(): they are in registers.
  // Key kk of every 16 is row kk with its lowest bit turned where bit 1 is set, so that the value rows that four threads read at once are
  // even and odd: rows are 64 bytes, banks repeat after 128.
  template <typename KeysRead, typename Values, typename ValuesRead>
  __device__ __forceinline__ bool block(const uint8_t* kp, float k_scale, float v_scale, int b, KeysRead keys_read, Values values,
                                        ValuesRead values_read) {
    const int kg = g ^ ((g >> 1) & 1), odd = t & 1;
    float sc[NT][4][4];  // of key tile i: keys g (first two), g + 8, of rows 2 t, 2 t + 1
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 lo = *reinterpret_cast<const uint4*>(kp + (16 * i + kg) * 64 + 16 * t);
      const uint4 hi = *reinterpret_cast<const uint4*>(kp + (16 * i + 8 + kg) * 64 + 16 * t);
      const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[n][i][0] = sc[n][i][1] = sc[n][i][2] = sc[n][i][3] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {  // dimensions 16 t + 4 s .. + 3 of every thread's share
        const uint32_t x = C::prepare(wl[s]), y = C::prepare(wh[s]);
        const uint32_t k[4] = {C::template pair<0>(x), C::template pair<0>(y), C::template pair<2>(x), C::template pair<2>(y)};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(sc[n][i], k, q[n][s][0], q[n][s][1]);
      }
    }
    __syncwarp();
    keys_read();
    const bool missing = k_scale < 0.f || v_scale < 0.f;
    const bool edge = b * 64 + 64 > least || missing;  // keys that some row of the tile does not see
    if (edge) {
      if (missing) {
        kv::index_error(err, kSiteCachedAttention);
        k_scale = v_scale = 0.f;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int e0 = missing ? 0 : lim[n][0], e1 = missing ? 0 : lim[n][1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = b * 64 + 16 * i + kg;
          if (key >= e0) sc[n][i][0] = -INFINITY;
          if (key >= e1) sc[n][i][1] = -INFINITY;
          if (key + 8 >= e0) sc[n][i][2] = -INFINITY;
          if (key + 8 >= e1) sc[n][i][3] = -INFINITY;
        }
      }
    }
    // The reference of a row follows its maximum when that has grown by more than 2^8.  A row that sees no key of the block is touched neither by
    // its scales nor by its own query, which may be no numbers.
    auto blind = [&](int n, int e) { return edge && b * 64 >= lim[n][e]; };
    float u[NT][2], c[NT][2];
    bool grown = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u[n][e] = fmaxf(unit[n][e] * k_scale, 1.17549435e-38f);  // at least the smallest normal number: -inf * 0 would be NaN
        c[n][e] = blind(n, e) ? 0.f : -bias[n][e] * k_scale;
        float x = fmaxf(fmaxf(sc[n][0][e], sc[n][0][e + 2]), fmaxf(sc[n][1][e], sc[n][1][e + 2]));
        x = fmaxf(x, fmaxf(fmaxf(sc[n][2][e], sc[n][2][e + 2]), fmaxf(sc[n][3][e], sc[n][3][e + 2])));
        grown |= fmaf(x, u[n][e], c[n][e]) > m[n][e] + kSlack;
      }
    float alpha[NT][2];
    const bool change = __any_sync(0xffffffffu, grown);
    if (change) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(fmaxf(sc[n][0][e], sc[n][0][e + 2]), fmaxf(sc[n][1][e], sc[n][1][e + 2]));
          x = fmaxf(x, fmaxf(fmaxf(sc[n][2][e], sc[n][2][e + 2]), fmaxf(sc[n][3][e], sc[n][3][e + 2])));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(m[n][e], fmaf(x, u[n][e], c[n][e]));
          alpha[n][e] = x == -INFINITY ? 1.f : ex2(m[n][e] - x);
          m[n][e] = x;
          l[n][e] *= alpha[n][e];
        }
    }
    // probabilities as halves, 2^7 times larger (halves keep all their bits down to 2^-21 of the reference), and turned into the operand P^T
    uint32_t p[NT][4][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // a row that has seen nothing yet: every exponential is 2^(-inf)
      const float c0 = c[n][0] - (m[n][0] == -INFINITY ? 0.f : m[n][0]) + kShift, c1 = c[n][1] - (m[n][1] == -INFINITY ? 0.f : m[n][1]) + kShift;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = ex2(fmaf(sc[n][i][0], u[n][0], c0)), e1 = ex2(fmaf(sc[n][i][1], u[n][1], c1));
        const float e2 = ex2(fmaf(sc[n][i][2], u[n][0], c0)), e3 = ex2(fmaf(sc[n][i][3], u[n][1], c1));
        p[n][i][0] = transpose8(kv::pack16<false>(e0, e1));
        p[n][i][1] = transpose8(kv::pack16<false>(e2, e3));
      }
    }
    // keys 2 t, + 1, + 8, + 9 of key tile i, dimensions 8 g .. 8 g + 7.  With 16 rows a tile they are read as they are needed: all at once
    // would not fit the registers.
    const int held = missing ? 0 : ctx;
    uint2 vw[NT == 1 ? 16 : 4];
    const uint8_t* vp = values();
    if (!vp) return false;
    auto load = [&](int i, uint2* w) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * i + 2 * t + ((e & 1) ^ odd) + 4 * (e & 2);
        w[e] = *reinterpret_cast<const uint2*>(vp + row * 64 + 8 * g);
        if (!INT8 && b * 64 + row >= held) w[e] = make_uint2(0, 0);  // places that hold no token may hold the code NaN
      }
    };
    if constexpr (NT == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) load(i, vw + 4 * i);
      __syncwarp();
      values_read();
    }
    float acc[NT][4][4], sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr uint32_t kOnes[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816(sum[n], kOnes, p[n][i][0], p[n][i][1]);
      if constexpr (NT > 1) load(i, vw);
      const uint2* w = NT == 1 ? vw + 4 * i : vw;
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // dimensions 8 g + 4 half .. + 3
        const uint32_t ka = half ? w[0].y : w[0].x, kb = half ? w[1].y : w[1].x;
        const uint32_t kc = half ? w[2].y : w[2].x, kd = half ? w[3].y : w[3].x;
        const uint32_t xa = C::prepare(ka), xb = C::prepare(kb), xc = C::prepare(kc), xd = C::prepare(kd);
        const uint32_t ab0 = kv::prmt(xa, xb, 0x5140u), ab1 = kv::prmt(xa, xb, 0x7362u);
        const uint32_t cd0 = kv::prmt(xc, xd, 0x5140u), cd1 = kv::prmt(xc, xd, 0x7362u);
        const uint32_t v0[4] = {C::template pair<0>(ab0), C::template pair<2>(ab0), C::template pair<0>(cd0), C::template pair<2>(cd0)};
        const uint32_t v1[4] = {C::template pair<0>(ab1), C::template pair<2>(ab1), C::template pair<0>(cd1), C::template pair<2>(cd1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816(acc[n][2 * half], v0, p[n][i][0], p[n][i][1]);
          mma16816(acc[n][2 * half + 1], v1, p[n][i][0], p[n][i][1]);
        }
      }
    }
    if constexpr (NT > 1) {
      __syncwarp();
      values_read();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float v0 = blind(n, 0) ? 0.f : v_scale, v1 = blind(n, 1) ? 0.f : v_scale, vs0 = v0 * C::kUnit, vs1 = v1 * C::kUnit;
      const float off0 = -C::kBias * v0 * sum[n][0], off1 = -C::kBias * v1 * sum[n][1];
      l[n][0] += sum[n][0];
      l[n][1] += sum[n][1];
      if (change) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[n][j][0] *= alpha[n][0];
          o[n][j][1] *= alpha[n][1];
          o[n][j][2] *= alpha[n][0];
          o[n][j][3] *= alpha[n][1];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[n][j][0] += fmaf(acc[n][j][0], vs0, off0);
        o[n][j][1] += fmaf(acc[n][j][1], vs1, off1);
        o[n][j][2] += fmaf(acc[n][j][2], vs0, off0);
        o[n][j][3] += fmaf(acc[n][j][3], vs1, off1);
      }
    }
    return true;
  }

  // un-normalised outputs and {m, l} of the tile's rows
  __device__ __forceinline__ void put(float (*out)[64], float2* ml, int valid) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + 2 * t + e;
        if (r >= valid) continue;
        if (g == 0) ml[r] = make_float2(m[n][e], l[n][e]);
        float4* at = reinterpret_cast<float4*>(&out[r][8 * g]);
        at[0] = make_float4(o[n][0][e], o[n][0][e + 2], o[n][1][e], o[n][1][e + 2]);
        at[1] = make_float4(o[n][2][e], o[n][2][e + 2], o[n][3][e], o[n][3][e + 2]);
      }
  }
};

// 1 / l for a row that saw something, 0 for one that saw nothing; NaN stays.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.0f / l; }

template <bool BF16>
__device__ __forceinline__ void store4(uint16_t* at, const float4& v, float l) {
  const float inv = inverse(l);
  *reinterpret_cast<uint2*>(at) = make_uint2(kv::pack16<BF16>(v.x * inv, v.y * inv), kv::pack16<BF16>(v.z * inv, v.w * inv));
}

// What a warp has on its way: keys and values of its blocks in turn, kSlots pieces of 4 KB ahead.  look(i): entry of the block table for the
// i-th block of the warp's list.
struct Ring {
  uint8_t codes[kSlots][kBlock];
};

template <typename Look>
struct Feed {
  const Args& a;
  Ring* ring;
  uint64_t* full;
  int head, count;         // key head, blocks of the list
  Look look;
  int slot = 0, done = 0;  // of the piece that is waited for next, pieces so far
  uint32_t phase = 0;
  float ks[2], vs[2];      // scales of the present block and the next; a negative one: there is no such block
  int64_t next = 0;        // the next block's place in the cache
  int later = 0;           // table entry of the block after that

  __device__ __forceinline__ Feed(const Args& args, Ring* r, uint64_t* f, int h, int n, Look l)
      : a(args), ring(r), full(f), head(h), count(n), look(l) {}

  __device__ __forceinline__ int64_t resolve(int page, float* k, float* v) {
    const bool bad = page < 0 || page >= a.cache.blocks;  // reported where it is left out
    const int64_t at = static_cast<int64_t>(bad ? 0 : page) * a.cache.heads + head;
    *k = bad ? -1.f : __ldg(a.cache.k_scale + at);
    *v = bad ? 0.f : __ldg(a.cache.v_scale + at);
    return at;
  }
  __device__ __forceinline__ void request(int s, const uint8_t* base, int64_t at) {
    if ((threadIdx.x & 31) == 0) {
      ptx::mbar_arrive_expect_tx(&full[s], kBlock);
      bulk_load(ring->codes[s], base + at * kBlock, kBlock, &full[s]);
    }
  }
  // entries: of the list's first blocks, as far as there are any
  __device__ __forceinline__ void begin(const int* entries) {
    static_assert(kSlots == 3, "keys and values of the first block, keys of the second");
    const int64_t at = resolve(entries[0], &ks[0], &vs[0]);
    request(0, a.cache.k, at);
    request(1, a.cache.v, at);
    if (count > 1) {
      next = resolve(entries[1], &ks[1], &vs[1]);
      request(2, a.cache.k, next);
    }
    later = entries[2];
  }
  // The next piece, once it is there; nullptr: gave up, with the pieces on their way landed.
  __device__ __forceinline__ const uint8_t* wait(const ptx::AbortCtx& ab) {
    if (__all_sync(0xffffffffu, ptx::mbar_wait(&full[slot], phase, ab, 330))) return ring->codes[slot];
    const long long t0 = clock64();
    int s = slot;
    uint32_t ph = phase;
    for (int k = 0; (threadIdx.x & 31) == 0 && k < kSlots && done + k < 2 * count; ++k) {
      while (!ptx::mbar_try_wait(&full[s], ph) && clock64() - t0 < ptx::kWaitCycles) {
      }
      if (++s == kSlots) {
        s = 0;
        ph ^= 1;
      }
    }
    __syncwarp();
    return nullptr;
  }
  __device__ __forceinline__ void advance() {
    ++done;
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  }
  // block i's keys have been read: its slot takes the values of block i + 1
  __device__ __forceinline__ void keys_read(int i) {
    if (i + 1 < count) request(slot, a.cache.v, next);
    advance();
  }
  // its values: the slot takes the keys of block i + 2
  __device__ __forceinline__ void values_read(int i) {
    ks[0] = ks[1];
    vs[0] = vs[1];
    if (i + 2 < count) {
      next = resolve(later, &ks[1], &vs[1]);
      request(slot, a.cache.k, next);
    }
    if (i + 3 < count) later = look(i + 3);
    advance();
  }
};

struct Smem {
  Ring ring[kWarps];  // afterwards the first 4 KB of a warp's ring are its output, fp32 [16][64]
  // of the cluster's CTAs, written by them: quads of the output that this CTA finishes, and {m, l} of all rows
  float4 part[16 * 16];
  float2 part_ml[kMaxSplits][16];
  float2 ml[kWarps][16];
  uint64_t full[kWarps][kSlots];
  alignas(16) int cost[kRanked + 4];
  int abort_flag;
};
static_assert(4 * (sizeof(Smem) + 1024) <= 228 * 1024, "four CTAs share an SM");

template <bool BF16, bool INT8, int NT>
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(NT)) few_rows_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  RT_PDL_WAIT();
  RT_PDL_LAUNCH_DEPENDENTS();  // not before: launches would queue up on the SMs (single tokens in a loop: 9.0 us a call, now 7.0)
  const int rank = blockIdx.x % a.splits;
  int rest = blockIdx.x / a.splits;
  const int tile = rest % a.tiles;
  rest /= a.tiles;
  const int head = rest % a.cache.heads;
  int seq = rest / a.cache.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.sorted) {
    const int tid = threadIdx.x;
    seq = index_by_cost(sm.cost, a.n_seq, tid < a.n_seq ? a.context[tid] : 0, seq);
  }

  // the warp's first table entries, before it is known how many of them there are
  const int32_t* table = a.table + static_cast<int64_t>(seq) * a.table_stride;
  const int step = a.splits * kWarps, b0 = rank * kWarps + warp;  // this warp's blocks: every step-th one
  int entry[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) entry[i] = b0 + i * step < a.table_stride ? __ldg(table + b0 + i * step) : -1;
  const CachedRows sr(a, seq);
  if (!sr.ok) return;
  using Tile = RowTile<BF16, INT8, NT>;
  const int row0 = tile * Tile::kRows;
  if (row0 >= sr.rows) return;
  const int valid = min(Tile::kRows, sr.rows - row0);
  if (a.splits > 1) ptx::cluster_arrive();  // waited for before another CTA's shared memory is written
  const int n_blocks = (sr.limit(a, row0 + valid - 1) + 63) / 64;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int s = 0; s < kSlots; ++s) ptx::mbar_init(&sm.full[w][s], 1);
    sm.abort_flag = 0;
    ptx::fence_barrier_init();
  }
  __syncthreads();
  ptx::AbortCtx ab{&sm.abort_flag, a.err};
  const int count = b0 < n_blocks ? (n_blocks - b0 + step - 1) / step : 0;
  auto look = [&](int i) { return __ldg(table + b0 + i * step); };
  Feed<decltype(look)> feed(a, &sm.ring[warp], sm.full[warp], head, count, look);
  if (count > 0) feed.begin(entry);

  Tile rows;
  rows.g = lane >> 2;
  rows.t = lane & 3;
  rows.begin(a, sr, head, row0);
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    const uint8_t* kp = feed.wait(ab);
    if (!kp) break;
    if (!rows.block(kp, feed.ks[0], feed.vs[0], b0 + i * step, [&] { feed.keys_read(i); }, [&] { return feed.wait(ab); },
                    [&] { feed.values_read(i); }))
      break;
  }

  // ---- the warps of the CTA
  auto out_of = [&](int w) { return reinterpret_cast<float(*)[64]>(sm.ring[w].codes[0]); };
  rows.put(out_of(warp), sm.ml[warp], valid);
  __syncthreads();
  auto store = [&](int r, int d, const float4& v, float l) { store4<BF16>(sr.output(a, head, row0 + r) + d, v, l); };
  const int per = 256 / a.splits;  // quads that a CTA finishes at most
  if (a.splits > 1) ptx::cluster_wait();  // the others run: their shared memory can be written
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
      continue;
    }
    const int owner = i % a.splits;
    kv::st_cluster_f4(kv::peer_address(ptx::smem_u32(&sm.part[rank * per + i / a.splits]), owner), v);
    if (d == 0)
      for (int w = 0; w < a.splits; ++w) kv::st_cluster_f2(kv::peer_address(ptx::smem_u32(&sm.part_ml[rank][r]), w), make_float2(M, L));
  }
  if (a.splits == 1) return;
  // ---- the CTAs of the cluster: each finishes its share of the tile's quads of dimensions, which the others have written to it
  __syncwarp();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  for (int k = threadIdx.x; rank + a.splits * k < valid * 16; k += kWarps * 32) {
    const int i = rank + a.splits * k, r = i >> 4, d = (i & 15) * 4;
    float M = -INFINITY, L = 0.f;
    float4 v = make_float4(0, 0, 0, 0);
    for (int w = 0; w < a.splits; ++w) M = fmaxf(M, sm.part_ml[w][r].x);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < a.splits; ++w) {
      const float2 ml = sm.part_ml[w][r];
      const float4 x = sm.part[w * per + k];
      const float f = ex2(ml.x - ref);
      L = fmaf(ml.y, f, L);
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
      v.z = fmaf(x.z, f, v.z);
      v.w = fmaf(x.w, f, v.w);
    }
    store(r, d, v, L);
  }
}

constexpr int kSms = 148;

// CTAs that share a tile's keys, a power of two (clusters of 3 or 6 run slower than of 2 or 4): as many as have a block for every warp, do not
// make more than 1.35 rounds of CTAs, and, beyond two CTAs an SM, leave a warp of the longest sequence four blocks.
// More than one round, with the long sequences first, is for ragged lengths, which a batch of answers has.  us by CTAs of a tile, all lengths equal and from 1/16 of
// that on at random: 96 tiles x 16384 keys 4: 42.9 and 34.2, 8: 45.3 and 27.4; 384 x 4096 1: 41.5 and 34.4, 2: 45.6 and 25.0; 384 x 8192 1: 76.0 and 63.8,
// 2: 80.3 and 43.7.  Fewer than four blocks a warp do not pay for the join: 96 x 4096 4: 14.7 and 13.1, 8: 17.5 and 15.4; 192 x 2048 2: 14.6 and 12.5, 4: 16.6 and
// 14.9; but while few CTAs run, they shorten the chain: 24 x 4096 4: 9.0 and 9.0, 8: 7.7 and 7.9.
// With 16 rows a tile results weigh more, and one round it is.
int splits_of(int64_t units, int tile_rows, int64_t keys) {
  const int64_t slots = kSms * ctas_per_sm(tile_rows / 8), room = tile_rows == 8 ? slots * 135 / 100 : slots;
  auto pays = [&](int64_t splits) { return tile_rows != 8 || units * splits <= 2 * kSms || keys >= 64 * kWarps * 4 * splits; };
  int splits = 1;
  while (splits < kMaxSplits && units * splits * 2 <= room && keys > 64 * kWarps * splits && pays(2 * splits)) splits *= 2;
  return splits;
}

// The same for the kernel of many rows, one CTA an SM: rounds of CTAs times the measured cost of one, 12 us and 0.85 us a block of keys (9 and 0.51
// for at most 128 rows, 0.45 for at most 64), 0.5 us more where a cluster joins its results.  Clusters of 2, 4 and 8 fit 74, 33 and 15 times on the chip.
int many_rows_splits(int64_t units, int rows, int64_t keys, double* us) {
  constexpr int kFit[4] = {kSms, 74, 33, 15};
  const double base = rows > 128 ? 12.0 : 9.0, block = rows > 128 ? 0.85 : rows > 64 ? 0.51 : 0.45, blocks = static_cast<double>((keys + 63) / 64);
  int best = 1;
  double least = 1e30;
  for (int k = 0; k < 4; ++k) {
    const int splits = 1 << k;
    const double rounds = static_cast<double>((units + kFit[k] - 1) / kFit[k]);
    const double cost = rounds * (base + (k > 0 ? 0.5 : 0.0) + block * blocks / splits);
    if (cost < least) {
      least = cost;
      best = splits;
    }
  }
  *us = least;
  return best;
}

template <bool BF16, bool INT8, int NT>
rt_status launch_few_rows(const Args& a, cudaStream_t st) {
  auto kern = few_rows_kernel<BF16, INT8, NT>;
  RT_TRY(ensure_kernel_smem(reinterpret_cast<const void*>(kern), sizeof(Smem), true));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(a.n_seq) * a.cache.heads * a.tiles * a.splits));
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

template <bool BF16, bool INT8>
rt_status launch_by_rows(const Args& a, cudaStream_t st) {
  return a.tile_rows == 8 ? launch_few_rows<BF16, INT8, 1>(a, st) : launch_few_rows<BF16, INT8, 2>(a, st);
}

}  // namespace
}  // namespace rt

using namespace rt;

namespace {

// Does the output [tokens][width] share memory with the rows of the queries (`width` values each, `stride` apart)?
bool overlaps(const void* out, const void* q, int64_t stride, int64_t tokens, int64_t width) {
  const int64_t row = 2 * width, step = 2 * stride, begin = reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(q), end = begin + tokens * row;
  if (end <= 0 || begin >= (tokens - 1) * step + row) return false;
  // the first row that ends behind the output's beginning
  const int64_t i = begin < row ? 0 : step == 0 ? tokens : std::min(tokens, (begin - row) / step + 1);
  return i < tokens && i * step < end;
}

}  // namespace

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
  if (n_seq == 0 || tokens == 0) return RT_OK;
  max_q += max_q == 0;
  RT_REQUIRE(out && q, RT_ERR_INVALID, "cached_attention: null pointer");
  RT_REQUIRE(((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0 && q_stride % 8 == 0 && q_stride >= 0,
             RT_ERR_INVALID, "cached_attention: queries and output must be 16-byte aligned, the query stride a multiple of 8 values");
  a.out = static_cast<uint16_t*>(out);
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_stride;
  a.table = table;
  a.table_stride = table_stride;
  a.context = context;
  a.first = first;
  a.n_seq = n_seq;
  a.tokens = tokens;
  a.max_q = std::min(max_q, tokens);
  a.heads = heads;
  a.group = heads / a.cache.heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  RT_REQUIRE(static_cast<int64_t>(a.max_q) * a.group < (int64_t{1} << 30), RT_ERR_UNSUPPORTED, "cached_attention: too many query rows");
  const int rows = a.max_q * a.group;
  const int64_t heads_of_all = static_cast<int64_t>(n_seq) * a.cache.heads;  // under 2^41
  RT_REQUIRE(heads_of_all < (int64_t{1} << 26), RT_ERR_UNSUPPORTED,
             "cached_attention: %d sequences of up to %d query tokens are too many for one call", n_seq, max_q);
  RT_REQUIRE(std::isfinite(a.scale_log2), RT_ERR_INVALID, "cached_attention: the scale is no number, or too large for one");
  RT_REQUIRE(!overlaps(out, q, q_stride, tokens, int64_t{64} * heads), RT_ERR_INVALID, "cached_attention: the output overlaps the queries");
  const int64_t widest = static_cast<int64_t>(table_stride) * 64;
  const int64_t keys = max_context > 0 ? std::min<int64_t>(max_context, widest) : widest;
  // Which kernel: the one of few rows pays for every 16 rows that there are (1.65 ns a tile and block of keys on the full chip), the one of many
  // rows for whole tiles.  12 x 4096 keys, 12 heads, 64 rows each: 60.5 and 39.8 us; 16 x 2000 keys 45.7 and 47.3; 16 x 512 to 4096 keys, 5 to
  // 64 rows: 41 and 53.
  const int64_t few_tiles = std::min(n_seq * static_cast<int64_t>((rows + 15) / 16), static_cast<int64_t>(tokens) * a.group / 16 + n_seq / 2);
  // Tiles of the kernel of many rows: as many for each sequence as the longest one has, or, where that is much more than the rows of the call
  // make, by a search for each CTA's sequence.  12 heads, causal, us: 8 sequences of 2048 rows with 64 tiles each 525 (most CTAs had no work and
  // were ranked all the same), searched for 133; 64 x 512 with 128 each 1038 and 237; with 2 each 227.
  a.tiles = (rows + 255) / 256;
  const int64_t direct = many_rows_items(a);
  a.listed = true;
  a.listed = static_cast<double>(direct) > static_cast<double>(many_rows_items(a)) * (1.5 + n_seq * 1e-3);
  double many_us = 0;
  const int many_splits = many_rows_splits(many_rows_items(a) * a.cache.heads, rows, keys, &many_us);
  const bool many = rows > kFewRows ||
                    (rows > 32 && many_us < 5.0 + 1.65e-3 * static_cast<double>(few_tiles * a.cache.heads) * ((keys + 63) / 64));
  a.tile_rows = many ? 256 : rows <= 8 ? 8 : 16;
  a.tiles = (rows + a.tile_rows - 1) / a.tile_rows;
  const int64_t units = heads_of_all * a.tiles;
  a.err = device_error_word();
  RT_REQUIRE(a.err != nullptr, RT_ERR_CUDA, "cached_attention: cannot allocate the device error word");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == RT_BF16, int8 = cache->format == RT_KV_INT8;
  if (many) {
    a.splits = many_splits;
    return launch_cached_attention_many_rows(a, bf16, int8, st);
  }
  a.splits = splits_of(units, a.tile_rows, keys);
  a.sorted = n_seq > 1 && n_seq <= kWarps * 32 && units * a.splits > kSms * ctas_per_sm(a.tile_rows / 8);
  if (bf16) return int8 ? launch_by_rows<true, true>(a, st) : launch_by_rows<true, false>(a, st);
  return int8 ? launch_by_rows<false, true>(a, st) : launch_by_rows<false, false>(a, st);
}
