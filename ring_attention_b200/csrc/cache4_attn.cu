// Attention over the 4-bit key/value cache (layout and code formula: cache4_layout.h).
//
// For a query row of head h and the rows (keys) of its key/value head:
//   s = scale * q . k (+ ALiBi, masks),  p = exp(s - max),  out = sum p v / sum p,  L = max + log sum p.
// With k = min + step * c over a group of 64 channels (c = code, 0..15):
//   q . k = sum over groups of  step * (q . c) + min * (sum of q over the group)
//   sum p v = sum over keys of (p step) c + p min
// so the matrix products run on the codes themselves and no key or value is ever rounded.  A code in bits 0-3 or 4-7
// of a half IS the fp16 number c 2^-24 or 16 c 2^-24 (a subnormal, which the tensor cores multiply exactly), so eight
// codes become operands with four ANDs and one shift.  Queries are scaled by a power of two per row into the fp16
// range, which keeps all bits of a bf16 query (down to 2^-24 of the row's largest); the one rounding of bf16 calls is
// that of p * step to fp16 (relative 2^-11).  fp32 calls split q and p * step into two fp16 parts, cut such that the sums
// that the tensor cores would truncate are exact (QueryTile, whole_number_scale): results are off by 1e-7 of themselves.
//
// The decoding form reads its cache once and does little with it (8 query rows share 144 bytes a key at 128
// channels): beside the stream of the cache most instructions are the integer work that turns codes
// into operands.  That is why the products are warp-level MMAs with the codes on the M side: fragments are made
// in registers straight from the packed words, where a tensor-memory MMA would want the decoded tile written to
// shared memory and read back (from 64 query rows on that pays: cache4_prompt.cu).
//
// A warp streams units of 64 keys through a ring of stages of its own that bulk copies fill (no barrier between
// warps until the end of a segment); the four warps of a CTA share a run of one item's units, an item being a (sequence,
// head, query tile), and join their partial softmaxes in shared memory.
//   Short caches (up to kShortUnits units): a cluster of 1 to 8 CTAs has an item and joins through shared memory too.
//   Others: all units of all items, in a row, are cut into as many equal runs as CTAs fit on the GPU, so that ragged
//   lengths leave no CTA idle; a run goes through segments of one or more items, and a second kernel joins the items
//   that were cut (cache4_sched.cuh).
//
// Measured, bf16, 128 channels, one token of 4 query heads a key/value head: 8 x 32768 keys of 8 heads 71 us (302 MB,
// 4.2 TB/s), 64 x 819 to 8192 keys 91 us (345 MB, 3.8 TB/s), one sequence of 131072 keys 42 us (151 MB, 3.6 TB/s), where
// a copy runs at 6.5 TB/s; the join 6 us.  What bounds it is latency at few warps: 168 registers leave 11 warps an SM, which use
// 49 to 53 % of issue slots and 51 to 57 % of the integer pipe, and wait longest for results of fixed latency (1.1 cycles an
// instruction) and for the pipe (0.7), less for memory (0.4 to 0.7).  From 151 to 302 MB the time grows at 5.2 TB/s; some 13 us do
// not depend on the length: launch, cuts, first copies, cold code and joining.
// 16 heads of 1024 keys take 7.4 us in a graph, of which the launch and the fetch of cold code are the most.
#include <cooperative_groups.h>

#include <climits>
#include <type_traits>

#include "cache4_sched.cuh"
#include "tc_common.cuh"

#include <cuda_fp16.h>

namespace ra {
namespace {

constexpr int kWarps = 4;

constexpr int kSub = kCacheUnit / 16;  // fragments of 16 keys of a unit
constexpr int kShortUnits = 4096 / kCacheUnit;  // of a capacity

// ---- fragments ---------------------------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with nothing to add to.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Codes as fp16 pairs: those in bits 0-3 of each half of x times 2^-24, those in bits 4-7 times 2^-20.
constexpr float kCodeUnit = 16777216.f;  // 2^24
__device__ __forceinline__ uint32_t codes_lo(uint32_t x) { return x & 0x000f000fu; }
__device__ __forceinline__ uint32_t codes_hi(uint32_t x) { return x & 0x00f000f0u; }
__device__ __forceinline__ uint32_t half2_of(float x0, float x1) {
  const __half2 h = __floats2half2_rn(x0, x1);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   ptx::smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(ptx::smem_u32(bar))
               : "memory");
}

// Load of 8 consecutive channels as floats.
template <typename T>
__device__ __forceinline__ void load_q8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = load_as_float(p + i);
  }
}

// The query rows of a tile as B fragments of q 2^-e (e: a row's own, the largest channel in [2^13, 2^14)), their group
// sums in the unit of the products, the factor that makes base-2 scores of them, positions and ALiBi slopes.
//
// fp32 queries go in as two fp16 parts, the first rounded to a multiple of 8 whatever the channel's size: its products
// with codes then add up to whole numbers (of 8 units) below 2^24, which the tensor cores add exactly, where they
// truncate otherwise (a bias of up to 4e-6 in L).  With the second part, a multiple of 2^-9 at most off, that is
// 2^-22 of the row's largest channel.
template <int D, int NT, int PARTS>
struct QueryTile {
  static constexpr int NG = D / kCacheGroup;
  uint32_t frag[NT][NG][4][2][PARTS];  // [..][2 j + hh][register]
  // Of rows 2t, 2t + 1: PARTS 1: the sum over the group; 2: -8 times the sums of the first parts and of the second ones.
  float sum[NT][NG][2][PARTS];
  float factor[NT][2];
  int32_t pos[NT][2];
  float slope[NT][2];  // times log2 e

  template <typename T>
  __device__ __forceinline__ void load(const AttnArgs& a, int b, int h, int tile) {
    const CacheAttnParams& p = a.p;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int per = p.h / p.c.hkv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = (tile * NT + nt) * 8 + g;
      const bool live = r < a.rows;
      const T* src = (const T*)p.q.ptr + b * p.q.sb + (int64_t)(r / per) * p.q.sl + (int64_t)(h * per + r % per) * p.q.sh;
      float x[NG][2][8], top = 0.f;
#pragma unroll
      for (int c = 0; c < NG; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[c][j][i] = 0.f;
          if (live) load_q8(src + c * kCacheGroup + 8 * (2 * t + j), a.vec, x[c][j]);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[c][j][i]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(13 - exponent of top), 1 for a row of zeros or infinities, within what a float holds
      const int e = (int)(__float_as_uint(top) >> 23);
      const float norm = top > 0.f && e < 255 ? __uint_as_float((uint32_t)min(13 + 254 - e, 253) << 23) : 1.f;
      // (never 0, so that a masked score of -inf stays one; a negative scale turns the queries' sign)
      const float f = fmaxf(kCodeUnit / norm * fabsf(p.scale) * 1.4426950408889634f, 1e-30f);
      factor[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
      factor[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
      for (int c = 0; c < NG; ++c) {
        float s[PARTS] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[c][j][i] *= p.scale < 0.f ? -norm : norm;
#pragma unroll
          for (int f = 0; f < PARTS; ++f) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y[i] = x[c][j][i];
              if constexpr (PARTS > 1) {
                if (f == 0) y[i] = (y[i] + 0x1.8p26f) - 0x1.8p26f;
                x[c][j][i] -= y[i];
              }
              s[f] += y[i];
            }
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {  // the second register meets codes_hi
              frag[nt][c][2 * j + hh][0][f] = half2_of(y[2 * hh], y[2 * hh + 4]);
              frag[nt][c][2 * j + hh][1][f] = half2_of(y[2 * hh + 1] * 0.0625f, y[2 * hh + 5] * 0.0625f);
            }
          }
        }
#pragma unroll
        for (int f = 0; f < PARTS; ++f) {
          s[f] += __shfl_xor_sync(0xffffffffu, s[f], 1);
          s[f] += __shfl_xor_sync(0xffffffffu, s[f], 2);
          s[f] *= (PARTS > 1 ? -8.f : 1.f) / kCodeUnit;
          sum[nt][c][0][f] = __shfl_sync(0xffffffffu, s[f], 8 * t);
          sum[nt][c][1][f] = __shfl_sync(0xffffffffu, s[f], 8 * t + 4);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = min((tile * NT + nt) * 8 + 2 * t + i, a.rows - 1);
        pos[nt][i] = 0;
        slope[nt][i] = 0.f;
        if (p.kinds) pos[nt][i] = p.q_pos ? p.q_pos[(int64_t)b * p.lq + row / per] : p.c.seen[b] - p.lq + row / per;
        if (p.kinds & RA_MOD_ALIBI) slope[nt][i] = p.slopes[h * per + row % per] * 1.4426950408889634f;
      }
    }
  }
};

// One stage: the codes and limits of a unit's keys, and their positions where a mask asks for them.
template <int D, bool kWithV>
struct Stage {
  static constexpr int NG = D / kCacheGroup;
  static constexpr int kCodes = kCacheUnit * D / 2, kLimits = kCacheUnit * NG * 4;
  static constexpr int kK = 0, kV = kCodes, kKl = kWithV ? 2 * kCodes : kCodes, kVl = kKl + kLimits;
  static constexpr int kPos = kWithV ? kVl + kLimits : kVl;
  static constexpr int kBytes = kPos + kCacheUnit * 4;

  // One copy for each array, by a lane each: lane i < kCopies of a warp owns array i.
  static constexpr int kCopies = kWithV ? 4 : 2;
  const char* src;  // unit 0 of the lane's array
  uint32_t bytes, at;
  bool mine;
  __device__ __forceinline__ void init(const CacheView& c, int64_t bh, bool with_pos) {
    const int lane = threadIdx.x & 31;
    const int64_t row = bh * c.cap;
    src = reinterpret_cast<const char*>(c.k + row * (D / 2));
    bytes = kCodes;
    at = kK;
    if (lane == 1) src = reinterpret_cast<const char*>(c.kl + row * NG), bytes = kLimits, at = kKl;
    if (kWithV && lane == 2) src = reinterpret_cast<const char*>(c.v + row * (D / 2)), bytes = kCodes, at = kV;
    if (kWithV && lane == 3) src = reinterpret_cast<const char*>(c.vl + row * NG), bytes = kLimits, at = kVl;
    if (lane == kCopies) src = reinterpret_cast<const char*>(c.pos + row), bytes = kCacheUnit * 4, at = kPos;
    mine = lane < kCopies + (with_pos ? 1 : 0);
  }
  __device__ __forceinline__ void fill(char* stage, uint64_t* bar, int unit) const {
    if (mine) {
      ptx::mbar_arrive_expect_tx(bar, bytes);
      bulk_load(stage + at, src + (int64_t)unit * bytes, bytes, bar);
    }
  }
};

// Words of K: this lane's 2 NG words of a row.
template <int D>
__device__ __forceinline__ void k_words(const char* row, int slot, int t, uint32_t (&w)[D / 32]) {
  if constexpr (D == 64) {
    const uint2 x = *reinterpret_cast<const uint2*>(row + 8 * t);
    w[0] = x.x, w[1] = x.y;
  } else if constexpr (D == 128) {
    const uint4 x = *reinterpret_cast<const uint4*>(row + 16 * t);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(row + ((i ^ slot) & 1) * 64 + 16 * t);
      w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
    }
  }
}
// Words of V: word g of every group of a row.
template <int D>
__device__ __forceinline__ void v_words(const char* row, int slot, int g, uint32_t (&w)[D / 64]) {
  const int at = g ^ cache_v_swizzle(D, slot);
  if constexpr (D == 64) {
    w[0] = *reinterpret_cast<const uint32_t*>(row + 4 * at);
  } else if constexpr (D == 128) {
    const uint2 x = *reinterpret_cast<const uint2*>(row + 8 * at);
    w[0] = x.x, w[1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(row + 16 * at);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  }
}

// Limits of a row's groups.
template <int D>
__device__ __forceinline__ void limit_words(const char* limits, int slot, uint32_t (&w)[D / 64]) {
  if constexpr (D == 64) {
    w[0] = *reinterpret_cast<const uint32_t*>(limits + 4 * slot);
  } else if constexpr (D == 128) {
    const uint2 x = *reinterpret_cast<const uint2*>(limits + 8 * slot);
    w[0] = x.x, w[1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(limits + 16 * slot);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  }
}
__device__ __forceinline__ float limit_step(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float limit_min(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Scores of 16 keys, halves 0 and 1 of the fragment rows, against the query tile, to be multiplied by its factors:
// s[nt][2 half + i] is key (half, g) and row 2t + i.
template <int D, int NT, int PARTS>
__device__ __forceinline__ void scores16(const char* stage, int kl_at, int u, const QueryTile<D, NT, PARTS>& q, float (&s)[NT][4]) {
  constexpr int NG = D / kCacheGroup;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t w[2][D / 32], lim[2][NG];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int slot = 16 * u + 8 * half + cache_kappa(g);
    k_words<D>(stage + slot * (D / 2), slot, t, w[half]);
    limit_words<D>(stage + kl_at, slot, lim[half]);
  }
#pragma unroll
  for (int c = 0; c < NG; ++c) {
    float acc[NT][PARTS][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const uint32_t x = w[0][2 * c + j] >> (8 * hh), y = w[1][2 * c + j] >> (8 * hh);
        const uint32_t a0 = codes_lo(x), a1 = codes_lo(y), a2 = codes_hi(x), a3 = codes_hi(y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int f = 0; f < PARTS; ++f) {
            const uint32_t(&b)[2][PARTS] = q.frag[nt][c][2 * j + hh];
            if (j + hh == 0) mma16816_first(acc[nt][f], a0, a1, a2, a3, b[0][f], b[1][f]);
            else mma16816(acc[nt][f], a0, a1, a2, a3, b[0][f], b[1][f]);
          }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float step = limit_step(lim[i >> 1][c]), low = limit_min(lim[i >> 1][c]);
        const float(&sum)[PARTS] = q.sum[nt][c][i & 1];
        float add = c == 0 ? 0.f : s[nt][i];
        if constexpr (PARTS == 1) {
          add = c == 0 ? low * sum[0] : fmaf(low, sum[0], add);
          s[nt][i] = fmaf(step, acc[nt][0][i], add);
        } else {  // of the codes less 8, with min + 8 step: smaller terms, of which less is lost
          add = fmaf(fmaf(low, -0.125f, -step), sum[0] + sum[1], add);
          s[nt][i] = fmaf(step, (acc[nt][0][i] + sum[0]) + (acc[nt][1][i] + sum[1]), add);
        }
      }
  }
}

// What is left between a raw score and the exponent's argument: the factor, where mod16 has not applied it.
template <bool MASKED>
__device__ __forceinline__ float finish(float s, float factor, float add) {
  return MASKED ? s + add : fmaf(s, factor, add);
}

// ALiBi and the masks on the scores of 16 keys; -inf where a row does not see a key.  The masked form leaves base-2
// scores, the other raw ones (factors are not negative).
template <bool MASKED, int D, int NT, int PARTS>
__device__ __forceinline__ void mod16(const AttnArgs& a, const char* stage, int pos_at, int u, int live_keys,
                                      const QueryTile<D, NT, PARTS>& q, float (&s)[NT][4]) {
  const int g = (threadIdx.x & 31) >> 2;
  const uint32_t kinds = MASKED ? a.p.kinds : 0u;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int key = 16 * u + 8 * half + cache_kappa(g);
    const bool live = key < live_keys;
    const int kpos = MASKED ? *reinterpret_cast<const int32_t*>(stage + pos_at + 4 * key) : 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float& x = s[nt][2 * half + i];
        bool vis = live;
        if constexpr (MASKED) {
          x *= q.factor[nt][i];
          if (kinds & RA_MOD_ALIBI) x = fmaf(-q.slope[nt][i], (float)(q.pos[nt][i] - kpos), x);
          if (kinds & RA_MOD_CAUSAL) vis = vis && kpos <= q.pos[nt][i];
          if (kinds & RA_MOD_WINDOW) vis = vis && q.pos[nt][i] - kpos < a.p.window;
        }
        if (!vis) x = -INFINITY;
      }
  }
}

// The exponent of the largest p * step: 2^6, times up to 2^8 before the reference moves, below fp16's 2^16.
constexpr float kHeadroom = 6.f;

// Codes less 8, in the same unit.
__device__ __forceinline__ uint32_t less_8(uint32_t x, bool high) {
  const uint32_t eight = high ? 0x00800080u : 0x00080008u;  // 8 in that unit
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&eight));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// fp32 calls: the power of two that brings the largest p * step of a unit's 64 keys, for a row and a group, into [2^12,
// 2^13), and the one that takes it back.  The first fp16 part is then rounded to a multiple of 4: its products with codes
// less 8 add up to whole numbers (of 4 units) below 2^24, which the tensor cores add exactly; the second part is 2^-24 of
// the largest off.  (Two parts that keep 22 bits of each number instead, in sums that truncate, were off by 4e-6 of a
// channel that others in its group drown.)
template <int NT, int NG>
__device__ __forceinline__ void whole_number_scale(const float (&p)[kSub][NT][4], const uint32_t (&vlim)[kSub][2][NG], int c,
                                                   float (&scale)[NT][2], float (&back)[NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float top = 0.f;  // (NaN is passed over)
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) top = fmaxf(top, p[u][nt][2 * half + i] * limit_step(vlim[u][half][c]));
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const int e = min(max(266 - (int)(__float_as_uint(top) >> 23), 1), 253);
      scale[nt][i] = __uint_as_float((uint32_t)e << 23);
      back[nt][i] = __uint_as_float((uint32_t)(254 - e) << 23);
    }
}

template <int D>
struct AttnShape {
  static constexpr int kStages = D == 64 ? 3 : 2;
  using St = Stage<D, true>;
  static constexpr int kRing = kWarps * kStages * St::kBytes;
  static constexpr int kJoin = (kWarps + 1) * 8 * (D + 2) * 4;  // the warps' results for 8 rows, and the CTA's
  static constexpr int kSmem = (kRing > kJoin ? kRing : kJoin) + kWarps * kStages * 8 + 64;
};

// CTAs of an SM that the registers are divided for; shared memory holds as many.
template <typename T, int D, int NT>
constexpr int kPerSm = D == 256 ? 1 : (sizeof(T) == 4 ? (D == 64 ? 3 : 2) : (D == 64 ? (NT == 1 ? 4 : 3) : (NT == 1 ? 3 : 2)));

template <typename T, int D, int NT, bool MASKED>
__global__ void __launch_bounds__(kWarps * 32, kPerSm<T, D, NT>) cache_attn_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
  using Shape = AttnShape<D>;
  using St = typename Shape::St;
  constexpr int NG = D / kCacheGroup, kStages = Shape::kStages;
  extern __shared__ __align__(128) char smem[];
  constexpr int kBars = Shape::kSmem - 64 - kWarps * kStages * 8;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBars);
  Run* s_run = reinterpret_cast<Run*>(smem + Shape::kSmem - 64);
  int* s_has = reinterpret_cast<int*>(smem + Shape::kSmem - 64 + 32);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(smem + Shape::kSmem - 64 + 36);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int per_seq = a.p.c.hkv * a.tiles;
  Run run;
  if (warp == 0) {
    const bool has = a.cluster || find_run<MASKED>(a.p.c, per_seq, blockIdx.x, a.ctas, run);
    if (lane == 0) {
      *s_run = run;
      *s_has = has;
      *s_abort = 0;
    }
  } else if (warp == 1 && lane < kWarps * kStages) {
    ptx::mbar_init(bars + lane, St::kCopies + (MASKED ? 1 : 0));
    ptx::fence_barrier_init();
  }
  __syncthreads();
  launch_dependents();
  if (!*s_has) return;
  run = *s_run;
  char* ring = smem + warp * kStages * St::kBytes;
  uint64_t* bar = bars + warp * kStages;
  uint32_t phase = 0;
  int slot = 0;
  for (bool again = false;; again = true) {  // segments of the run
    Segment w;
    if (a.cluster) {
      const int item = blockIdx.x / a.cluster;
      w.b = item / per_seq;
      w.h = item % per_seq / a.tiles;
      w.tile = item % a.tiles;
      w.first = blockIdx.x % a.cluster * kWarps;
      w.last = INT_MAX;
      w.step = a.cluster * kWarps;
      w.whole = a.cluster == 1;
    } else {
      if (again) {
        if (*s_abort) return;
        // what the join has read and written is written by bulk copies next
        ptx::fence_proxy_async_smem();
        __syncthreads();
      }
      if (!next_segment<MASKED>(a, per_seq, run, w)) return;
      w.step = kWarps;
    }
    const int64_t bh = (int64_t)w.b * a.p.c.hkv + w.h;
    const int len = min(max(a.p.c.len[w.b], 0), a.p.c.cap);

    QueryTile<D, NT, PARTS> q;
    q.template load<T>(a, w.b, w.h, w.tile);
    UnitWalk<MASKED> walk;
    if constexpr (MASKED) {
      int least = q.pos[0][0], most = q.pos[0][0];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) least = min(least, q.pos[nt][i]), most = max(most, q.pos[nt][i]);
      walk.see(a, bh, __reduce_min_sync(0xffffffffu, least), __reduce_max_sync(0xffffffffu, most));
    }
    walk.init(len, w.first + warp, w.last, w.step);
    St copy;
    copy.init(a.p.c, bh, MASKED);

    // o: of the products with codes, in units of 2^-24 (2^-20 where the second index is odd); mid: of p min;
    // m: reference of the exponents, l: sum of p
    float o[NT][NG][4][4], mid[NT][NG][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) m[nt][i] = -INFINITY, l[nt][i] = 0.f;
#pragma unroll
      for (int c = 0; c < NG; ++c) {
        mid[nt][c][0] = mid[nt][c][1] = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][c][x][i] = 0.f;
      }
    }

    int queue[kStages];  // units in flight, the next one first
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      const int to = slot + i < kStages ? slot + i : slot + i - kStages;
      queue[i] = walk.next();
      if (queue[i] >= 0) copy.fill(ring + to * St::kBytes, bar + to, queue[i]);
    }
    bool stuck = false;
#pragma unroll 1
    while (queue[0] >= 0) {
      // (the vote keeps the warp together: a lane whose own wait ran out must not leave alone)
      stuck = !__all_sync(0xffffffffu, ptx::mbar_wait(bar + slot, phase, s_abort, a.status, kStCacheWait));
      if (stuck) break;
      char* stage = ring + slot * St::kBytes;
      const int live_keys = len - queue[0] * kCacheUnit;
      float s[kSub][NT][4];
      uint32_t vlim[kSub][2][NG];
      bool grow = false;
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        scores16<D, NT, PARTS>(stage, St::kKl, u, q, s[u]);
        if (MASKED || live_keys < kCacheUnit) mod16<MASKED, D, NT, PARTS>(a, stage, St::kPos, u, live_keys, q, s[u]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = 16 * u + 8 * half + cache_kappa(g);
          limit_words<D>(stage + St::kVl, key, vlim[u][half]);
          if (live_keys < kCacheUnit && key >= live_keys) {  // rows behind the last hold anything
#pragma unroll
            for (int c = 0; c < NG; ++c) vlim[u][half][c] = 0u;
          }
        }
      }
      // The exponents' reference m is the largest score + log2 of the key's largest step, less kHeadroom: p * step then
      // fills the fp16 range from the top and what falls below it is less than 2^-30 of the largest term.  It moves only
      // when a score exceeds it by 2^8, so that most units neither shuffle nor rescale.
      float cand[NT][2];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float st = limit_step(vlim[u][half][0]);
#pragma unroll
          for (int c = 1; c < NG; ++c) st = fmaxf(st, limit_step(vlim[u][half][c]));
          float lg;
          asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(st));
          lg = fmaxf(lg, -64.f) - kHeadroom;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float x = finish<MASKED>(s[u][nt][2 * half + i], q.factor[nt][i], lg);
              cand[nt][i] = u == 0 && half == 0 ? x : fmaxf(cand[nt][i], x);
            }
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) grow |= cand[nt][i] > m[nt][i] + 8.f;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x = cand[nt][i];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x, m[nt][i]);
            const float root = m[nt][i] == -INFINITY ? 0.f : ptx::ex2(0.5f * (m[nt][i] - x)), f = root * root;  // (part_root)
            m[nt][i] = x;
            l[nt][i] *= root;
            l[nt][i] *= root;
#pragma unroll
            for (int c = 0; c < NG; ++c) {
              mid[nt][c][i] *= f;
#pragma unroll
              for (int y = 0; y < 4; ++y) o[nt][c][y][i] *= f, o[nt][c][y][2 + i] *= f;
            }
          }
      }
      if constexpr (MASKED) {
        // A group of V that is NaN has to reach every row that sees its key, and below p = 0 stands for a key that is hidden: p of
        // such keys stays above 0.
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int c = 0; c < NG; ++c) sum += limit_step(vlim[u][half][c]);
        if (__any_sync(0xffffffffu, sum != sum)) {
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float key = 0.f;
#pragma unroll
              for (int c = 0; c < NG; ++c) key += limit_step(vlim[u][half][c]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float& x = s[u][nt][2 * half + i];
                  if (key != key && x > -INFINITY) x = fmaxf(x, m[nt][i] - 120.f);
                }
            }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float base = m[nt][i] == -INFINITY ? 0.f : m[nt][i];
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float& x = s[u][nt][2 * half + i];
              x = ptx::ex2(finish<MASKED>(x, q.factor[nt][i], -base));
              l[nt][i] += x;
            }
        }
      // out += P V, a group of 64 channels at a time.  A unit is summed apart from the running total, which the tensor
      // cores would add to with truncation: codes are not negative, so that the loss would grow with the length.
      // (fp32 calls: whole_number_scale.)
#pragma unroll
      for (int c = 0; c < NG; ++c) {
        float fresh[NT][PARTS][4][4], fresh_mid[NT][2] = {};
        float scale[NT][2], back[NT][2];  // fp32 calls: into the range of whole numbers, and back
        if constexpr (PARTS > 1)
          whole_number_scale<NT, NG>(s, vlim, c, scale, back);
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          uint32_t pb[NT][2][PARTS];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float vs = limit_step(vlim[u][half][c]);
            const float vm = PARTS > 1 ? fmaf(8.f, vs, limit_min(vlim[u][half][c])) : limit_min(vlim[u][half][c]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float x[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float pr = s[u][nt][2 * half + i];
                float& m_sum = PARTS > 1 ? fresh_mid[nt][i] : mid[nt][c][i];
                x[i] = pr * vs;
                if constexpr (MASKED) {  // what a mask hides may be NaN
                  if (pr == 0.f) x[i] = 0.f;
                  else m_sum = fmaf(pr, vm, m_sum);
                } else {
                  m_sum = fmaf(pr, vm, m_sum);
                }
                if constexpr (PARTS > 1) x[i] *= scale[nt][i];
              }
              if constexpr (PARTS > 1) {
                const float y0 = (x[0] + 0x1.8p25f) - 0x1.8p25f, y1 = (x[1] + 0x1.8p25f) - 0x1.8p25f;
                pb[nt][half][0] = half2_of(y0, y1);
                pb[nt][half][1] = half2_of(x[0] - y0, x[1] - y1);
              } else {
                pb[nt][half][0] = half2_of(x[0], x[1]);
              }
#pragma unroll
              for (int f = 0; f < PARTS; ++f) pb[nt][half][f] = transpose8(pb[nt][half][f]);
            }
          }
          uint32_t lo[2], hi[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int s0 = 16 * u + 8 * half + cache_kappa(2 * t), s1 = 16 * u + 8 * half + cache_kappa(2 * t + 1);
            uint32_t w0[NG], w1[NG];
            v_words<D>(stage + St::kV + s0 * (D / 2), s0, g, w0);
            v_words<D>(stage + St::kV + s1 * (D / 2), s1, g, w1);
            lo[half] = __byte_perm(w0[c], w1[c], 0x5410);
            hi[half] = __byte_perm(w0[c], w1[c], 0x7632);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int sh = 8 * (x >> 1);
            uint32_t af[4] = {lo[0] >> sh, hi[0] >> sh, lo[1] >> sh, hi[1] >> sh};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              af[i] = (x & 1) ? codes_hi(af[i]) : codes_lo(af[i]);
              // fp32 calls take the codes less 8: the running sums then have no offset to lose digits to
              if constexpr (PARTS > 1) af[i] = less_8(af[i], x & 1);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int f = 0; f < PARTS; ++f) {
                if (u == 0) mma16816_first(fresh[nt][f][x], af[0], af[1], af[2], af[3], pb[nt][0][f], pb[nt][1][f]);
                else mma16816(fresh[nt][f][x], af[0], af[1], af[2], af[3], pb[nt][0][f], pb[nt][1][f]);
              }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (PARTS > 1) {
            mid[nt][c][0] += fresh_mid[nt][0], mid[nt][c][1] += fresh_mid[nt][1];
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[nt][c][x][i] = fmaf(fresh[nt][0][x][i] + fresh[nt][PARTS - 1][x][i], back[nt][i & 1], o[nt][c][x][i]);
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int i = 0; i < 4; i += 2)
                ptx::unpack2(ptx::add2(ptx::pack2(o[nt][c][x][i], o[nt][c][x][i + 1]),
                                       ptx::pack2(fresh[nt][0][x][i], fresh[nt][0][x][i + 1])),
                             o[nt][c][x][i], o[nt][c][x][i + 1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      const int next = walk.next();
      if (next >= 0) copy.fill(stage, bar + slot, next);
#pragma unroll
      for (int i = 0; i + 1 < kStages; ++i) queue[i] = queue[i + 1];
      queue[kStages - 1] = next;
      if (++slot == kStages) {
        slot = 0;
        phase ^= 1;
      }
    }
    // A wait that ran out: what is still in flight into this CTA's shared memory gets time to land before it is used
    // again or the CTA ends.
    if (stuck) {
#pragma unroll 1
      for (int i = 0; i < kStages; ++i) {
        const int at = (slot + i) % kStages;
        const uint32_t ph = slot + i >= kStages ? phase ^ 1 : phase;
        bool flying = false;
#pragma unroll
        for (int x = 0; x < kStages; ++x) flying |= x == i && queue[x] >= 0;
        for (int spin = 0; spin < 1 << 16 && flying && !ptx::mbar_try_wait(bar + at, ph); ++spin) {
        }
      }
    }

    // join the warps, 8 rows at a time
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], x);
#pragma unroll
          for (int c = 0; c < NG; ++c) mid[nt][c][i] += __shfl_xor_sync(0xffffffffu, mid[nt][c][i], x);
        }
      }
    const int per = a.p.h / a.p.c.hkv;
    float* jo = reinterpret_cast<float*>(smem);  // [warp][8][D]
    float* jm = jo + kWarps * 8 * D;             // [warp][8]
    float* jl = jm + kWarps * 8;
    float* jc = jl + kWarps * 8;  // [8][D + 2]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float* dst = jo + (warp * 8 + 2 * t + i) * D;
#pragma unroll
        for (int c = 0; c < NG; ++c) {
          const float x = mid[nt][c][i], e = kCodeUnit, f = kCodeUnit / 16;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int j = 2 * half + i;
            *reinterpret_cast<float4*>(dst + 64 * c + 8 * g + 4 * half) =
                make_float4(fmaf(e, o[nt][c][0][j], x), fmaf(f, o[nt][c][1][j], x), fmaf(e, o[nt][c][2][j], x), fmaf(f, o[nt][c][3][j], x));
          }
        }
        if (g == 0) {
          jm[warp * 8 + 2 * t + i] = m[nt][i];
          jl[warp * 8 + 2 * t + i] = l[nt][i];
        }
      }
      __syncthreads();
      for (int r = warp; r < 8; r += kWarps) {
        const int row = (w.tile * NT + nt) * 8 + r;
        if (row >= a.rows) continue;
        float top = -INFINITY, f[kWarps], total = 0.f;
#pragma unroll
        for (int x = 0; x < kWarps; ++x) top = fmaxf(top, jm[x * 8 + r]);
#pragma unroll
        for (int x = 0; x < kWarps; ++x) {
          const float pl = jl[x * 8 + r], root = part_root(jm[x * 8 + r], pl, top);
          f[x] = root * root;
          total = fmaf(root, root * pl, total);
        }
        // cut at its start: this CTA's first part, else its second; a cluster's parts stay in its shared memory
        float* part = a.cluster ? jc + r * (D + 2) : a.part + (((int64_t)blockIdx.x * 2 + (w.first == 0)) * NT * 8 + nt * 8 + r) * kPartPitch<D>;
        T* dst = (T*)const_cast<void*>(a.p.out.ptr) + w.b * a.p.out.sb + (int64_t)(row / per) * a.p.out.sl +
                 (int64_t)(w.h * per + row % per) * a.p.out.sh;
#pragma unroll
        for (int c = lane; c < D; c += 32) {
          float x = 0.f;
#pragma unroll
          for (int y = 0; y < kWarps; ++y) x += f[y] * jo[(y * 8 + r) * D + c];
          if (!w.whole) part[c] = x;
          else if constexpr (sizeof(T) == 4) dst[c] = x / total;
          else dst[c] = __float2bfloat16_rn(x / total);
        }
        if (lane == 0) {
          if (!w.whole) {
            part[D] = top;
            part[D + 1] = total;
          } else if (a.p.lse) {
            a.p.lse[((int64_t)w.b * a.p.h + w.h * per + row % per) * a.p.lq + row / per] = top * 0.6931471805599453f + logf(total);
          }
        }
      }
      if (a.cluster > 1) {  // the rows go round the cluster's CTAs, a warp each
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        for (int r = (int)cluster.block_rank() * kWarps + warp; r < 8; r += a.cluster * kWarps) {
          const int row = (w.tile * NT + nt) * 8 + r;
          if (row >= a.rows) continue;
          float top = -INFINITY, total = 0.f, x[D / 32] = {};
          for (int y = 0; y < a.cluster; ++y) top = fmaxf(top, cluster.map_shared_rank(jc, y)[r * (D + 2) + D]);
          for (int y = 0; y < a.cluster; ++y) {
            const float* part = cluster.map_shared_rank(jc, y) + r * (D + 2);
            const float pl = part[D + 1], root = part_root(part[D], pl, top), f = root * root;
            total = fmaf(root, root * pl, total);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) x[c] = fmaf(f, part[lane + 32 * c], x[c]);
          }
          T* dst = (T*)const_cast<void*>(a.p.out.ptr) + w.b * a.p.out.sb + (int64_t)(row / per) * a.p.out.sl +
                   (int64_t)(w.h * per + row % per) * a.p.out.sh;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            if constexpr (sizeof(T) == 4) dst[lane + 32 * c] = x[c] / total;
            else dst[lane + 32 * c] = __float2bfloat16_rn(x[c] / total);
          }
          if (lane == 0 && a.p.lse)
            a.p.lse[((int64_t)w.b * a.p.h + w.h * per + row % per) * a.p.lq + row / per] = top * 0.6931471805599453f + logf(total);
        }
        cluster.sync();  // no CTA writes its parts again, or leaves, while another reads them
      }
    }
    if (a.cluster) return;
  }
}

// Joins the CTAs that shared an item.  The warps of a block, or with many rows (SOLO) each warp alone, have a query row
// and take its parts in turn, four in flight each, a lane D / 32 channels.  What bounds it is the latency of reading the
// parts: up to 592 of a row where there are few rows.
constexpr int kJoinWarps = 8;
constexpr int64_t kSoloRows = 2048;  // rows from which on the GPU is full with a warp a row
template <typename T, int D, bool SOLO>
__global__ void __launch_bounds__(kJoinWarps * 32) cache_join_kernel(const __grid_constant__ AttnArgs a, int tile_rows, int64_t rows) {
  launch_dependents();
  wait_for_launch_before();  // (every block: the kernel after this one counts on it)
  constexpr int V = D / 32, kStep = SOLO ? 1 : kJoinWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t id = SOLO ? (int64_t)blockIdx.x * kJoinWarps + warp : blockIdx.x;
  if (id >= rows) return;
  const int64_t bh = id / a.rows;
  const int row = (int)(id - bh * a.rows);
  const int64_t item = bh * a.tiles + row / tile_rows;
  const int first = a.item[2 * item], last = a.item[2 * item + 1];
  if (!cache_note_holds(first, last, a.ctas)) return;  // (the status word tells; the whole block or warp has the one item)
  const int splits = last - first + 1;
  if (splits == 1) return;
  // the first CTA's second part, the others' first
  const float* part = a.part + ((int64_t)first * 2 * tile_rows + row % tile_rows) * kPartPitch<D>;
  const int64_t step = (int64_t)2 * tile_rows * kPartPitch<D>, second = (int64_t)tile_rows * kPartPitch<D>;
  auto part_of = [&](int i) { return part + (i ? i * step : second); };
  __shared__ float s_top[kJoinWarps], s_sum[kJoinWarps];
  __shared__ __align__(16) float s_out[SOLO ? 1 : kJoinWarps][D];  // (written in pairs)
  float top = -INFINITY;
  for (int i = SOLO ? lane : threadIdx.x; i < splits; i += kStep * 32) top = fmaxf(top, part_of(i)[D]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if constexpr (!SOLO) {
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) top = fmaxf(top, s_top[i]);
  }
  float x[V] = {}, total = 0.f;
#pragma unroll 4
  for (int i = SOLO ? 0 : warp; i < splits; i += kStep) {
    const float* src = part_of(i);
    const float m = src[D], l = src[D + 1];
    float y[V];
#pragma unroll
    for (int j = 0; j < V; j += 2) *reinterpret_cast<float2*>(y + j) = *reinterpret_cast<const float2*>(src + 2 * lane + 32 * j);
    const float root = part_root(m, l, top), f = root * root;
    total = fmaf(root, root * l, total);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = fmaf(f, y[j], x[j]);
  }
  const int per = a.p.h / a.p.c.hkv, b = (int)(bh / a.p.c.hkv), head = (int)(bh % a.p.c.hkv) * per + row % per;
  T* dst = (T*)const_cast<void*>(a.p.out.ptr) + b * a.p.out.sb + (int64_t)(row / per) * a.p.out.sl + (int64_t)head * a.p.out.sh;
  auto put = [&](int c, float y) {
    if constexpr (sizeof(T) == 4) dst[c] = y / total;
    else dst[c] = __float2bfloat16_rn(y / total);
  };
  if constexpr (SOLO) {
#pragma unroll
    for (int j = 0; j < V; ++j) put(2 * lane + 32 * (j & ~1) + (j & 1), x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) *reinterpret_cast<float2*>(&s_out[warp][2 * lane + 32 * j]) = make_float2(x[j], x[j + 1]);
    if (lane == 0) s_sum[warp] = total;
    __syncthreads();
    total = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) total += s_sum[i];
    if (threadIdx.x < D) {
      float y = 0.f;
#pragma unroll
      for (int i = 0; i < kJoinWarps; ++i) y += s_out[i][threadIdx.x];
      put(threadIdx.x, y);
    }
  }
  if ((SOLO ? lane : threadIdx.x) == 0 && a.p.lse)
    a.p.lse[((int64_t)b * a.p.h + head) * a.p.lq + row / per] = top * 0.6931471805599453f + logf(total);
}

// weights_out = weight + the sum over the query rows of exp(s - L): the scores are formed again from the keys, now that
// every row's L is known.  With few tiles of 8 rows a warp has units of keys to itself and takes the rows in a fixed order
// (a tile alone is loaded once); from kSplitFrom tiles on the warps of a CTA divide the tiles, each goes over all kGroup
// units that the CTA holds, and their sums are added in the order of the warps.  The next units are on their way
// meanwhile.  Under a mask, units that no row sees are found by their positions and not fetched.
// It reads half the cache and forms 64 scores a key; what bounds it is waiting for its own loads (5.4 cycles an instruction with 18
// warps an SM; 45 % of issue slots are used): 8 x 32768 keys of 8 heads, 4 rows each, 51 us (168 MB).  Divided / not, us of the pass: 8 x 8 heads of 4096 keys, 16 rows (2 tiles) 16 / 19, 24
// rows 18 / 26, 256 rows 116 / 200, 4 x 8 heads of 16384, d 64, 16 rows 22 / 20, 24 rows 25 / 27; 4 heads of 2048 keys, 256 rows 10 / 104 (a tile's loading is 2 us that nothing hides).
constexpr int kSplitFrom = 3;
template <int D>
struct WeightsShape {
  using St = Stage<D, false>;
  static constexpr int kRing = 2 * kWarps * St::kBytes, kUsed = kRing + 2 * kWarps * 8, kSums = kUsed + 2 * kWarps * 4 + 16;
  static constexpr int kMostWarps = D == 256 ? 8 : 16;  // of a CTA that divides tiles: with few keys more of them, for one tile each
};

// What of the keys the rows of a sequence can see by their positions: lo < position <= hi.
struct SeenRange {
  long long lo = LLONG_MIN, hi = LLONG_MAX;
  __device__ void init(const AttnArgs& a, int b, int lane) {
    int least = INT_MAX, most = INT_MIN;
    for (int i = lane; i < a.p.lq; i += 32) {
      const int p = a.p.q_pos ? a.p.q_pos[(int64_t)b * a.p.lq + i] : a.p.c.seen[b] - a.p.lq + i;
      least = min(least, p), most = max(most, p);
    }
    least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
    if (a.p.kinds & RA_MOD_CAUSAL) hi = most;
    if (a.p.kinds & RA_MOD_WINDOW) lo = (long long)least - a.p.window;
  }
  // Whether a row may see a key of the unit; if none does, the unit's weights are passed on as they are.
  __device__ bool seen_or_passed_on(const AttnArgs& a, int64_t bh, int unit, int len, int lane) const {
    const int64_t at = bh * a.p.c.cap + (int64_t)unit * kCacheUnit;
    bool use = false;
#pragma unroll
    for (int j = 0; j < kCacheUnit; j += 32) {
      const bool live = unit * kCacheUnit + j + lane < len;
      const int p = live ? a.p.c.pos[at + j + lane] : 0;
      use |= live && p > lo && p <= hi;
    }
    if (__any_sync(0xffffffffu, use)) return true;
#pragma unroll
    for (int j = 0; j < kCacheUnit; j += 32)
      if (unit * kCacheUnit + j + lane < len && a.p.weights_out != a.p.c.weight) a.p.weights_out[at + j + lane] = a.p.c.weight[at + j + lane];
    return false;
  }
};

// The logarithms (base 2) of the rows 2t, 2t + 1 of a tile.
__device__ __forceinline__ void row_logs(const AttnArgs& a, int b, int h, int tile, int t, float lse2[2]) {
  const int per = a.p.h / a.p.c.hkv;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = tile * 8 + 2 * t + i;
    // a row that is not there, or sees nothing, weighs nothing
    lse2[i] = row < a.rows ? a.p.lse[((int64_t)b * a.p.h + h * per + row % per) * a.p.lq + row / per] * 1.4426950408889634f : INFINITY;
    if (lse2[i] == -INFINITY) lse2[i] = INFINITY;
  }
}
// sum[u][half] += exp(s - L) over the rows of a tile that this lane holds, key (half, g) of sub-unit u.
template <int D, bool MASKED, int PARTS>
__device__ __forceinline__ void add_weights(const AttnArgs& a, const char* stage, int live_keys, const QueryTile<D, 1, PARTS>& q,
                                            const float lse2[2], float sum[kSub][2]) {
  using St = Stage<D, false>;
#pragma unroll
  for (int u = 0; u < kSub; ++u) {
    float s[1][4];
    scores16<D, 1, PARTS>(stage, St::kKl, u, q, s);
    if (MASKED || live_keys < kCacheUnit) mod16<MASKED, D, 1, PARTS>(a, stage, St::kPos, u, live_keys, q, s);
#pragma unroll
    for (int half = 0; half < 2; ++half)
      sum[u][half] += ptx::ex2(finish<MASKED>(s[0][2 * half], q.factor[0][0], -lse2[0])) +
                      ptx::ex2(finish<MASKED>(s[0][2 * half + 1], q.factor[0][1], -lse2[1]));
  }
}

// For the copies of a stage that nothing waited for to the end.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  for (int spin = 0; spin < 1 << 16 && !ptx::mbar_try_wait(bar, parity); ++spin) {
  }
}

template <typename T, int D, bool MASKED, bool SPLIT>
__global__ void __launch_bounds__((SPLIT ? WeightsShape<D>::kMostWarps : kWarps) * 32, SPLIT ? 1 : D == 256 ? 3 : sizeof(T) == 4 ? 4 : 5)
    cache_weights_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int PARTS = sizeof(T) == 4 ? 2 : 1, kGroup = D == 256 || PARTS == 2 ? 2 : 4;
  using St = Stage<D, false>;
  using Shape = WeightsShape<D>;
  extern __shared__ __align__(128) char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Shape::kRing);
  float* sums = reinterpret_cast<float*>(smem + Shape::kSums);
  int* used = reinterpret_cast<int*>(smem + Shape::kUsed);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(smem + Shape::kUsed + 2 * kWarps * 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) *s_abort = 0;
  if (threadIdx.x < 2 * kWarps) {
    ptx::mbar_init(bars + threadIdx.x, St::kCopies + (MASKED ? 1 : 0));
    ptx::fence_barrier_init();
  }
  __syncthreads();
  wait_for_launch_before();
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.p.c.hkv), h = (int)(bh % a.p.c.hkv);
  const int len = min(max(a.p.c.len[b], 0), a.p.c.cap), units = (len + kCacheUnit - 1) / kCacheUnit;
  const int tiles = (a.rows + 7) / 8, warps = blockDim.x >> 5;
  St copy;
  copy.init(a.p.c, bh, MASKED);
  SeenRange range;
  if constexpr (MASKED) range.init(a, b, lane);
  uint32_t phase = 0;  // bit i: of barrier i, stage i of the ring
  QueryTile<D, 1, PARTS> q;
  float lse2[2];

  if constexpr (SPLIT) {
    const int group = a.weights_group, groups = (units + group - 1) / group;
    auto fetch = [&](int i, int buf) {  // the copies of group i into half `buf` of the ring, a warp a unit
      const int unit = i * group + warp;
      if (warp >= group) return;
      bool use = unit < units;
      if constexpr (MASKED)
        if (use) use = range.seen_or_passed_on(a, bh, unit, len, lane);
      if (use) copy.fill(smem + (buf * kWarps + warp) * St::kBytes, bars + buf * kWarps + warp, unit);
      if (lane == 0) used[buf * kWarps + warp] = use;
    };
    if ((int)blockIdx.y < groups) fetch(blockIdx.y, 0);
    __syncthreads();
    int buf = 0;
#pragma unroll 1
    for (int i = blockIdx.y; i < groups; i += gridDim.y, buf ^= 1) {
      const int next = i + gridDim.y;
      if (next < groups) fetch(next, buf ^ 1);
      uint32_t mine = 0;  // bit x: unit x of the group is to be read
      bool bad = false;
      for (int x = 0; x < group; ++x) {
        if (!used[buf * kWarps + x]) continue;
        const int at = buf * kWarps + x;
        mine |= 1u << x;
        if (!ptx::mbar_wait(bars + at, phase >> at & 1, s_abort, a.status, kStCacheWait)) bad = true;
        phase ^= 1u << at;
      }
      if (__syncthreads_or(bad)) {  // nothing is written for these keys; a warp waits for the copies that it began
        if (warp < group) {
          if (mine >> warp & 1) drain(bars + buf * kWarps + warp, (phase >> (buf * kWarps + warp) & 1) ^ 1);
          if (next < groups && used[(buf ^ 1) * kWarps + warp]) drain(bars + (buf ^ 1) * kWarps + warp, phase >> ((buf ^ 1) * kWarps + warp) & 1);
        }
        return;
      }
      float sum[kGroup][kSub][2] = {};
      if (mine) {
#pragma unroll 1
        for (int tile = warp; tile < tiles; tile += warps) {
          q.template load<T>(a, b, h, tile);
          row_logs(a, b, h, tile, t, lse2);
#pragma unroll
          for (int x = 0; x < kGroup; ++x)
            if (mine >> x & 1)
              add_weights<D, MASKED, PARTS>(a, smem + (buf * kWarps + x) * St::kBytes, len - (i * group + x) * kCacheUnit, q, lse2, sum[x]);
        }
      }
#pragma unroll
      for (int x = 0; x < kGroup; ++x)
        if (mine >> x & 1)
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float y = sum[x][u][half];
              y += __shfl_xor_sync(0xffffffffu, y, 1);
              y += __shfl_xor_sync(0xffffffffu, y, 2);
              if (t == 0) sums[(warp * kGroup + x) * kCacheUnit + 16 * u + 8 * half + cache_kappa(g)] = y;
            }
      __syncthreads();  // the sums are there, and every warp has read the stages
      for (int j = threadIdx.x; j < group * kCacheUnit; j += blockDim.x) {
        const int key = i * group * kCacheUnit + j;
        if (!(mine >> j / kCacheUnit & 1) || key >= len) continue;
        float y = 0.f;
        for (int w = 0; w < warps; ++w) y += sums[w * kGroup * kCacheUnit + j];
        a.p.weights_out[bh * a.p.c.cap + key] = a.p.c.weight[bh * a.p.c.cap + key] + y;
      }
      __syncthreads();
    }
  } else {
    char* ring = smem + warp * 2 * St::kBytes;
    uint64_t* bar = bars + warp * 2;
    if (tiles == 1) q.template load<T>(a, b, h, 0), row_logs(a, b, h, 0, t, lse2);
    const int stride = gridDim.y * kWarps;
    auto seek = [&](int unit) {  // the next unit of this warp from `unit` on that is to be read
      if constexpr (MASKED)
        while (unit < units && !range.seen_or_passed_on(a, bh, unit, len, lane)) unit += stride;
      return unit;
    };
    int unit = seek(blockIdx.y * kWarps + warp), slot = 0;
    if (unit < units) copy.fill(ring, bar, unit);
#pragma unroll 1
    while (unit < units) {
      const int next = seek(unit + stride);
      if (next < units) copy.fill(ring + (slot ^ 1) * St::kBytes, bar + (slot ^ 1), next);
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(bar + slot, phase >> slot & 1, s_abort, a.status, kStCacheWait))) {
        drain(bar + slot, phase >> slot & 1);
        if (next < units) drain(bar + (slot ^ 1), phase >> (slot ^ 1) & 1);
        return;  // nothing is written for these keys
      }
      phase ^= 1u << slot;
      const char* stage = ring + slot * St::kBytes;
      const int live_keys = len - unit * kCacheUnit;
      float sum[kSub][2] = {};
      for (int tile = 0; tile < tiles; ++tile) {
        if (tiles > 1) q.template load<T>(a, b, h, tile), row_logs(a, b, h, tile, t, lse2);
        add_weights<D, MASKED, PARTS>(a, stage, live_keys, q, lse2, sum);
      }
      __syncwarp();  // every lane has read the stage
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = sum[u][half];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          const int key = 16 * u + 8 * half + cache_kappa(g);
          const int64_t at = bh * a.p.c.cap + (int64_t)unit * kCacheUnit + key;
          if (t == 0 && key < live_keys) a.p.weights_out[at] = a.p.c.weight[at] + x;
        }
      unit = next;
      slot ^= 1;
    }
  }
}

int sm_count() {
  static int known[64] = {};
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess) return n;
  if (dev < 64 && known[dev]) return known[dev];
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && dev < 64) known[dev] = n;
  return n;
}

// When the matrix form (cache4_prompt.cu) is taken: from this many query rows of a key/value head on, if the caches' capacity
// times the 16-row tiles is at least this many keys.  It reads the cache once for 128 rows and not once for 16, but its
// CTAs take longer to start.  All rules here go by the capacity, since the lengths are on the device and a captured call has to
// stay right while the cache grows; they were measured with full caches, and one that holds little of its capacity takes the
// form of a full one.  Graph replays, us, this form / that one:
//   8 x 8 heads, 4096 keys, d 128: 32 rows 34 / 49, 64 rows 52 / 50, 256 rows 183 / 90;  d 256: 32 rows 87 / 112, 64 rows
//   172 / 116, 256 rows 601 / 218
//   4 heads, 16384 keys, d 128: 32 rows 20 / 27, 64 rows 29 / 28;  d 256: 48 rows 44 / 42, 64 rows 52 / 43
//   4 x 8 heads, 16384 keys, d 64: 48 rows 52 / 56, 64 rows 60 / 55
//   by keys times tiles, d 128: 65536 (4 heads, 2048 keys, 128 rows) 12 / 22, 262144 (4096 keys, 256 rows) 24 / 24, 655360
//   (640 rows) 52 / 38;  d 64: 65536 (2 heads, 8192 keys, 64 rows) 13 / 15, 131072 (128 rows) 21 / 16
constexpr int kPromptFrom = 64;
constexpr int64_t kPromptKeys = 3 << 16;

// Query rows of a tile: 8 NT.  16 read the cache half as often as 8, but the kernel is the longer one to start, has fewer
// warps an SM, and an odd number of 8-row tiles leaves half of its last one empty.  d 128, us of 8 / 16 rows, by keys (of the
// capacity) times 8-row tiles:  16 rows 2^16 (8 heads of 4096 keys) 12 / 16, 2^18 (4 x 8 heads) 16 / 19, 2^19 (8 x 8 heads) 24
// / 24, 2^20 (8 heads of 65536 keys) 43 / 33;  24 rows 2^18.6 (4 x 8 heads of 4096 keys) 21 / 24, 2^21.6 (8 x 8 heads of 16384
// keys) 101 / 99, under a mask 128 / 152;  40 rows under a mask, 8 x 8 heads of 4096 keys 66 / 74.  d 64:  16 rows 2^15 (8
// heads of 2048 keys) 8 / 11, 24 rows 2^19.6 (8 x 8 heads of 4096 keys) 27 / 32 under a mask, 40 rows 45 / 40, 64 rows 2^17 (2
// heads of 8192 keys) 15 / 13.
int tile_parts(int64_t keys, int rows, int d, int dtype, bool masked) {
  const int eights = (rows + 7) / 8;
  if (dtype == RA_DTYPE_F32 || d == 256) return 1;  // what the registers hold
  const bool many = d == 64 && eights > 4;
  return eights > 1 && keys * eights >= (many ? 1 << 17 : 1 << 19) && !(masked && eights % 2 && !many) ? 2 : 1;
}

// Blocks of a kernel that fit on an SM, looked up once a device.  `most`: the largest shared memory that any call of the
// kernel asks for (the attribute outlasts the call, and other threads launch by it).
template <typename K>
cudaError_t blocks_per_sm(K kernel, int threads, int smem, int most, int* n) {
  struct Known {
    const void* kernel;
    int dev, threads, n;
  };
  static thread_local Known known[8] = {};  // (kernels of one signature share this function)
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const void* id = reinterpret_cast<const void*>(kernel);
  for (const Known& k : known)
    if (k.kernel == id && k.dev == dev && k.threads == threads) {
      *n = k.n;
      return cudaSuccess;
    }
  if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) != cudaSuccess) return e;
  if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kernel, threads, smem)) != cudaSuccess) return e;
  if (*n < 1) return cudaErrorInvalidConfiguration;
  static thread_local int at = 0;
  known[at++ % 8] = Known{id, dev, threads, *n};
  return cudaSuccess;
}

// f(type tag, head dim, NT, whether masked) of a call
template <typename F>
auto by_shape(int dtype, int d, int nt, bool masked, F f) {
  auto by_mask = [&](auto tag, auto dim, auto rows) {
    return masked ? f(tag, dim, rows, std::true_type{}) : f(tag, dim, rows, std::false_type{});
  };
  auto by_nt = [&](auto tag, auto dim) {
    if constexpr (sizeof(tag) == 2 && decltype(dim)::value != 256)
      if (nt == 2) return by_mask(tag, dim, std::integral_constant<int, 2>{});
    return by_mask(tag, dim, std::integral_constant<int, 1>{});
  };
  auto by_dim = [&](auto tag) {
    if (d == 64) return by_nt(tag, std::integral_constant<int, 64>{});
    if (d == 128) return by_nt(tag, std::integral_constant<int, 128>{});
    return by_nt(tag, std::integral_constant<int, 256>{});
  };
  return dtype == RA_DTYPE_F32 ? by_dim(float{}) : by_dim(__nv_bfloat16{});
}

struct Plan {
  cudaError_t err;
  bool prompt;
  int nt, rows, tiles, cluster, ctas;
  size_t part, item, lse, total;
};
Plan make_plan(int b, int hkv, int cap, int d, int h, int lq, int dtype, bool masked) {
  Plan p;
  p.rows = h / hkv * lq;
  const int units = cap / kCacheUnit;
  int per_sm = 1, tile_rows = kPromptRows;
  p.prompt = dtype == RA_DTYPE_BF16 && p.rows >= kPromptFrom &&
             (int64_t)b * hkv * cap * ((p.rows + 15) / 16) >= kPromptKeys;
  if (p.prompt) {
    p.err = cache_prompt_prepare(d, masked);
    per_sm = d == 256 ? kPromptPerSm<256> : kPromptPerSm<128>;
  } else {
    p.nt = tile_parts((int64_t)b * hkv * cap, p.rows, d, dtype, masked);
    tile_rows = 8 * p.nt;
    p.err = by_shape(dtype, d, p.nt, masked, [&](auto tag, auto dim, auto nt, auto mask) {
      return blocks_per_sm(cache_attn_kernel<decltype(tag), decltype(dim)::value, decltype(nt)::value, decltype(mask)::value>, kWarps * 32,
                         AttnShape<decltype(dim)::value>::kSmem, AttnShape<decltype(dim)::value>::kSmem, &per_sm);
    });
  }
  p.tiles = (p.rows + tile_rows - 1) / tile_rows;
  const int slots = per_sm * sm_count();
  const int64_t items = (int64_t)b * hkv * p.tiles;
  // A short cache is divided as far as all items still fit on the GPU at once and its warps have a unit each.  Clusters of 8
  // leave SMs of a GPC over: 16 of them are 128 CTAs, but at one CTA an SM they ran in two waves (2 heads of 2048 keys, d 256,
  // 64 rows: 23 us, in clusters of 4 13).
  p.cluster = 0;
  if (units <= kShortUnits && !p.prompt)
    for (p.cluster = 1; p.cluster < 8 && 2 * p.cluster * items <= (p.cluster == 4 ? slots * 4 / 5 : slots) && p.cluster * kWarps < units;)
      p.cluster *= 2;
  // (cuts count up to kItemCost + kSpread - 1 units more for an item)
  const int64_t most = p.cluster ? items * p.cluster : (items * (units + kItemCost + kSpread) + kMinUnits - 1) / kMinUnits;
  p.ctas = (int)(p.cluster || most < slots ? most : slots);
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  p.part = 0;
  p.item = p.cluster ? 0 : up((size_t)p.ctas * 2 * tile_rows * (d + 4) * 4);
  p.lse = p.item + (p.cluster ? 0 : up(items * 8));
  p.total = p.lse + up((size_t)b * h * lq * 4);
  return p;
}

// Launches a kernel whose blocks may start while the one before is ending.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

template <typename T, int D, int NT, bool MASKED>
cudaError_t run_rows(const AttnArgs& a, cudaStream_t s) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.ctas);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = AttnShape<D>::kSmem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, cache_attn_kernel<T, D, NT, MASKED>, a);
}

// What follows either form: the joining of what was cut, and the sums of probabilities.
template <typename T, int D, bool MASKED>
cudaError_t run_after(AttnArgs a, int tile_rows, cudaStream_t s) {
  cudaError_t e;
  if (!a.cluster) {
    const int64_t rows = (int64_t)a.p.c.b * a.p.c.hkv * a.rows;
    e = rows >= kSoloRows
            ? launch_after(cache_join_kernel<T, D, true>, dim3((unsigned)((rows + kJoinWarps - 1) / kJoinWarps)), kJoinWarps * 32, 0, s, a, tile_rows, rows)
            : launch_after(cache_join_kernel<T, D, false>, dim3((unsigned)rows), kJoinWarps * 32, 0, s, a, tile_rows, rows);
    if (e != cudaSuccess) return e;
    count_launch();
  }
  if (a.p.weights_out) {
    const int bh = a.p.c.b * a.p.c.hkv, units = a.p.c.cap / kCacheUnit;
    using Shape = WeightsShape<D>;
    constexpr int kGroup = D == 256 || sizeof(T) == 4 ? 2 : 4;
    const int tiles = (a.rows + 7) / 8, sms = sm_count();
    const bool split = tiles >= kSplitFrom;
    auto kernel = split ? cache_weights_kernel<T, D, MASKED, true> : cache_weights_kernel<T, D, MASKED, false>;
    int warps = kWarps, smem = Shape::kSums, per_sm = 1;
    a.weights_group = kWarps;  // units a CTA holds at a time
    if (split) {  // several where that leaves no SM without one, then more warps where an SM has few
      a.weights_group = kGroup;
      auto ctas = [&] { return (int64_t)bh * ((units + a.weights_group - 1) / a.weights_group); };
      while (a.weights_group > 1 && ctas() < sms) a.weights_group /= 2;
      while (warps < Shape::kMostWarps && 2 * warps <= tiles && ctas() * warps < 16 * sms) warps *= 2;
      smem += warps * kGroup * kCacheUnit * 4;
    }
    if ((e = blocks_per_sm(kernel, warps * 32, smem, Shape::kSums + Shape::kMostWarps * kGroup * kCacheUnit * 4, &per_sm)) != cudaSuccess) return e;
    const int want = per_sm * sms / bh > 1 ? per_sm * sms / bh : 1;  // CTAs a (sequence, head) that make a wave
    int y = (units + a.weights_group - 1) / a.weights_group;
    if (y > want) y = want;
    if (y > 65535) y = 65535;
    if ((e = launch_after(kernel, dim3(bh, y), warps * 32, smem, s, a)) != cudaSuccess) return e;
    count_launch();
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t cache_attn_workspace(int b, int hkv, int cap, int d, int h, int lq, int dtype, size_t* bytes) {
  // the larger of the two forms' needs: they differ in how many CTAs fit on an SM
  const Plan p = make_plan(b, hkv, cap, d, h, lq, dtype, false), m = make_plan(b, hkv, cap, d, h, lq, dtype, true);
  *bytes = p.total > m.total ? p.total : m.total;
  return p.err != cudaSuccess ? p.err : m.err;
}

cudaError_t launch_cache_attn(const CacheAttnParams& p, cudaStream_t s) {
  AttnArgs a;
  a.p = p;
  const Plan plan = make_plan(p.c.b, p.c.hkv, p.c.cap, p.c.d, p.h, p.lq, p.dtype, p.kinds != 0);
  if (plan.err != cudaSuccess) return plan.err;
  const int es = p.dtype == RA_DTYPE_F32 ? 4 : 2;
  a.rows = plan.rows;
  a.tiles = plan.tiles;
  a.cluster = plan.cluster;
  a.vec_out = reinterpret_cast<uintptr_t>(p.out.ptr) % 16 == 0 && p.out.sb * es % 16 == 0 && p.out.sl * es % 16 == 0 && p.out.sh * es % 16 == 0;
  a.ctas = plan.ctas;
  a.vec = reinterpret_cast<uintptr_t>(p.q.ptr) % 16 == 0 && p.q.sb * es % 16 == 0 && p.q.sl * es % 16 == 0 && p.q.sh * es % 16 == 0;
  a.wide = (reinterpret_cast<uintptr_t>(p.c.k) | reinterpret_cast<uintptr_t>(p.c.v)) % 32 == 0;
  char* ws = (char*)p.ws;
  a.part = (float*)(ws + plan.part);
  a.item = (int32_t*)(ws + plan.item);
  if (!a.p.lse) a.p.lse = (float*)(ws + plan.lse);
  a.status = device_status_word();
  if (!a.status) return cudaErrorInvalidSymbol;
  cudaError_t e = plan.prompt ? launch_cache_prompt(a, s)
                              : by_shape(p.dtype, p.c.d, plan.nt, p.kinds != 0, [&](auto tag, auto dim, auto nt, auto mask) {
                                  return run_rows<decltype(tag), decltype(dim)::value, decltype(nt)::value, decltype(mask)::value>(a, s);
                                });
  if (e != cudaSuccess) return e;
  count_launch();
  return by_shape(p.dtype, p.c.d, 1, p.kinds != 0, [&](auto tag, auto dim, auto, auto mask) {
    return run_after<decltype(tag), decltype(dim)::value, decltype(mask)::value>(a, plan.prompt ? kPromptRows : 8 * plan.nt, s);
  });
}

}  // namespace ra
