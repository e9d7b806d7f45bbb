// Filling, reading and evicting the 4-bit key/value cache (layout and code formula: cache4_layout.h).
#include <cooperative_groups.h>

#include <cfloat>
#include <climits>
#include <type_traits>

#include "cache4.cuh"
#include "tc_common.cuh"

namespace ra {
namespace {

// ---- append ------------------------------------------------------------------------------------------
__device__ __forceinline__ void load8(const float* p, bool vec, float (&x)[8]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ void store8(float* p, bool vec, const float (&x)[8]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, bool vec, const float (&x)[8]) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = make_uint4(ptx::pack_bf16(x[0], x[1]), ptx::pack_bf16(x[2], x[3]), ptx::pack_bf16(x[4], x[5]),
                                              ptx::pack_bf16(x[6], x[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(x[i]);
  }
}

// bf16 at or below x, as a float.
__device__ __forceinline__ float bf16_down(float x) {
  const uint32_t u = __float_as_uint(x), cut = u & 0xffff0000u;
  return __uint_as_float((u >> 31) && cut != u ? cut + 0x10000u : cut);
}
// bf16 at or above (hi - mn) / 15, formed in 64 bits.
__device__ __noinline__ float step_in_64_bits(float hi, float mn) {
  const float up = __double2float_ru(((double)hi - (double)mn) / 15.0);
  return __uint_as_float((__float_as_uint(up) + 0xffffu) & 0xffff0000u);
}
// The same; the fp32 quotient is off by less than 4 units of its last place, and where that leaves open which bf16
// value is next (or the quotient is out of the normal range) it goes the long way.
__device__ __forceinline__ float step_of(float hi, float mn) {
  const float q = (hi - mn) * (1.f / 15.f);
  const uint32_t u = __float_as_uint(q), low = u & 0xffffu;
  if (low - 8u < 0xfff0u && q > 1e-30f && q < 1e38f) return __uint_as_float((u & 0xffff0000u) + 0x10000u);
  return step_in_64_bits(hi, mn);
}

// Smallest and largest that are NaN where an operand is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float c;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
// Smallest and largest of the 64 channels that the lanes of an octet hold, 8 each.  bf16 channels stay packed: the pair
// (largest, -smallest) takes one shuffle a step.
__device__ __forceinline__ unsigned int octet_mask() { return 0xffu << (threadIdx.x & 24); }
__device__ __forceinline__ void octet_limits(const float (&x)[8], float& lo, float& hi) {
  lo = min_nan(min_nan(min_nan(x[0], x[1]), min_nan(x[2], x[3])), min_nan(min_nan(x[4], x[5]), min_nan(x[6], x[7])));
  hi = max_nan(max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3])), max_nan(max_nan(x[4], x[5]), max_nan(x[6], x[7])));
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(octet_mask(), lo, s));
    hi = max_nan(hi, __shfl_xor_sync(octet_mask(), hi, s));
  }
}
__device__ __forceinline__ void octet_limits(const uint4& raw, float& lo, float& hi) {
  const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&raw);
  const __nv_bfloat162 mn = __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3]));
  const __nv_bfloat162 mx = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
  __nv_bfloat162 m = __hmax2_nan(__lows2bfloat162(mx, __hneg2(mn)), __highs2bfloat162(mx, __hneg2(mn)));
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) m = __hmax2_nan(m, __shfl_xor_sync(octet_mask(), m, s));
  hi = __low2float(m);
  lo = -__high2float(m);
}

// Word of codes where a difference or the step's reciprocal is beyond fp32.
__device__ __noinline__ uint32_t codes_in_64_bits(const float* x, float mn, float step) {
  uint32_t w = 0;
  for (int i = 0; i < 8; ++i) w |= (uint32_t)rint(((double)x[i] - (double)mn) / (double)step) << (4 * i);
  return w;
}

// The codes of this lane's 8 channels, and the group's limits from its smallest and largest channel.  Rounding is the
// addition of 1.5 * 2^23 and packing is by fused products (conversions run at an eighth of their rate).  The level is
// decided as in exact arithmetic: the fp32 quotient is off by less than 4e-6 of a level (15 * 3 * 2^-24), and where it
// lies that near to the middle of two the remainder decides: a - n step is
// exact, as is the part `rest` of x - mn that rounding took from a, so that the sign of their sum is right.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float lo, float hi, uint32_t& limits) {
  const float mn = bf16_down(lo), step = step_of(hi, mn);
  if (!(hi <= FLT_MAX) || !(fabsf(mn) <= FLT_MAX) || !(step <= FLT_MAX)) {
    limits = 0x7fc07fc0u;
    return 0;
  }
  limits = (__float_as_uint(step) >> 16) | (__float_as_uint(mn) & 0xffff0000u);
  if (!(step > 0.f)) return 0;
  float inv;  // (off by one unit of its last place)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
  const float magic = 12582912.f;
  if (!(inv <= FLT_MAX) || !(hi - mn <= FLT_MAX)) {
    const float y[8] = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
    return codes_in_64_bits(y, mn, step);
  }
  float n[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {  // (two share a branch)
    float d[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float a = x[i + j] - mn;
      n[i + j] = fmaf(a, inv, magic) - magic;
      d[j] = fabsf(fmaf(a, inv, -n[i + j]));
    }
    if (fmaxf(d[0], d[1]) >= 0.499996f) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float a = x[i + j] - mn, back = a - x[i + j], rest = (x[i + j] - (a - back)) + (-mn - back);
        const float rem = fmaf(-n[i + j], step, a), past = (fabsf(rem) - 0.5f * step) + (rem < 0.f ? -rest : rest);
        if (past > 0.f || (past == 0.f && (__float_as_uint(n[i + j] + magic) & 1u))) n[i + j] += copysignf(1.f, rem);
      }
    }
  }
  const float w0 = fmaf(n[3], 4096.f, fmaf(n[2], 256.f, fmaf(n[1], 16.f, n[0])));
  const float w1 = fmaf(n[7], 4096.f, fmaf(n[6], 256.f, fmaf(n[5], 16.f, n[4])));
  return __byte_perm(__float_as_uint(w0 + 8388608.f), __float_as_uint(w1 + 8388608.f), 0x5410);
}

// A lane's 8 channels of a group as they are in memory, and the word of their codes.
struct Eight {
  float x[8];
};
__device__ __forceinline__ Eight load_group(const float* p, bool vec) {
  Eight r;
  load8(p, vec, r.x);
  return r;
}
__device__ __forceinline__ uint4 load_group(const __nv_bfloat16* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint4 raw;
  __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = p[i];
  return raw;
}
__device__ __forceinline__ uint32_t quantise_group(const Eight& r, uint32_t& limits) {
  float lo, hi;
  octet_limits(r.x, lo, hi);
  return quantise8(r.x, lo, hi, limits);
}

__device__ __noinline__ uint2 quantise_any_bf16(uint4 raw, float lo, float hi) {  // {codes, limits}
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  uint2 r;
  r.x = quantise8(x, lo, hi, r.y);
  return r;
}
// bf16 channels.  Where the smallest channel's exponent is at most 16 below the range's, all differences a = x - min are
// exact in fp32 (the last bit of a bf16 number is 7 below its exponent, that of a difference 23 at most), and the level
// needs no case for the middle of two: q = a / step is refined by its exact remainder, comes out as the middle exactly if
// it is there (13 bits) and on the right side if not (24 bits of a keep it 2^-24 away), and is then rounded to even.  The
// step, too, follows from the sign of an exact remainder.  Other groups go the general way.
__device__ __forceinline__ uint32_t quantise_group(const uint4& raw, uint32_t& limits) {
  float lo, hi;
  octet_limits(raw, lo, hi);
  const __nv_bfloat162* w = reinterpret_cast<const __nv_bfloat162*>(&raw);
  const __nv_bfloat162 abs2 = __hmin2(__hmin2(__habs2(w[0]), __habs2(w[1])), __hmin2(__habs2(w[2]), __habs2(w[3])));
  const float least = fminf(fminf(__low2float(abs2), __high2float(abs2)), fminf(fabsf(lo), fabsf(hi))), range = hi - lo;
  const float floor16 = __uint_as_float((__float_as_uint(range) & 0x7f800000u) - (16u << 23));
  if (!(least >= floor16 && range >= 1e-26f && range <= 1e37f)) {  // (NaN and infinity, too)
    const uint2 r = quantise_any_bf16(raw, lo, hi);
    limits = r.y;
    return r.x;
  }
  const uint32_t near = (__float_as_uint(range * (1.f / 15.f)) + 0x8000u) & 0xffff0000u;
  const uint32_t up = near + (fmaf(__uint_as_float(near), -15.f, range) > 0.f ? 0x10000u : 0u);
  const float step = __uint_as_float(up);
  limits = up >> 16 | (__float_as_uint(lo) & 0xffff0000u);
  float inv;  // (off by one unit of its last place)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
  const uint64_t mn2 = ptx::pack2(-lo, -lo), inv2 = ptx::pack2(inv, inv), step2 = ptx::pack2(-step, -step), magic2 = ptx::pack2(12582912.f, 12582912.f);
  const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t codes = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const uint64_t a = ptx::add2(ptx::pack2(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xffff0000u)), mn2);
    const uint64_t q = ptx::mul2(a, inv2);
    const uint64_t n = ptx::add2(ptx::fma2(ptx::fma2(q, step2, a), inv2, q), magic2);
    codes = (((codes << 4) + (uint32_t)(n >> 32)) << 4) + (uint32_t)n;
  }
  // each number above came with 0x4b400000, the bits of 1.5 * 2^23
  constexpr uint32_t kBits = 0x4b400000u * 0x11111111u;
  return codes - kBits;
}

struct AppendParams {
  CacheView c;
  TensorView k, v;
  const int32_t *counts, *start, *positions;
  int32_t t, vec;
  unsigned int* status;
};

// Accesses to a position that several blocks may make at once.
__device__ __forceinline__ int load_relaxed(const int32_t* p) {
  int x;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(x) : "l"(p) : "memory");
  return x;
}
__device__ __forceinline__ void store_relaxed(int32_t* p, int x) { asm volatile("st.relaxed.gpu.global.s32 [%0], %1;" ::"l"(p), "r"(x) : "memory"); }

struct AppendSpan {
  int at, count, pos;  // first slot, rows, default position of the first row
};
// Where rows are dropped, the first of them had the position to go on from, unless the row before it went further (branches of
// drafts: 10, 11, 11, of which two stay).  Rows that eviction has moved lie earlier, and all heads hold the same last rows.
// Another block, or the counters below, may find the position in place of the dropped row's that is formed here, which gives
// the same again.  (Or one of the caller's; then this one stands for no row and no counter.)
__device__ __forceinline__ AppendSpan append_span(const AppendParams& p, int b) {
  const int len = min(max(p.c.len[b], 0), p.c.cap);
  AppendSpan s;
  s.at = p.start ? min(max(p.start[b], 0), len) : len;
  s.count = p.counts ? min(max(p.counts[b], 0), p.t) : p.t;
  s.pos = p.c.seen[b];
  if (s.at < len) {
    const int32_t* pos = p.c.pos + (int64_t)b * p.c.hkv * p.c.cap;
    s.pos = load_relaxed(pos + s.at);
    if (s.at > 0) s.pos = max(s.pos, load_relaxed(pos + s.at - 1) + 1);
  }
  return s;
}
// The counters after the rows are there: one thread a sequence.
__device__ __forceinline__ void append_counters(const AppendParams& p, int b, const AppendSpan& s) {
  const int n = min(s.count, p.c.cap - s.at);
  if (n < s.count) atomicOr(p.status, kStCacheFull);
  p.c.len[b] = s.at + n;
  p.c.seen[b] = p.positions && n > 0 ? p.positions[(int64_t)b * p.t + n - 1] + 1 : s.pos + n;
}

// A block takes kRowTile tokens of a sequence.  An octet of lanes has one group of 64 channels of K and of V and walks
// down the tokens: reads run along a token's heads, and the rows of a head that the block writes are neighbours in the
// cache.  Issue slots bound it (76 % used; 160 instructions for a lane's 8 channels, loads and stores with them): 2 x 32768
// tokens of 16 heads, 128 channels, bf16, 694 MB in 210 us, 3.3 TB/s, where 106 us would be a copy's; 304 us before the
// bf16 form above of deciding levels.
constexpr int kRowThreads = 256, kOctets = kRowThreads / 8, kRowTile = 16;
struct OctetWalk {
  int across, first_group, first_row, rows_at_once;  // first_row is past any tile where an octet has nothing to do
  __device__ __forceinline__ explicit OctetWalk(int groups) {
    const int octet = threadIdx.x / 8;
    across = min(groups, kOctets);
    rows_at_once = kOctets / across;
    first_group = octet % across;
    first_row = octet / across < rows_at_once ? octet / across : kRowTile;
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, 4) cache_append_kernel(AppendParams p, int tiles, int counters) {
  constexpr int NG = D / kCacheGroup;
  const int b = blockIdx.x / tiles, e = threadIdx.x & 7, groups = p.c.hkv * NG;
  const AppendSpan s = append_span(p, b);
  // a sequence of one block: nothing else reads its counters, so they are brought up to date here
  if (counters) __syncthreads();
  const int row0 = (int)(blockIdx.x % tiles) * kRowTile;
  const int rows = min(min(kRowTile, s.count - row0), p.c.cap - s.at - row0);  // rows that do not fit are left out
  const OctetWalk walk(groups);
  for (int hc = walk.first_group; hc < groups; hc += walk.across) {
    const int h = hc / NG, c = hc % NG;
    int row = walk.first_row;
    if (row >= rows) continue;
    const T* ksrc = (const T*)p.k.ptr + b * p.k.sb + (row0 + row) * p.k.sl + h * p.k.sh + c * kCacheGroup + 8 * e;
    const T* vsrc = (const T*)p.v.ptr + b * p.v.sb + (row0 + row) * p.v.sl + h * p.v.sh + c * kCacheGroup + 8 * e;
    const int64_t kstep = walk.rows_at_once * p.k.sl, vstep = walk.rows_at_once * p.v.sl;
    int slot = s.at + row0 + row;
    const int64_t head = ((int64_t)b * p.c.hkv + h) * p.c.cap;  // cache row of the head's first slot
    uint32_t* const kdst = reinterpret_cast<uint32_t*>(p.c.k) + head * (D / 8);
    uint32_t* const vdst = reinterpret_cast<uint32_t*>(p.c.v) + head * (D / 8);
    // lanes 0 and 1 of an octet store the limits, 2 and 3 of a row's first the position and the weight
    uint32_t* const ldst = (e == 0 ? p.c.kl : p.c.vl) + head * NG + c;
    auto kraw = load_group(ksrc, p.vec);
    auto vraw = load_group(vsrc, p.vec);
#pragma unroll 1
    for (; row < rows; row += walk.rows_at_once, slot += walk.rows_at_once) {
      uint32_t xl, yl;
      const uint32_t xw = quantise_group(kraw, xl), yw = quantise_group(vraw, yl);
      if (row + walk.rows_at_once < rows) {  // on their way while this row is stored
        ksrc += kstep, vsrc += vstep;
        kraw = load_group(ksrc, p.vec);
        vraw = load_group(vsrc, p.vec);
      }
      kdst[(int64_t)slot * (D / 8) + cache_k_word(D, c, e, slot)] = xw;
      vdst[(int64_t)slot * (D / 8) + cache_v_word(D, c, e, slot)] = yw;
      if (e < 2) ldst[(int64_t)slot * NG] = e ? yl : xl;
      else if (c == 0 && e == 2) store_relaxed(p.c.pos + head + slot, p.positions ? p.positions[(int64_t)b * p.t + row0 + row] : s.pos + row0 + row);
      else if (c == 0 && e == 3) p.c.weight[head + slot] = 0.f;
    }
  }
  if (counters && threadIdx.x == 0) append_counters(p, b, s);
}

__global__ void cache_counters_kernel(AppendParams p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < p.c.b) append_counters(p, b, append_span(p, b));
}

// ---- read --------------------------------------------------------------------------------------------
// The same walk the other way: value = min + code step, rounded once.  2 x 32768 tokens of 16 heads, 128 channels, to bf16:
// 694 MB in 143 us, 4.9 TB/s; it waits longest for its loads (8.3 cycles an instruction; 55 % of issue slots are used).
// Code j of a word as a float (2^23 + code is 0x4b000000 | code; a conversion instruction runs at an eighth of the rate).
__device__ __forceinline__ float code_of(uint32_t w, int j) {
  return __uint_as_float(((w >> (4 * j)) & 15u) | 0x4b000000u) - 8388608.f;
}

struct ReadParams {
  CacheView c;
  TensorView k, v;
  const int32_t* start;
  int32_t t, vec;
};

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) cache_read_kernel(ReadParams p, int tiles) {
  constexpr int NG = D / kCacheGroup;
  const int b = blockIdx.x / tiles, e = threadIdx.x & 7, groups = p.c.hkv * NG;
  const int len = min(max(p.c.len[b], 0), p.c.cap), row0 = (int)(blockIdx.x % tiles) * kRowTile;
  const int64_t first = (int64_t)(p.start ? p.start[b] : 0) + row0;
  const int rows = min(kRowTile, p.t - row0);
  const OctetWalk walk(groups);
  for (int hc = walk.first_group; hc < groups; hc += walk.across) {
    const int h = hc / NG, c = hc % NG;
    T* kdst = (T*)const_cast<void*>(p.k.ptr) + b * p.k.sb + row0 * p.k.sl + h * p.k.sh + c * kCacheGroup + 8 * e;
    T* vdst = (T*)const_cast<void*>(p.v.ptr) + b * p.v.sb + row0 * p.v.sl + h * p.v.sh + c * kCacheGroup + 8 * e;
    const int64_t head = ((int64_t)b * p.c.hkv + h) * p.c.cap;
#pragma unroll 4
    for (int row = walk.first_row; row < rows; row += walk.rows_at_once) {
      const int64_t slot = first + row;
      float x[8], y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
      if (slot >= 0 && slot < len) {
        const int64_t at = head + slot;
        const uint32_t xw = reinterpret_cast<const uint32_t*>(p.c.k)[at * (D / 8) + cache_k_word(D, c, e, (int)slot)];
        const uint32_t yw = reinterpret_cast<const uint32_t*>(p.c.v)[at * (D / 8) + cache_v_word(D, c, e, (int)slot)];
        const uint32_t xl = p.c.kl[at * NG + c], yl = p.c.vl[at * NG + c];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = fmaf(code_of(xw, j), __uint_as_float(xl << 16), __uint_as_float(xl & 0xffff0000u));
          y[j] = fmaf(code_of(yw, j), __uint_as_float(yl << 16), __uint_as_float(yl & 0xffff0000u));
        }
      }
      store8(kdst + row * p.k.sl, p.vec, x);
      store8(vdst + row * p.v.sl, p.vec, y);
    }
  }
}

// ---- evict -------------------------------------------------------------------------------------------
// A row's rank as an unsigned key: recent rows above all, NaN weights below all, -0 as 0.
__device__ __forceinline__ uint32_t rank_key(float w, int pos, int64_t recent_from) {
  if (pos >= recent_from) return 0xffffffffu;
  if (!(w == w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return max((u >> 31) ? ~u : (u | 0x80000000u), 1u);
}

constexpr int kSelThreads = 512;
constexpr int kSelBlocks = 8;    // of a (sequence, head) at most
constexpr int kSelKeys = 40960;  // keys of a block that shared memory holds

// Sum of `x` over the threads before this one; *total gets the block's.
__device__ __forceinline__ int block_exclusive(int x, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = s;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kSelThreads / 32; ++i) {
    const int y = sums[i];
    before += i < warp ? y : 0;
    all += y;
  }
  *total = all;
  return s - x + before;
}

// Which slot goes where: src[i] for the slots i < keep of one (sequence, head).  A kept row below `keep` stays,
// the kept rows above fill the gaps in ascending order: the fewest rows move, none of them over one that is
// still to be read, and the order in a cache means nothing, since every row carries its position.
//
// One cluster of blocks for each (sequence, head): each block has a run of slots, whose keys it reads once and keeps
// in shared memory, and they add up one another's digit counts and totals through it.  What bounds it is the latency
// of seven cluster barriers, four digits and three totals: 4 x 8 heads of 22938 to 32768 rows take 29 us with cold caches, of
// which reading their 7 MB would be 1.
// ws: src [b hkv, keep], then the gaps [b hkv, keep].
__global__ void __launch_bounds__(kSelThreads) cache_select_kernel(CacheView c, int keep, int recent, int held, int32_t* ws) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ uint32_t s_key[];  // `held` keys
  __shared__ int hist[2][256];         // digit counts of this block, of even and odd digits
  __shared__ int sums[kSelThreads / 32];
  __shared__ int s_totals[3];  // of this block: rows at the last key, gaps, fills
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t bh = blockIdx.x / size, pairs = gridDim.x / size;
  const int b = (int)(bh / c.hkv), n = min(max(c.len[b], 0), c.cap);
  const float* w = c.weight + bh * c.cap;
  const int32_t* pos = c.pos + bh * c.cap;
  int32_t* src = ws + bh * keep;
  int32_t* gap_slot = ws + (pairs + bh) * keep;
  const int64_t from = recent > 0 ? (int64_t)c.seen[b] - recent : INT64_MAX;
  if (n <= keep) {  // (every block of the cluster)
    for (int i = rank * kSelThreads + threadIdx.x; i < n; i += size * kSelThreads) src[i] = i;
    return;
  }
  // This block's slots [lo, hi), and this thread's run of them: an odd number, so that the runs lie on different banks
  const int share = (n + size - 1) / size, lo = min(rank * share, n), hi = min(lo + share, n);
  const int run = ((hi - lo + kSelThreads - 1) / kSelThreads) | 1;
  const int mine = min(lo + (int)threadIdx.x * run, hi), mine_end = min(mine + run, hi);
  const bool cached = share <= held;
  auto key_at = [&](int i) { return cached ? s_key[i - lo] : rank_key(w[i], pos[i], from); };
  if (cached)
    for (int i = lo + threadIdx.x; i < hi; i += kSelThreads) s_key[i - lo] = rank_key(w[i], pos[i], from);
  // the key of the last kept row, digit by digit from the top
  uint32_t prefix = 0;
  int need = keep;
  for (int digit = 3; digit >= 0; --digit) {
    const int shift = 8 * digit;
    int* h = hist[digit & 1];
    if (threadIdx.x < 256) h[threadIdx.x] = 0;
    __syncthreads();
    for (int i = lo + threadIdx.x; i < hi; i += kSelThreads) {
      const uint32_t key = key_at(i);
      if (digit == 3 || (key >> (shift + 8)) == prefix) atomicAdd(&h[(key >> shift) & 255u], 1);
    }
    cluster.sync();
    int count = 0;
    if (threadIdx.x < 256) {
      int part[kSelBlocks];  // (all on their way before the first is waited for)
#pragma unroll
      for (int r = 0; r < kSelBlocks; ++r) part[r] = r < size ? cluster.map_shared_rank(h, r)[255 - threadIdx.x] : 0;
#pragma unroll
      for (int r = 0; r < kSelBlocks; ++r) count += part[r];
    }
    int total;
    const int above = block_exclusive(count, sums, &total);  // rows of a larger digit
    if (threadIdx.x < 256 && above < need && above + count >= need) {
      s_prefix = (prefix << 8) | (255u - threadIdx.x);
      s_need = need - above;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // `need` of the rows whose key is `prefix` stay, the lowest slots first
  auto before = [&](int which) {  // of the blocks with lower slots
    int part[kSelBlocks], x = 0;
#pragma unroll
    for (int r = 0; r < kSelBlocks; ++r) part[r] = r < rank ? cluster.map_shared_rank(s_totals, r)[which] : 0;
#pragma unroll
    for (int r = 0; r < kSelBlocks; ++r) x += part[r];
    return x;
  };
  int total, equal = 0;
  for (int i = mine; i < mine_end; ++i) equal += key_at(i) == prefix;
  int eq = block_exclusive(equal, sums, &total);
  if (threadIdx.x == 0) s_totals[0] = total;
  cluster.sync();
  eq += before(0);
  int gaps = 0, fills = 0;
  auto each = [&](auto f) {
    int seen = eq;
    for (int i = mine; i < mine_end; ++i) {
      const uint32_t key = key_at(i);
      const bool kept = key > prefix || (key == prefix && seen < need);
      seen += key == prefix;
      f(i, kept);
    }
  };
  each([&](int i, bool kept) {
    gaps += i < keep && !kept;
    fills += i >= keep && kept;
  });
  int gap = block_exclusive(gaps, sums, &total);
  if (threadIdx.x == 0) s_totals[1] = total;
  int fill = block_exclusive(fills, sums, &total);
  if (threadIdx.x == 0) s_totals[2] = total;
  cluster.sync();
  gap += before(1);
  fill += before(2);
  each([&](int i, bool kept) {
    if (i >= keep) return;
    if (kept) src[i] = i;
    else gap_slot[gap++] = i;
  });
  cluster.sync();  // (also: no block leaves while another reads its totals)
  each([&](int i, bool kept) {
    if (i >= keep && kept) src[gap_slot[fill++]] = i;
  });
}

// Copies the rows src[i] -> i and brings the destination's counters up to date.  In place only the gaps are
// written (slots below `keep`) and only rows from `keep` on are read.  Where a row's words lie depends on its slot in
// steps of 16 bytes, so a lane moves 16 bytes of K and of V.  32 x 4096 rows that come one by one from the whole cache take
// 19 us (38 MB), in sectors of 32 bytes.
template <int D>
__global__ void __launch_bounds__(256) cache_move_kernel(CacheView c, CacheView dst, int keep, const int32_t* src) {
  constexpr int NG = D / kCacheGroup, kPieces = D / 32, kRows = 256 / kPieces;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / c.hkv), n = min(min(max(c.len[b], 0), c.cap), keep);
  const bool in_place = dst.k == c.k;
  const int lane = threadIdx.x % kPieces;
#pragma unroll 2
  for (int i = blockIdx.y * kRows + threadIdx.x / kPieces; i < n; i += gridDim.y * kRows) {
    const int from = src[bh * keep + i];
    if (in_place && from == i) continue;
    const int64_t a = bh * c.cap + from, z = bh * dst.cap + i;
    const uint4 kw = reinterpret_cast<const uint4*>(c.k)[a * kPieces + (lane ^ cache_k_swap(D, from))];
    const uint4 vw = reinterpret_cast<const uint4*>(c.v)[a * kPieces + (lane ^ cache_v_swap(D, from))];
    reinterpret_cast<uint4*>(dst.k)[z * kPieces + (lane ^ cache_k_swap(D, i))] = kw;
    reinterpret_cast<uint4*>(dst.v)[z * kPieces + (lane ^ cache_v_swap(D, i))] = vw;
    if (lane < NG) dst.kl[z * NG + lane] = c.kl[a * NG + lane];
    if (lane < NG) dst.vl[z * NG + lane] = c.vl[a * NG + lane];
    if (lane == 0) dst.pos[z] = c.pos[a];
    if (lane == 1) dst.weight[z] = c.weight[a];
  }
  // in place min(length, keep) reads the same before and after this store
  if (blockIdx.y == 0 && bh % c.hkv == 0 && threadIdx.x == 0) {
    dst.len[b] = n;
    if (!in_place) dst.seen[b] = c.seen[b];
  }
}

bool aligned16(const TensorView& t, int es) {
  return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0 && t.sb * es % 16 == 0 && t.sl * es % 16 == 0 && t.sh * es % 16 == 0;
}

// f(type tag, integral constant of the head dim)
template <typename F>
cudaError_t by_type_and_dim(int dtype, int d, F f) {
  auto dim = [&](auto tag) {
    if (d == 64) f(tag, std::integral_constant<int, 64>{});
    else if (d == 128) f(tag, std::integral_constant<int, 128>{});
    else f(tag, std::integral_constant<int, 256>{});
  };
  if (dtype == RA_DTYPE_F32) dim(float{});
  else dim(__nv_bfloat16{});
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_cache_append(const CacheView& c, TensorView k, TensorView v, int dtype, int t, const int32_t* counts,
                                const int32_t* start, const int32_t* positions, cudaStream_t s) {
  AppendParams p;
  p.c = c;
  p.k = k;
  p.v = v;
  p.counts = counts;
  p.start = start;
  p.positions = positions;
  p.t = t;
  const int es = dtype == RA_DTYPE_F32 ? 4 : 2;
  p.vec = aligned16(k, es) && aligned16(v, es);
  p.status = device_status_word();
  if (!p.status) return cudaErrorInvalidSymbol;
  // One launch where one block a sequence does all its rows (a token each, or a few), else the counters that the
  // blocks of a sequence all read are brought up to date by a launch of their own.
  const int tiles = (t + kRowTile - 1) / kRowTile;
  const bool one = tiles == 1;
  cudaError_t e = by_type_and_dim(dtype, c.d, [&](auto tag, auto dim) {
    cache_append_kernel<decltype(tag), decltype(dim)::value><<<(unsigned)c.b * tiles, kRowThreads, 0, s>>>(p, tiles, one);
  });
  if (e != cudaSuccess) return e;
  count_launch();
  if (!one) {
    cache_counters_kernel<<<(c.b + 127) / 128, 128, 0, s>>>(p);
    count_launch();
  }
  return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheView& c, TensorView k, TensorView v, int dtype, int t, const int32_t* start,
                              cudaStream_t s) {
  ReadParams p;
  p.c = c;
  p.k = k;
  p.v = v;
  p.start = start;
  p.t = t;
  const int es = dtype == RA_DTYPE_F32 ? 4 : 2;
  p.vec = aligned16(k, es) && aligned16(v, es);
  const int tiles = (t + kRowTile - 1) / kRowTile;
  count_launch();
  return by_type_and_dim(dtype, c.d, [&](auto tag, auto dim) {
    cache_read_kernel<decltype(tag), decltype(dim)::value><<<(unsigned)c.b * tiles, kRowThreads, 0, s>>>(p, tiles);
  });
}

cudaError_t launch_cache_evict(const CacheView& c, const CacheView& dst, int keep, int recent, int32_t* ws, cudaStream_t s) {
  const int bh = c.b * c.hkv;
  // Up to eight blocks for a (sequence, head) where one would read more than a few keys a thread (their barriers cost about
  // as much as that) and they are not more than run at once, or one could not hold its keys.  One block / eight, us of an
  // eviction: 32 pairs of 5000 keys 21 / 20, 16384 keys 38 / 22, 32768 keys 63 / 26; 512 pairs of 8192 keys 54 / 170.
  int size = 1, dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  if (c.cap > 8 * kSelThreads)
    while (size < kSelBlocks && ((int64_t)bh * 2 * size <= 2048 / kSelThreads * sms || c.cap / size > kSelKeys)) size *= 2;
  const int share = (c.cap + size - 1) / size, held = share < kSelKeys ? share : kSelKeys;
  if ((e = cudaFuncSetAttribute(cache_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelKeys * 4)) != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)bh * size);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = held * 4;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, cache_select_kernel, c, keep, recent, held, ws)) != cudaSuccess) return e;
  count_launch(2);
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  const int rows = 256 / (c.d / 32), blocks = (keep + 2 * rows - 1) / (2 * rows);
  cfg.gridDim = dim3(bh, blocks < 1024 ? blocks : 1024);
  const int32_t* src = ws;
  if (c.d == 64) return cudaLaunchKernelEx(&cfg, cache_move_kernel<64>, c, dst, keep, src);
  if (c.d == 128) return cudaLaunchKernelEx(&cfg, cache_move_kernel<128>, c, dst, keep, src);
  return cudaLaunchKernelEx(&cfg, cache_move_kernel<256>, c, dst, keep, src);
}

}  // namespace ra
