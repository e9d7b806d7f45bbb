// How the attention kernels over the 4-bit cache divide their work, and what they share (cache4_attn.cu: few query rows,
// cache4_prompt.cu: many).
//
// An item is one (sequence, key/value head, query tile).  All units (64 keys) of all items, in a row, are cut into as many
// equal runs as CTAs fit on the GPU, so that ragged lengths leave no CTA idle; a run goes through segments of one or more
// items, and a second kernel joins the items that were cut.  Where the cuts lie follows from the lengths, which only the
// device knows: every CTA works them out from there, so that a captured call stays right while the cache grows.
#pragma once
#include <climits>

#include "cache4.cuh"
#include "ptx_sm100.cuh"

namespace ra {

// Floats of a row of a part: 16-byte rows.
template <int D>
constexpr int kPartPitch = D + 4;

struct AttnArgs {
  CacheAttnParams p;
  int32_t rows;      // query rows of a key/value head: (h / hkv) * lq
  int32_t tiles;     // query tiles of 8 NT rows
  int32_t cluster;   // CTAs of an item of a short cache; 0: a long one
  int32_t ctas;      // CTAs launched
  int32_t vec;       // q rows on 16-byte boundaries
  int32_t vec_out;   // out rows on 16-byte boundaries
  int32_t wide;      // k and v of the cache on 32-byte boundaries, and so all of their rows
  int32_t weights_group;  // units a CTA of the weights pass holds at a time
  float* part;       // [ctas][2][rows of a tile][kPartPitch]: unnormalised out, then max, then sum
  int32_t* item;     // [items][2]: first and last CTA
  unsigned int* status;
};

namespace {

constexpr int kMinUnits = 4;  // units of a run at least


// Programmatic dependent launch: the kernel after this one may start its blocks / waits until the one before has ended.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The root of the factor 2^(m - top) by which a part with reference m counts: 0 for one that saw nothing, NaN for one of NaN
// alone (l is its sum).  The references follow the size of the values, so that the factor itself may be less than a float
// holds where l, of smaller values, still counts; l is multiplied by the root twice.
__device__ __forceinline__ float part_root(float m, float l, float top) {
  return m == -INFINITY ? (l == l ? 0.f : NAN) : ptx::ex2(0.5f * (m - top));
}

// ---- schedule ----------------------------------------------------------------------------------------
__device__ __forceinline__ int units_of(const CacheView& c, int b) {
  return (min(max(c.len[b], 0), c.cap) + kCacheUnit - 1) / kCacheUnit;
}
// Units of an item as the cuts count them: an empty cache has one, whose CTA writes that there is nothing to see, and
// taking up an item costs about as much as kItemCost units, which come first.
constexpr int kItemCost = 2;
// Under a mask units are taken in the order of a matrix of kSpread columns read by columns, so that what is visible
// spreads over all warps and runs wherever it lies: number i is unit (i % kSpread) * rows + i / kSpread.
constexpr int kSpread = 64;
__device__ __forceinline__ int spread_rows(int units) { return (units + kSpread - 1) / kSpread; }
template <bool MASKED>
__device__ __forceinline__ int cut_units(const CacheView& c, int b) {
  const int u = max(units_of(c, b), 1);
  return (MASKED ? spread_rows(u) * kSpread : u) + kItemCost;
}

struct Run {
  long long at, end;  // units of all items in a row
  long long seq_at;   // first unit of sequence b
  int b;
};
// The run of CTA number `cta` (one warp calls it); false: none.
template <bool MASKED>
__device__ bool find_run(const CacheView& c, int per_seq, int cta, int ctas, Run& run) {
  const int lane = threadIdx.x & 31;
  unsigned int sum = 0;
  for (int b = lane; b < c.b; b += 32) sum += cut_units<MASKED>(c, b);
  const long long total = (long long)__reduce_add_sync(0xffffffffu, sum) * per_seq;
  const long long n = min((long long)ctas, (total + kMinUnits - 1) / kMinUnits);
  if (cta >= n) return false;
  run.at = total * cta / n;
  run.end = total * (cta + 1) / n;
  long long before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    const long long own = b < c.b ? (long long)cut_units<MASKED>(c, b) * per_seq : 0;
    long long end = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += y;
    }
    const unsigned int hit = __ballot_sync(0xffffffffu, run.at < before + end);
    if (hit) {
      const int at = __ffs(hit) - 1;
      run.b = b0 + at;
      run.seq_at = before + __shfl_sync(0xffffffffu, end - own, at);
      return true;
    }
    before += __shfl_sync(0xffffffffu, end, 31);
  }
}

struct Segment {
  int b, h, tile, first, last, step;  // units first, first + step, ... below last
  bool whole;                         // all of the item
};

// The next segment of a run and the notes about its item (every thread calls it); false after the last.
template <bool MASKED>
__device__ bool next_segment(const AttnArgs& a, int per_seq, Run& run, Segment& w) {
  do {
    if (run.at >= run.end) return false;
    int units = cut_units<MASKED>(a.p.c, run.b);
    while (run.at >= run.seq_at + (long long)units * per_seq) {
      run.seq_at += (long long)units * per_seq;
      units = cut_units<MASKED>(a.p.c, ++run.b);
    }
    w.b = run.b;
    const int in_seq = (int)((run.at - run.seq_at) / units);
    w.h = in_seq / a.tiles;
    w.tile = in_seq % a.tiles;
    const int from = (int)(run.at - run.seq_at - (long long)in_seq * units), to = (int)min((long long)units, from + (run.end - run.at));
    run.at += to - from;
    units -= kItemCost;
    w.first = max(from - kItemCost, 0);
    w.last = to - kItemCost;
    w.whole = w.first == 0 && w.last == units;
    if (threadIdx.x == 0 && w.last > 0) {
      const int64_t item = ((int64_t)w.b * a.p.c.hkv + w.h) * a.tiles + w.tile;
      if (w.first == 0) a.item[2 * item] = blockIdx.x;
      if (w.last == units) a.item[2 * item + 1] = blockIdx.x;
    }
  } while (w.last <= 0);  // the cut left this CTA the cost alone
  return true;
}

// The units [first, last) of an item, every stride-th from `first` on; the whole warp calls it.
template <bool MASKED>
struct UnitWalk {
  int unit, stride, left;
  __device__ __forceinline__ void init(int len, int first, int last, int step) {
    last = min(last, (len + kCacheUnit - 1) / kCacheUnit);
    left = first < last ? (last - first + step - 1) / step : 0;
    unit = first;
    stride = step;
  }
  // The next unit, -1 after the last.
  __device__ __forceinline__ int next() {
    const int u = left > 0 ? unit : -1;
    unit += stride;
    --left;
    return u;
  }
};
// Where there is a mask: of the numbers [first, last) (see kSpread), the units that some row of the tile may see.  The
// positions of kLook units are looked through at a time.
template <>
struct UnitWalk<true> {
  static constexpr int kLook = 16, kLanes = kCacheUnit / 4, kAtOnce = 32 / kLanes;  // a lane reads four positions
  const int32_t* kpos;
  int at, stride, left, rows, live;
  uint32_t found;  // bit i: the i-th number from `at` on is of use
  int looked;      // numbers from `at` on that `found` stands for
  long long lo, hi;  // a key is of use where lo < its position <= hi

  // Positions of the tile's queries.
  __device__ __forceinline__ void see(const AttnArgs& a, int64_t bh, int least, int most) {
    kpos = a.p.c.pos + bh * a.p.c.cap;
    hi = a.p.kinds & RA_MOD_CAUSAL ? most : LLONG_MAX;
    lo = a.p.kinds & RA_MOD_WINDOW ? (long long)least - a.p.window : LLONG_MIN;
  }
  __device__ __forceinline__ void init(int len, int first, int last, int step) {
    rows = spread_rows((len + kCacheUnit - 1) / kCacheUnit);
    last = min(last, rows * kSpread);
    live = len;
    left = first < last ? (last - first + step - 1) / step : 0;
    found = 0;
    looked = 0;
    at = first;
    stride = step;
  }
  __device__ __forceinline__ int unit_of(int n) const {
    const int i = at + n * stride;
    return i % kSpread * rows + i / kSpread;
  }
  __device__ __forceinline__ int next() {
    const int lane = threadIdx.x & 31, sub = lane / kLanes;
    while (!found) {
      at += looked * stride;
      left -= looked;
      if (left <= 0) {
        looked = 0;
        return -1;
      }
      looked = min(left, kLook);
      constexpr int kLoads = 4;
#pragma unroll 1
      for (int base = 0; base < looked; base += kLoads * kAtOnce) {
        int4 x[kLoads];
        int key[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int n = base + kAtOnce * i + sub;
          key[i] = n < looked ? unit_of(n) * kCacheUnit + 4 * (lane % kLanes) : INT_MAX;
          x[i] = key[i] < live ? *reinterpret_cast<const int4*>(kpos + key[i]) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int room = live - key[i];  // (negative where there is no key)
          const bool use = (room > 0 && x[i].x > lo && x[i].x <= hi) || (room > 1 && x[i].y > lo && x[i].y <= hi) ||
                           (room > 2 && x[i].z > lo && x[i].z <= hi) || (room > 3 && x[i].w > lo && x[i].w <= hi);
          const uint32_t votes = __ballot_sync(0xffffffffu, use);
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j)
            if (votes >> (j * kLanes) & ((1ull << kLanes) - 1)) found |= 1u << (base + kAtOnce * i + j);
        }
      }
    }
    const int u = unit_of(__ffs(found) - 1);
    found &= found - 1;
    return u;
  }
};

}  // namespace

cudaError_t cache_prompt_prepare(int d, bool masked);
cudaError_t launch_cache_prompt(const AttnArgs& a, cudaStream_t s);
constexpr int kPromptRows = 128;  // of its query tiles
// CTAs of the kernel for many query rows that fit on an SM: by registers, shared memory and tensor memory.  (The driver's
// count says 1 for any kernel that allocates tensor memory.)
template <int D>
constexpr int kPromptPerSm = D == 256 ? 1 : 2;

}  // namespace ra
