// Attention over the 4-bit cache for many query rows: a prompt's next chunk, many drafted tokens.  Same results as
// cache4_attn.cu, whose products are made from codes in registers; here the work is a matrix product (128 query rows to
// every key) and goes to the tensor-memory MMAs.
//
// A CTA has 128 query rows and walks over units of 64 keys.  It decodes a unit's K and V once, into fp16 operands in
// shared memory,   k' = step (code - 8) 2^(9 - e)   and   v' = (min + step code) 2^(15 - f),
// and then per unit:  S = Q K'^T + (group sums of q) (mid 2^(9 - e))^T,  p = exp2(S 2^(e - 9) factor + f - m),  O += P V'.
// step has 8 significant bits and |code - 8| is at most 8, so k' is exact in fp16 where step 2^(9 - e) is 2^-17 or more (a row
// with a smaller one takes a power of two of its own, and what is smaller still, below 2^-25 of its row's largest value, loses
// 2^-30 of that); the other part of a key, its groups' mid = min + 8 step times the sums of q over the groups, is one
// more step of the product, of two-part factors (22 bits each).  Scores, and L with them, so have fp32 accuracy as in the
// other form.  v' and P are rounded by 2^-11 of themselves, values below 2^-19 of their row's largest by 2^-29 of that.
// e and f are powers of two that bring the rows into fp16's range: largest values below 2^9 for K, where the two-part mids
// are the limit, and 2^15 for V.  They are one number for a unit, a scalar in the exponent, as long as the largest values of
// its rows are within 2^8 of one another; a unit where they are not, or that holds NaN or infinities, gives such rows their
// own and takes the form of the softmax that reads them per key, which is also the form for masks and ALiBi.  m, the
// reference of the exponents, is the largest s + f less kHeadroom.
//
// Warps 0 to 3 form the exponentials (a thread has a row of the tile, its lane of tensor memory), warps 4 to 7 decode (a
// thread has a K or a V row of the unit), warp 8 issues the products.  Operands and S are double-buffered, so that the next
// unit is decoded and multiplied while this one's exponentials are formed, and two CTAs of an SM (one at 256 channels:
// 203 KB of operands) fill one another's waits.
// Four pairs of barriers, one of a pair for each buffer: KV (operands are there), S, P (written by the softmax warps), O (the
// products that read the operands and P are done).  A segment ends with an operand buffer marked as the end, and all
// warps meet before the next one.
//
// What bounds it is the chain of a unit (scores, exponentials, P, its product) with 18 warps an SM to fill its waits, which
// registers limit: 44 % of issue slots are used, and a warp waits longest for what it reads of tensor memory and for the
// other roles.  Measured, 16 heads over 4, 128 channels, 448 tokens that end a cache of 8192, causal: 89 us (29 GFLOP, 330
// TFLOP/s), and 14 for the join; 256 channels, 640 rows on 2 heads of 28838 keys, causal: 146 us, 514 in the other form.
// TMEM columns: S0 [0, 64), S1 [64, 128), O [128, 128 + D); P lies in the first half of its S.
#include <cuda_fp16.h>

#include <type_traits>

#include "cache4_sched.cuh"
#include "tc_common.cuh"

namespace ra {
namespace {

using namespace ptx;

constexpr int kThreads = 288, kRows = kPromptRows, kKeys = kCacheUnit;
constexpr float kLog2e = 1.4426950408889634f, kHeadroom = 6.f, kGrow = 8.f;
// A row's largest value is below 2^exponent, and below 2^kTopK or 2^kTopV as an operand.
constexpr int kTopK = 9, kTopV = 15;
constexpr int kLeastExp = -64;  // of that value, and that of a row that is not there
constexpr float kLeastStep = 0x1p-17f;  // of K, from which on its products with codes are exact
// p 2^(f - m) of a unit whose f lies below the first may be less than a float holds where larger values elsewhere set m, while p
// itself still counts in the sum of probabilities, which is then formed without f; so it is where 2^-f is no normal float.
constexpr int kFarExp = -11, kMostExp = 126;
constexpr int kRoom = 2, kSpan = 10;  // a unit's exponents may lie this far below its common one, which starts kRoom above
// The common exponent after a unit of largest exponent `most` that did not fit.
__device__ __forceinline__ int next_common(int common, int most) {
  return most > common || most < common - kSpan ? most + kRoom : common;
}
static_assert(kKeys == 64 && kRows == 128, "tile shapes are written out below");

__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn_major) {
  return make_idesc_bf16(m, n, false, b_mn_major) & ~((1u << 7) | (1u << 10));  // operand format 0: fp16
}

template <int D>
struct PromptShape {
  static constexpr int NG = D / 64;
  static constexpr int kQPanel = kRows * 128, kKvPanel = kKeys * 128;  // bytes of 64 channels
  // sums of q and mids of K: 16 halves a row, without swizzle: groups of 8 rows, each 16 bytes of every row and then the
  // other 16
  static constexpr int kQSum = kRows * 32, kKMid = kKeys * 32;
  static constexpr int kQ = 0, kK = kQ + NG * kQPanel, kV = kK + 2 * NG * kKvPanel, kQs = kV + 2 * NG * kKvPanel, kKm = kQs + kQSum,
                       kSide = kKm + 2 * kKMid;
};

// What the other warps need to know of a unit besides its operands.
struct alignas(16) Side {
  int pos[kKeys];
  int e[kKeys], f[kKeys];               // exponents of K and V rows
  uint32_t bad_k[kKeys], bad_v[kKeys];  // != 0: K is NaN; bit c: group c of V is
  int most[4];                          // by decoding warp: the largest exponent of its rows,
  int odd[4];                           // and whether exponents differ or something is NaN
  int least_pos[2], most_pos[2];        // of the K warps'
  int unit;                             // -1: the segment has ended
};
enum Bars { KV_FULL = 0, S_FULL = 2, P_FULL = 4, O_DONE = 6, kBars = 8 };
template <bool MASKED>
struct Shared {
  Side side[2];
  uint64_t bars[kBars];
  int unit[4];           // number i of the segment: i % 4
  int first[4];          // largest exponents in the segment's first unit, by decoding warp
  Run run;
  Segment seg;
  UnitWalk<MASKED> walk;  // of the last decoding warp alone
  int has;
  uint32_t abort, tmem;
};

// Barrier of the four decoding warps that tells whether all of their threads are well.
__device__ __forceinline__ bool decoders_meet(bool ok) {
  int all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 128, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((int)ok)
      : "memory");
  return all != 0;
}

template <int D>
constexpr uint32_t kTmemColumns = D == 256 ? 512 : 256;
// The same as tmem_alloc and tmem_dealloc, with the number of columns an immediate: a number in a register counts as all
// 512 when the driver works out how many CTAs fit on an SM.
template <int D>
__device__ __forceinline__ void tmem_take(uint32_t* smem_result) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "n"(kTmemColumns<D>)
               : "memory");
}
template <int D>
__device__ __forceinline__ void tmem_give_back(uint32_t taddr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "n"(kTmemColumns<D>) : "memory");
}

// Barrier of the softmax warps and the one that issues products: the queries are in shared memory.
__device__ __forceinline__ void queries_there() { asm volatile("barrier.cta.sync 2, 160;" ::: "memory"); }

template <int D, bool MASKED>
constexpr int kPromptSmem = PromptShape<D>::kSide + (int)sizeof(Shared<MASKED>) + 1024;

__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

__device__ __forceinline__ uint32_t plain_at(int row, int chunk) { return (uint32_t)((row >> 3) * 256 + chunk * 128 + (row & 7) * 16); }
constexpr uint32_t kPlainDescHi = (256u >> 4) | (1u << 14);  // 256 bytes between groups of 8 rows, no swizzle
__device__ __forceinline__ uint64_t plain_desc(uint32_t lo) { return ((uint64_t)kPlainDescHi << 32) | lo; }
// x as two fp16 values, the larger in the low half.
__device__ __forceinline__ uint32_t two_parts(float x) {
  const __half hi = __float2half_rn(x);
  const __half2 r = __halves2half2(hi, __float2half_rn(x - __half2float(hi)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Exponent of a row of K or V whose largest value is x >= 0 (infinity, too: a sum of limits that is just beyond).
__device__ __forceinline__ int row_exponent(float x) {
  return max((int)(__float_as_uint(x) >> 23) - 126, kLeastExp);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Eight codes as fp16 values in the order 0 4 1 5 2 6 3 7:  K: step (code - 8), exact;  V: min + step code.  0x6400 | code is
// 1024 + code, and 0x5400 | 16 code, a code in the upper half of a byte, is 64 + code.
template <bool V>
__device__ __forceinline__ uint4 decode8(uint32_t w, __half2 step, __half2 mn) {
  constexpr float base = V ? 0.f : 8.f;
  const __half2 lo0 = __float2half2_rn(1024.f + base), hi0 = __float2half2_rn(64.f + base);
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = ((w >> (8 * i)) & 0x000f000fu) | 0x64006400u, hi = ((w >> (8 * i)) & 0x00f000f0u) | 0x54005400u;
    const __half2 a = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&lo), lo0), step, mn);
    const __half2 b = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&hi), hi0), step, mn);
    r[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
    r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// 32 bytes at once: shared memory leaves next to no L1 cache, so that two halves of a sector would be fetched twice.  Arrays
// that lie on 16-byte boundaries alone (`wide` false) are read that way all the same.
__device__ __forceinline__ void load32(const uint4* p, bool wide, uint4& lo, uint4& hi) {
  if (!wide) {
    lo = p[0];
    hi = p[1];
    return;
  }
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
               : "l"(p));
}

// One decoding thread's row of a unit: the first 64 threads have the K rows, the others the V rows.  Loaded a unit ahead
// into registers, decoded into shared memory when the operands' buffer is free.
template <int D>
struct KeyRow {
  static constexpr int NG = D / 64, kVec = D / 32;  // 16-byte pieces of a row
  uint4 word[kVec];
  uint32_t limits[NG];
  int pos;

  // `thread`: of the decoding warps, 0 to 127
  __device__ __forceinline__ void load(const AttnArgs& a, int64_t bh, int unit, int thread, bool with_pos) {
    const CacheView& c = a.p.c;
    const bool v = thread >= 64;
    const int slot = unit * kKeys + (thread & 63);
    const int64_t at = bh * c.cap + slot;
    const uint4* src = reinterpret_cast<const uint4*>(v ? c.v : c.k) + at * kVec;
    const int swap = v ? cache_v_swap(D, slot) : cache_k_swap(D, slot);  // (of whole 32 bytes)
#pragma unroll
    for (int i = 0; i < kVec; i += 2) load32(src + (i ^ swap), a.wide, word[i], word[i + 1]);
#pragma unroll
    for (int i = 0; i < NG; ++i) limits[i] = (v ? c.vl : c.kl)[at * NG + i];
    pos = with_pos && !v ? c.pos[at] : 0;
  }
  // Largest value of the row, groups that are not finite left out.
  __device__ __forceinline__ float most() const {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const float st = __uint_as_float(limits[i] << 16), mn = __uint_as_float(limits[i] & 0xffff0000u);
      if (fabsf(mn) <= 3.4e38f && st <= 3.4e38f) x = fmaxf(x, fmaxf(fabsf(mn), fabsf(fmaf(15.f, st, mn))));
    }
    return x;
  }

  __device__ __forceinline__ void decode(char* smem, int buf, Side& side, int live, int thread, int common, bool with_pos) const {
    using Sh = PromptShape<D>;
    const int row = thread & 63, warp = thread >> 5;
    const bool v = thread >= 64, there = row < live;
    float step[NG], mn[NG], least = INFINITY;  // smallest step that is not 0
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      step[i] = __uint_as_float(limits[i] << 16);
      mn[i] = __uint_as_float(limits[i] & 0xffff0000u);
      const bool finite = fabsf(mn[i]) <= 3.4e38f && step[i] <= 3.4e38f;
      if (there && !finite) bad |= 1u << i;
      if (!there || !finite) step[i] = mn[i] = 0.f;  // (rows behind the last hold anything)
      if (step[i] > 0.f) least = fminf(least, step[i]);
    }
    const int own = there ? row_exponent(most()) : kLeastExp;
    const bool fits = !there || (own <= common && own >= common - kSpan && (v || least * two_to(kTopK - common) >= kLeastStep));
    const int e = fits ? common : own;
    (v ? side.f : side.e)[row] = e;
    (v ? side.bad_v : side.bad_k)[row] = bad;
    const int largest = __reduce_max_sync(0xffffffffu, own);
    const bool odd = __any_sync(0xffffffffu, !fits || bad);
    if ((thread & 31) == 0) {
      side.most[warp] = largest;
      side.odd[warp] = odd;
    }
    const float scale = two_to((v ? kTopV : kTopK) - e);
    __half2 st[NG], off[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      st[i] = __float2half2_rn(step[i] * scale);
      off[i] = __float2half2_rn(v ? mn[i] * scale : 0.f);
    }
    char* const to = smem + (v ? Sh::kV : Sh::kK) + buf * NG * Sh::kKvPanel + row * 128;
    const int turn = row & 7;  // 128-byte swizzle: chunk i of a row lies at i ^ turn
    // words of the row in slot 0's order: K of more than 64 channels runs e by e in pairs within a quad's lane, V group by
    // group (cache_k_word, cache_v_word)
    auto decode_row = [&](auto is_v) {
      constexpr bool kIsV = decltype(is_v)::value;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t w[4] = {word[i].x, word[i].y, word[i].z, word[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = 4 * i + j;
          const int c = kIsV ? n % NG : D == 64 ? 0 : 2 * (n >> 4) + ((n >> 1) & 1);
          const int chunk = kIsV ? n / NG : D == 64 ? n : 2 * ((n >> 2) & 3) + (n & 1);
          *reinterpret_cast<uint4*>(to + c * Sh::kKvPanel + ((chunk ^ turn) << 4)) = decode8<kIsV>(w[j], st[c], off[c]);
        }
      }
    };
    if (v) {
      decode_row(std::true_type{});
    } else {
      decode_row(std::false_type{});
      // mid 2^(6 - e) of the groups, against sums 2^-6: hi hi, hi lo, lo hi, lo lo
      uint32_t m[8] = {};
#pragma unroll
      for (int c = 0; c < NG; ++c) m[2 * c] = m[2 * c + 1] = two_parts(fmaf(8.f, step[c], mn[c]) * scale * 64.f);
      char* mid = smem + Sh::kKm + buf * Sh::kKMid;
      *reinterpret_cast<uint4*>(mid + plain_at(row, 0)) = make_uint4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<uint4*>(mid + plain_at(row, 1)) = make_uint4(m[4], m[5], m[6], m[7]);
      if (with_pos) {
        side.pos[row] = pos;
        const int lo = __reduce_min_sync(0xffffffffu, there ? pos : INT_MAX), hi = __reduce_max_sync(0xffffffffu, there ? pos : INT_MIN);
        if ((thread & 31) == 0) side.least_pos[warp] = lo, side.most_pos[warp] = hi;
      }
    }
  }
};

// Scores of a row against the keys of a unit that cannot all be treated alike, finished in place in tensor memory: each by
// its key's powers of two, ALiBi and the masks (-inf).  The result is the groups of V that are NaN in a key the row sees.
// A rolled loop out of line, so that the main loop keeps its registers.  The whole warp calls it.
template <bool MASKED>
__device__ __noinline__ uint32_t scores_by_key(uint32_t taddr, const Side& side, int live, uint32_t kinds, int window, int qpos,
                                               float slope, float factor) {
  uint32_t nan_groups = 0;
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 8) {
    uint32_t r[8];
    tmem_ld8(taddr + c, r);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = c + j;
      float x = fmaf(__uint_as_float(r[j]), factor * two_to(side.e[key] - kTopK), (float)side.f[key]);
      bool vis = key < live;
      if constexpr (MASKED) {
        const int kpos = side.pos[key];
        if (kinds & RA_MOD_ALIBI) x = fmaf(-slope, (float)(qpos - kpos), x);
        if (kinds & RA_MOD_CAUSAL) vis = vis && kpos <= qpos;
        if (kinds & RA_MOD_WINDOW) vis = vis && qpos - kpos < window;
      }
      if (vis) nan_groups |= side.bad_v[key];
      if (side.bad_k[key]) x = NAN;
      r[j] = __float_as_uint(vis ? x : -INFINITY);
    }
    tmem_st8(taddr + c, r);
  }
  tc_wait_st();
  return nan_groups;
}

// A wait of a whole warp: its lanes leave it together.
#define WARP_WAIT(bar, parity) __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status, kStCacheWait))

template <int D, bool MASKED>
__global__ void __launch_bounds__(kThreads, kPromptPerSm<D>) cache_prompt_kernel(const __grid_constant__ AttnArgs a) {
  using Sh = PromptShape<D>;
  constexpr int NG = Sh::NG;
  extern __shared__ uint8_t smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared<MASKED>& sh = *reinterpret_cast<Shared<MASKED>*>(smem + Sh::kSide);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_seq = a.p.c.hkv * a.tiles, per = a.p.h / a.p.c.hkv;
  if (warp == 8) {
    Run r;
    const bool has = find_run<MASKED>(a.p.c, per_seq, blockIdx.x, a.ctas, r);
    if (lane == 0) {
      sh.run = r;
      sh.has = has;
      sh.abort = 0;
      for (int i = 0; i < kBars; ++i) mbar_init(&sh.bars[i], i < S_FULL || (i >= P_FULL && i < O_DONE) ? 128 : 1);
      fence_barrier_init();
    }
    __syncwarp();
    if (has) {
      tmem_take<D>(&sh.tmem);
      tmem_relinquish();
      tc_fence_before();
    }
  }
  __syncthreads();
  tc_fence_after();
  launch_dependents();
  if (!sh.has) return;
  const uint32_t tmem = sh.tmem, tmem_o = tmem + 128;
  volatile uint32_t* abort_flag = &sh.abort;

  bool ok = true;
  uint32_t kv_phase = 0, unit_phase = 0;  // bit b: parity of the next use of buffer b, by operands (or the end) / by units
  while (true) {
    Segment w;
    {
      Run run = sh.run;
      if (!next_segment<MASKED>(a, per_seq, run, w)) break;
      __syncthreads();  // everyone has read the run, and is done with the segment before
      if (threadIdx.x == 0) {
        sh.run = run;
        sh.seg = w;
      }
    }
    const int64_t bh = (int64_t)w.b * a.p.c.hkv + w.h;
    const int len = min(max(a.p.c.len[w.b], 0), a.p.c.cap);
    // positions of the tile's queries (of the rows that are there), for the whole warp
    auto pos_of = [&](int r) { return a.p.q_pos ? a.p.q_pos[(int64_t)w.b * a.p.lq + r / per] : a.p.c.seen[w.b] - a.p.lq + r / per; };
    int q_least = 0, q_most = 0;
    if (MASKED && (warp < 4 || warp == 7)) {
      q_least = INT_MAX, q_most = INT_MIN;
#pragma unroll
      for (int i = 0; i < kRows / 32; ++i) {
        const int p = pos_of(min(w.tile * kRows + 32 * i + lane, a.rows - 1));
        q_least = min(q_least, p), q_most = max(q_most, p);
      }
      q_least = __reduce_min_sync(0xffffffffu, q_least), q_most = __reduce_max_sync(0xffffffffu, q_most);
    }

    if (warp < 4) {
      // ================================================================ softmax: a row of the tile
      const int row = threadIdx.x, at_row = min(w.tile * kRows + row, a.rows - 1);
      const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
      // ---- the rows as fp16, each scaled to [2^13, 2^14), channels of a chunk in the order of decode8, and their group
      // sums.  A warp copies its 32 rows as they are, D / 8 lanes a row, then each thread works on its own.  (Rolled loops:
      // what runs once should be few instructions to fetch; unrolled this took 11 us of a CTA.)
      {
        constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kPasses = 32 / kAtOnce;
        const int i = lane % kLanes;
        int rr = warp * 32 + lane / kLanes, token = (w.tile * kRows + rr) / per, head = w.tile * kRows + rr - token * per;
#pragma unroll 1
        for (int p = 0; p < kPasses; ++p, rr += kAtOnce) {
          const int qr = w.tile * kRows + rr;
          char* to = smem + Sh::kQ + i / 8 * Sh::kQPanel + swizzled(rr, i % 8);
          const __nv_bfloat16* src = (const __nv_bfloat16*)a.p.q.ptr + w.b * a.p.q.sb + token * a.p.q.sl + (w.h * per + head) * a.p.q.sh + 8 * i;
          for (head += kAtOnce; head >= per; head -= per) ++token;
          if (qr >= a.rows) {
            *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
          } else if (a.vec) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(src) : "memory");
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) reinterpret_cast<__nv_bfloat16*>(to)[j] = src[j];
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
      }
      auto chunk_at = [&](int i) { return reinterpret_cast<uint4*>(smem + Sh::kQ + i / 8 * Sh::kQPanel + swizzled(row, i % 8)); };
      __nv_bfloat162 most = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 2
      for (int i = 0; i < D / 8; ++i) {
        const uint4 r = *chunk_at(i);
        const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&r);
        most = __hmax2(most, __hmax2(__hmax2(__habs2(v[0]), __habs2(v[1])), __hmax2(__habs2(v[2]), __habs2(v[3]))));
      }
      const float top = fmaxf(__low2float(most), __high2float(most));
      const int top_e = (int)(__float_as_uint(top) >> 23);
      const float norm = top > 0.f && top_e < 255 ? __uint_as_float((uint32_t)min(13 + 254 - top_e, 253) << 23) : 1.f;
      // (never 0, so that a masked score of -inf stays one; a negative scale turns the queries' sign)
      const float factor = fmaxf(1.f / norm * fabsf(a.p.scale) * kLog2e, 1e-30f), by = a.p.scale < 0.f ? -norm : norm;
      uint32_t sums[8] = {};
#pragma unroll
      for (int c = 0; c < NG; ++c) {
        float sum = 0.f;
#pragma unroll 2
        for (int i = 0; i < 8; ++i) {
          const uint4 r = *chunk_at(8 * c + i);
          const uint32_t v[4] = {r.x, r.y, r.z, r.w};
          float x[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[2 * j] = __uint_as_float(v[j] << 16) * by, x[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u) * by;
          uint32_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sum += x[j] + x[j + 4];
            const __half2 h2 = __floats2half2_rn(x[j], x[j + 4]);
            h[j] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          *chunk_at(8 * c + i) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        // sums 2^-6 of the groups, against mids: hi hi, hi lo, lo hi, lo lo
        const uint32_t t = two_parts(sum * 0.015625f);
        sums[2 * c] = __byte_perm(t, t, 0x1010);
        sums[2 * c + 1] = __byte_perm(t, t, 0x3232);
      }
      *reinterpret_cast<uint4*>(smem + Sh::kQs + plain_at(row, 0)) = make_uint4(sums[0], sums[1], sums[2], sums[3]);
      *reinterpret_cast<uint4*>(smem + Sh::kQs + plain_at(row, 1)) = make_uint4(sums[4], sums[5], sums[6], sums[7]);
      fence_proxy_async_smem();
      const int qpos = MASKED ? pos_of(at_row) : 0;
      const float slope = MASKED && (a.p.kinds & RA_MOD_ALIBI) ? a.p.slopes[w.h * per + at_row % per] * kLog2e : 0.f;
      queries_there();

      float m = -INFINITY, l = 0.f;
      uint32_t nan_groups = 0;
      int n = 0;  // units done
#pragma unroll 1
      for (; ok; ++n) {
        const int buf = n & 1;
        const Side& side = sh.side[buf];
        if (!(ok = WARP_WAIT(&sh.bars[KV_FULL + buf], kv_phase >> buf & 1))) break;
        kv_phase ^= 1u << buf;
        const int unit = side.unit;
        if (unit < 0) break;
        const int live = len - unit * kKeys, f_unit = side.f[0];
        const int4 odds = *reinterpret_cast<const int4*>(side.odd);
        const bool odd = (odds.x | odds.y | odds.z | odds.w) != 0, apart = odd || f_unit < kFarExp || f_unit > kMostExp;
        bool plain = !odd && live >= kKeys;
        if constexpr (MASKED) {
          const int lo = min(side.least_pos[0], side.least_pos[1]), hi = max(side.most_pos[0], side.most_pos[1]);
          plain = plain && !(a.p.kinds & RA_MOD_ALIBI) && (!(a.p.kinds & RA_MOD_CAUSAL) || hi <= q_least) &&
                  (!(a.p.kinds & RA_MOD_WINDOW) || (long long)q_most - lo < a.p.window);
        }
        float scale = factor * two_to(side.e[0] - kTopK), off = (float)f_unit;
        const uint32_t phase = unit_phase >> buf & 1;
        if (!(ok = WARP_WAIT(&sh.bars[S_FULL + buf], phase))) break;
        tc_fence_after();
        const uint32_t tmem_s = tmem + buf * 64 + lane_off;
        if (!plain) {
          nan_groups |= scores_by_key<MASKED>(tmem_s, side, live, a.p.kinds, a.p.window, qpos, slope, factor);
          scale = 1.f, off = 0.f;
        }
        // (32 scores at a time, read twice: registers are scarcer than the way to tensor memory)
        uint32_t r[32];
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tmem_ld32(tmem_s + 32 * c, r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 2) t[(j >> 1) & 3] = max3(t[(j >> 1) & 3], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
        }
        const float peak = fmaf(max3(t[0], t[1], fmaxf(t[2], t[3])), scale, off - kHeadroom);
        if (__any_sync(0xffffffffu, peak > m + kGrow)) {
          const float to = fmaxf(m, peak), root = m == -INFINITY ? 0.f : ex2(0.5f * (m - to)), by = root * root;  // (part_root)
          m = to;
          l = l * root * root;
          if (n > 0) {  // O is complete up to the unit before
            if (!(ok = WARP_WAIT(&sh.bars[O_DONE + (buf ^ 1)], (unit_phase >> (buf ^ 1) & 1) ^ 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 8) {
              uint32_t o[8];
              tmem_ld8(tmem_o + lane_off + c, o);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * by);
              tmem_st8(tmem_o + lane_off + c, o);
            }
          }
        }
        const float add = off - (m == -INFINITY ? 0.f : m);
        const uint64_t s2 = pack2(scale, scale), a2 = pack2(add, add);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          tmem_ld32(tmem_s + 32 * c, r);
          tc_wait_ld();
          uint32_t pk[16];
          uint64_t sum2 = 0;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x0, x1;
            unpack2(fma2(pack2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s2, a2), x0, x1);
            r[2 * j] = __float_as_uint(x0), r[2 * j + 1] = __float_as_uint(x1);
            x0 = ex2(x0), x1 = ex2(x1);
            const __half2 h2 = __floats2half2_rn(x0, x1);
            pk[j] = *reinterpret_cast<const uint32_t*>(&h2);
            sum2 = add2(sum2, pack2(x0, x1));
          }
          tmem_st16(tmem_s + c * 16, pk);
          if (!apart) {
            float s0, s1;
            unpack2(sum2, s0, s1);
            sum += s0 + s1;
          } else {  // each key by its own power of two, which P may have taken below what a float holds
#pragma unroll
            for (int j = 0; j < 32; ++j) sum += ex2(__uint_as_float(r[j]) - (float)side.f[32 * c + j]);
          }
        }
        l = fmaf(sum, apart ? 1.f : two_to(-f_unit), l);
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(&sh.bars[P_FULL + buf]);
        unit_phase ^= 1u << buf;
      }
      if (ok && n > 0) {
        const int buf = (n - 1) & 1;
        ok = WARP_WAIT(&sh.bars[O_DONE + buf], (unit_phase >> buf & 1) ^ 1);
        tc_fence_after();
      }
      // ---- results (the segment from shared memory again, out of the registers of the loop)
      if (ok) {
        const volatile Segment& sg = sh.seg;
        const int b = sg.b, h = sg.h, q_row = sg.tile * kRows + row, at_row = min(q_row, a.rows - 1), first = sg.first;
        const bool row_live = q_row < a.rows, whole = sg.whole;
        // cut at its start: this CTA's first part, else its second
        float* part = a.part + (((int64_t)blockIdx.x * 2 + (first == 0)) * kRows + row) * kPartPitch<D>;
        __nv_bfloat16* dst = (__nv_bfloat16*)const_cast<void*>(a.p.out.ptr) + b * a.p.out.sb + (int64_t)(at_row / per) * a.p.out.sl +
                             (int64_t)(h * per + at_row % per) * a.p.out.sh;
#pragma unroll 1
        for (int col = 0; col < D; col += 16) {
          uint32_t o[16] = {};
          if (n > 0) {
            tmem_ld16(tmem_o + lane_off + col, o);
            tc_wait_ld();
          }
          float x[16];
#pragma unroll
          for (int j = 0; j < 16; ++j)  // column j of a chunk of 8 is channel (j >> 1) + 4 (j & 1)
            x[(j & 8) + ((j & 7) >> 1) + 4 * (j & 1)] = nan_groups >> (col / 64) & 1 ? NAN : __uint_as_float(o[j]) * two_to(-kTopV);
          if (!row_live) continue;
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(part + col + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
          } else if (a.vec_out) {
#pragma unroll
            for (int j = 0; j < 16; j += 8)
              *reinterpret_cast<uint4*>(dst + col + j) = make_uint4(pack_bf16(x[j] / l, x[j + 1] / l), pack_bf16(x[j + 2] / l, x[j + 3] / l),
                                                                    pack_bf16(x[j + 4] / l, x[j + 5] / l), pack_bf16(x[j + 6] / l, x[j + 7] / l));
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) dst[col + j] = __float2bfloat16_rn(x[j] / l);
          }
        }
        if (row_live) {
          if (!whole) {
            part[D] = m;
            part[D + 1] = l;
          } else if (a.p.lse) {
            a.p.lse[((int64_t)b * a.p.h + h * per + at_row % per) * a.p.lq + at_row / per] = m * 0.6931471805599453f + logf(l);
          }
        }
        tc_fence_before();
      }
    } else if (warp < 8) {
      // ================================================================ decoding
      const int thread = threadIdx.x - 128;
      if (warp == 7) {
        UnitWalk<MASKED> walk;
        if constexpr (MASKED) walk.see(a, bh, q_least, q_most);
        walk.init(len, w.first, w.last, 1);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int u = walk.next();
          if (lane == 0) sh.unit[i] = u;
        }
        if (lane == 0) sh.walk = walk;
      }
      decoders_meet(true);
      KeyRow<D> raw;
      int unit = sh.unit[0], next = sh.unit[1];
      int common = 0;
      if (unit >= 0) {
        raw.load(a, bh, unit, thread, MASKED);
        // the first unit's largest exponent is the one to go by
        const int own = (thread & 63) < len - unit * kKeys ? row_exponent(raw.most()) : kLeastExp;
        const int largest = __reduce_max_sync(0xffffffffu, own);
        if (lane == 0) sh.first[warp - 4] = largest;
      }
      decoders_meet(true);
      common = max(sh.first[(warp - 4) & 2], sh.first[(warp - 4) | 1]) + kRoom;

#pragma unroll 1
      for (int i = 0;; ++i) {
        const int buf = i & 1;
        Side& side = sh.side[buf];
        // the buffer's operands have been read, and what was noted beside them
        if (i >= 2) ok = WARP_WAIT(&sh.bars[O_DONE + buf], (unit_phase >> buf & 1) ^ 1);
        if (ok) {
          if (thread == 0) side.unit = unit;
          if (unit >= 0) {
            raw.decode(smem, buf, side, len - unit * kKeys, thread, common, MASKED);
            if (next >= 0) raw.load(a, bh, next, thread, MASKED);
          }
          fence_proxy_async_smem();
          mbar_arrive(&sh.bars[KV_FULL + buf]);
        }
        if (unit < 0) break;
        unit_phase ^= 1u << buf;
        if (warp == 7) {
          UnitWalk<MASKED> walk = sh.walk;
          const int u = walk.next();
          __syncwarp();
          if (lane == 0) {
            sh.walk = walk;
            sh.unit[(i + 2) & 3] = u;
          }
        }
        ok = decoders_meet(ok);  // the unit after the next is there, and what each warp noted of its rows
        if (!ok) break;
        const int first = (warp - 4) & 2;
        if (side.odd[first] | side.odd[first | 1]) common = next_common(common, max(side.most[first], side.most[first | 1]));
        unit = next;
        next = sh.unit[(i + 2) & 3];
      }
    } else {
      // ================================================================ products
      queries_there();
      constexpr uint32_t kQk = idesc_f16(128, kKeys, false), kPv = idesc_f16(128, D, true);
      const uint32_t q_lo = desc_lo(smem_u32(smem + Sh::kQ), 16), k_lo = desc_lo(smem_u32(smem + Sh::kK), 16);
      const uint32_t qs_lo = desc_lo(smem_u32(smem + Sh::kQs), 128), km_lo = desc_lo(smem_u32(smem + Sh::kKm), 128);
      const uint32_t v_lo = desc_lo(smem_u32(smem + Sh::kV), Sh::kKvPanel);  // MN-major: panels kKvPanel bytes apart
      // Numbers of units: S of unit i, then P V of unit i - 1.  (S goes where P of unit i - 2 was: the pipe takes products
      // in order.)
#pragma unroll 1
      for (int i = 0;; ++i) {
        const int buf = i & 1;
        if (!(ok = WARP_WAIT(&sh.bars[KV_FULL + buf], kv_phase >> buf & 1))) break;
        kv_phase ^= 1u << buf;
        const bool more = sh.side[buf].unit >= 0;
        if (more) {
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t qo = (kk >> 2) * (Sh::kQPanel >> 4) + (kk & 3) * 2, ko = (buf * NG + (kk >> 2)) * (Sh::kKvPanel >> 4) + (kk & 3) * 2;
            mma_ss_warp(tmem + buf * 64, desc_from_lo(q_lo + qo), desc_from_lo(k_lo + ko), kQk, kk > 0);
          }
          mma_ss_warp(tmem + buf * 64, plain_desc(qs_lo), plain_desc(km_lo + buf * (Sh::kKMid >> 4)), kQk, 1u);
          tc_commit_warp(&sh.bars[S_FULL + buf]);
        }
        if (i > 0) {
          const int was = buf ^ 1;
          if (!(ok = WARP_WAIT(&sh.bars[P_FULL + was], unit_phase >> was & 1))) break;
          unit_phase ^= 1u << was;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            mma_ts_warp(tmem_o, tmem + was * 64 + kk * 8, desc_from_lo(v_lo + was * NG * (Sh::kKvPanel >> 4) + kk * (2048 >> 4)), kPv,
                        i > 1 || kk > 0);
          tc_commit_warp(&sh.bars[O_DONE + was]);
        }
        if (!more) break;
      }
    }
    ok = __syncthreads_and(ok);
    if (!ok) break;
  }
  if (!ok) {  // a wait ran out: what the tensor pipe still has gets time to end before its memory is given back
    for (int spin = 0; spin < 1 << 14; ++spin) {
      if (mbar_try_wait(&sh.bars[O_DONE], 0) && mbar_try_wait(&sh.bars[O_DONE + 1], 0) && spin > 1 << 12) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_give_back<D>(tmem);
  }
}

template <int D, bool MASKED>
cudaError_t prepare() {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && done[dev])) return e;
  e = cudaFuncSetAttribute(cache_prompt_kernel<D, MASKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPromptSmem<D, MASKED>);
  if (e == cudaSuccess && dev < 64) done[dev] = true;
  return e;
}

}  // namespace

// f(head dim, whether masked) of a call, as integral constants
template <typename F>
static cudaError_t by_dim_and_mask(int d, bool masked, F f) {
  auto dim = [&](auto mask) {
    if (d == 64) return f(std::integral_constant<int, 64>{}, mask);
    if (d == 128) return f(std::integral_constant<int, 128>{}, mask);
    return f(std::integral_constant<int, 256>{}, mask);
  };
  return masked ? dim(std::true_type{}) : dim(std::false_type{});
}

cudaError_t cache_prompt_prepare(int d, bool masked) {
  return by_dim_and_mask(d, masked, [](auto dim, auto mask) { return prepare<decltype(dim)::value, decltype(mask)::value>(); });
}

cudaError_t launch_cache_prompt(const AttnArgs& a, cudaStream_t s) {
  return by_dim_and_mask(a.p.c.d, a.p.kinds != 0, [&](auto dim, auto mask) {
    constexpr int D = decltype(dim)::value;
    constexpr bool kMask = decltype(mask)::value;
    cache_prompt_kernel<D, kMask><<<a.ctas, kThreads, kPromptSmem<D, kMask>, s>>>(a);
    return cudaGetLastError();
  });
}

}  // namespace ra
