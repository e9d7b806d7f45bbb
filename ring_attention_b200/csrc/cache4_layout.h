// The 4-bit key/value cache: layout of a row and the formula of its codes, shared by the kernels that
// fill, read, move and attend over it (cache4_store.cu, cache4_attn.cu).  Compiles for the host too.
//
// A row holds the d channels of one token and key/value head in groups of 64.  A group is 16 levels:
//   min  = bf16 at or below the smallest channel, step = bf16 at or above (largest - min) / 15,
//   code = rint((x - min) / step) in 0..15, standing for min + code * step (off by at most step / 2).
// step and min are one 32-bit word (step in the low half).  A group that holds a NaN or an infinity, or
// a channel beyond the bf16 range, has step = min = NaN and reads back as NaN.
//
// Codes are packed eight to a 32-bit word: nibble i of word e of group c is channel 64 c + 8 e + i.  Words
// sit in the row in the order in which a warp's matrix fragments want them, so that the attention kernel's
// shared-memory reads are 4 to 16 contiguous bytes a lane with no two lanes of a phase on one bank:
//   K  word e belongs to lane pair (t, j) = (e / 2, e % 2): lane t of a quad reads its 2 NG words at once
//      (d = 256: two 16-byte pieces, which change places in odd slots, 128-byte rows having all the same banks)
//   V  word e belongs to lane group g = e, which reads its NG words at once; g is XORed with bits of the slot
// Both depend on the slot by its lowest three bits only; a row that moves to another slot is permuted.
#pragma once
#include "score_mod.h"

namespace ra {

constexpr int kCacheGroup = 64;
constexpr int kCacheUnit = 64;  // keys of one step of a warp; capacities are multiples of kCacheAlign
constexpr int kCacheAlign = 64;

// Word (of d / 8) that holds word e (0..7) of group c in the row of `slot`.
RA_HD int cache_k_word(int d, int c, int e, int slot) {
  const int t = e >> 1, j = e & 1;
  if (d == 64) return 2 * t + j;
  if (d == 128) return 4 * t + 2 * c + j;
  return (((c >> 1) ^ slot) & 1) * 16 + 4 * t + 2 * (c & 1) + j;
}
RA_HD int cache_v_swizzle(int d, int slot) {
  if (d == 64) return 0;
  if (d == 128) return slot & 4;
  return (slot & 4) | ((slot & 1) << 1);
}
RA_HD int cache_v_word(int d, int c, int e, int slot) {
  return (e ^ cache_v_swizzle(d, slot)) * (d / 64) + c;
}
// The same in 16-byte pieces of a row: piece i of slot 0's order lies at i ^ swap.
RA_HD int cache_k_swap(int d, int slot) { return d == 256 ? (slot & 1) << 2 : 0; }
RA_HD int cache_v_swap(int d, int slot) { return cache_v_swizzle(d, slot) >> (d == 128 ? 1 : 0); }
// Row r (0..7) of an 8-row half of a matrix fragment is key kappa(r) of the half: neighbouring rows then differ in
// parity and rows 0, 2, 4, 6 in (bit 0, bit 2), which is what keeps the reads of K and V rows off one another's banks.
RA_HD int cache_kappa(int r) { return r ^ ((r >> 1) & 1); }

// Whether the note of an item's first and last CTA can be followed: a CTA whose wait ran out leaves items without one, and
// the workspace there holds anything.
RA_HD bool cache_note_holds(int first, int last, int ctas) { return first >= 0 && last >= first && last < ctas; }

}  // namespace ra
