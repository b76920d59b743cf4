// dip_kv8.h — the paged 8-bit key/value cache: its layout in memory and the device
// code that packs and unpacks it.
//
// Values.  A page holds 64 consecutive rows (positions) of a sequence, of every
// key/value head 128 keys and 128 values per row.  The keys of a page and head share
// a scale s, a power of two, and so do the values; each is an e4m3 number n of 8
// bits and stands for n * s.  With a the largest magnitude of the rows written,
//   s = 2^(floor(log2 a) - 7), at least 2^-100; 0 while all are 0,
//   n = x / s rounded to the nearest, ties to even, so |n| <= 256 (at s = 2^120, where
//       256 s is beyond bf16, 240 at most).
// A power of two costs a number with an exponent of its own nothing: its rounding is
// 2^-4 of it at any scale, down to the 2^-14 of the largest where its exponents end.
// And it makes n * s a bf16 number (n has 4 significant bits, s n >= 2^-109), so every
// reader computes with the same values; and the change to a larger scale is exact but
// for numbers that leave that range.
// A group of 32 neighbouring dimensions of a row with a NaN or an infinity stands for
// NaN, and does not count in a.
//
// Writes.  A write of rows r .. of a page takes the larger of the scale that the page
// has (none where r is 0: the page begins) and the one of the rows written; where that
// raises it, rows 0 .. r - 1 are rounded again to it.  Rows behind the written ones no
// longer stand for anything.
//
// Layout.  Pages are numbered; a sequence's table has the number of each of its
// pages.  Per page and key/value head
//   keys   [64 rows][128] bytes;
//   values [128 dims][64] bytes, row r at 16 ((r / 4) % 4) + 4 (r / 16) + r % 4;
//   scales fp32, the keys' and the values'.
// A lane's 16 bytes of keys are dimensions of one row, and its 16 bytes of values the
// rows of one dimension that it has scores of in the result of four 16x16x32 MFMAs:
// both are operands of the next ones once they are converted.
#pragma once

#include "dip_attn.h"
#include "dip_head_rope.h"
#include "dip_internal.h"

namespace dip {

constexpr int kPageRows = 64;
constexpr int kPageBytes = kPageRows * kKvHeadDim;  // of keys, and of values, of a head
constexpr int kNanByte4 = 0x7F7F7F7F;

struct Kv8Pages {
  uint8_t* k;
  uint8_t* v;
  float* scales;  // [pages][nkv][2]
  int pages, nkv;
};

// The number of a sequence's page, or -1 where the table has none of the cache's.
DIP_DEV int page_number(const int32_t* table, int64_t page, int pages) {
  const int id = table[page];
  return (unsigned)id < (unsigned)pages ? id : -1;
}

// Two neighbouring numbers of a word, times a scale, as bf16 (exact).
template <bool kHigh>
DIP_DEV uint32_t kv8_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHigh));
}
// Two words as an operand of 8 bf16 values.
DIP_DEV bf16x8_t kv8_operand(uint32_t lo, uint32_t hi, float scale) {
  return __builtin_bit_cast(bf16x8_t,
                            u32x4_t{kv8_pair<false>(lo, scale), kv8_pair<true>(lo, scale),
                                    kv8_pair<false>(hi, scale), kv8_pair<true>(hi, scale)});
}

// 0xFF in each byte of w that is a NaN.
DIP_DEV uint32_t kv8_nan_bytes(uint32_t w) {
  const uint32_t m = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  return (m - (m >> 7)) | m;
}

// The odd rows (of 16, 32 lanes) of a exchanged with the even rows of b.
DIP_DEV void rows_swap16(uint32_t& a, uint32_t& b) {
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
DIP_DEV void rows_swap32(uint32_t& a, uint32_t& b) {
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}

// Between the two orders of four rows' bytes, of which lane 16 g + i has, as rows, the
// dimensions 8 i .. 8 i + 7 of row g in w0, w1, and as columns the four rows of
// dimension 8 i + 2 g in w0 and of 8 i + 2 g + 1 in w1.
DIP_DEV void kv8_rows_to_columns(uint32_t& w0, uint32_t& w1) {
  rows_swap32(w0, w1);
  uint32_t x = __builtin_amdgcn_perm(w1, w0, 0x05010400u);
  uint32_t y = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
  rows_swap16(x, y);
  w0 = __builtin_amdgcn_perm(y, x, 0x05010400u);
  w1 = __builtin_amdgcn_perm(y, x, 0x07030602u);
}
DIP_DEV void kv8_columns_to_rows(uint32_t& w0, uint32_t& w1) {
  uint32_t x = __builtin_amdgcn_perm(w1, w0, 0x06040200u);
  uint32_t y = __builtin_amdgcn_perm(w1, w0, 0x07050301u);
  rows_swap16(x, y);
  w0 = __builtin_amdgcn_perm(y, x, 0x06040200u);
  w1 = __builtin_amdgcn_perm(y, x, 0x07050301u);
  rows_swap32(w0, w1);
}

// What the C entry points ask of a cache and its tables.
inline int check_pages(const void* k, const void* v, const void* scales, int64_t pages,
                       int64_t nkv, const void* table, int64_t seqs, int64_t width) {
  if (pages <= 0 || pages > (1 << 28) || nkv <= 0 || nkv > 4096 || seqs < 0 || seqs > (1 << 24) ||
      width <= 0 || width > (1 << 24))
    return DIP_ERR_SHAPE;
  if (!k || !v || !scales || (seqs > 0 && !table)) return DIP_ERR_NULL;
  if (!aligned16(k) || !aligned16(v) || (reinterpret_cast<uintptr_t>(scales) & 7) ||
      (reinterpret_cast<uintptr_t>(table) & 3))
    return DIP_ERR_ALIGN;
  return DIP_OK;
}

}  // namespace dip
