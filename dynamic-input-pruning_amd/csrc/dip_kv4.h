// dip_kv4.h — the 4-bit key/value cache: its layout in memory and the device
// code that packs and unpacks it.
//
// Values.  Each row (position) of each key/value head has 128 keys and 128
// values, in groups of 32 consecutive dimensions.  A group is a bf16 scale s
// and whole numbers q in [-7, 7] (4 bits, two's complement) and stands for
// q * s.  With a the group's largest magnitude,
//   s = a / 7 with the significand cut to 5 bits (0 below 2^-100),
//   q = rint(x / s).
// Cutting s keeps 7 s <= a (nothing overflows) and a / s < 7.5, so every error
// is at most s / 2; and |q| <= 7 has 3 bits, so q * s has at most 8: it is a
// bf16 number, and every reader of the cache computes with the same values.
// A group that holds a NaN or an infinity has s = NaN and stands for NaN.
//
// Layout (per key/value head; max_len a multiple of 32):
//   scales bf16 [max_len][2][4]: a row's 4 key scales, then its 4 value scales.
//   keys   [max_len][16 words]: word 4 c + g of a row holds dimensions
//          32 g + 8 c .. + 7, so one 16-byte load per lane is the A operand of
//          four 16x16x32 MFMAs (lane quarter c, 16 rows), one per group: a
//          group's scale then multiplies a finished product.
//   values [max_len / 32][512 words]: 32 rows together.  Word
//          256 (d / 64) + 64 c + 4 (d % 16) + (d / 16) % 4 holds dimension d of
//          the rows 4 c .. 4 c + 3 and 16 + 4 c .. 16 + 4 c + 3: as many rows as
//          a lane of quarter c has scores of in the result of the key MFMAs, so
//          the softmax's weights are the value MFMA's B operand where they are.
// In a word, element j (a dimension of a key, a row of a value) is nibble
// n = j / 2 + 4 (j % 2), at the bits 4 n + 3 .. of the word (modulo 32): v_bitop3
// turns nibbles m and m + 4 into one register of the operand (elements 2 m and
// 2 m + 1), the first pair where it lies, the others after one shift.
#pragma once

#include "dip_attn.h"
#include "dip_head_rope.h"
#include "dip_internal.h"

namespace dip {

constexpr int kKvGroups = 4;           // scale groups of a row
constexpr int kKvKeyBytes = 64;        // a row's packed keys
constexpr int kKvScaleVals = 8;        // a row's scales (keys, then values)
constexpr int kKvBlock = 32;           // rows of a value block
constexpr int kKvBlockWords = 512;

// Element j of a word, as a shift; the last one's nibble wraps around.
DIP_DEV int kv4_shift(int j) { return 4 * ((j >> 1) + 4 * (j & 1)) + 3; }
DIP_DEV uint32_t kv4_rotl(uint32_t v, int s) { return __builtin_rotateleft32(v, (uint32_t)s); }
// The word of a value block that holds dimension d for lane quarter c.
DIP_DEV int kv4_value_word(int d, int c) {
  return 256 * (d >> 6) + 64 * c + 4 * (d & 15) + ((d >> 4) & 3);
}
// Row r (0 .. 31) of a block: lane quarter and element of the word.
DIP_DEV int kv4_row_quarter(int r) { return (r >> 2) & 3; }
DIP_DEV int kv4_row_elem(int r) { return 4 * (r >> 4) + (r & 3); }

// One word as an MFMA operand of 8 bf16 values (1.5 + q / 16) * 2^-kLower (exact).
template <int kLower = 0>
DIP_DEV bf16x8_t kv4_biased(uint32_t w) {
  constexpr uint32_t kFlip = kPairMagicFlip - kLower * 0x00800080u;
  u32x4_t r;
  r.x = (w & kPairMask) ^ kFlip;
  r.y = ((w >> 4) & kPairMask) ^ kFlip;
  r.z = ((w >> 8) & kPairMask) ^ kFlip;
  r.w = (__builtin_amdgcn_alignbit(w, w, 12) & kPairMask) ^ kFlip;
  return __builtin_bit_cast(bf16x8_t, r);
}

// Keys are taken 2^-8 lower, so that the 1.5 times 32 of bf16's largest queries stays
// finite.
constexpr int kKeyLower = 8;
constexpr float kKeyUnit = 1.f / (1 << kKeyLower);

// Nibble at `shift` as a signed number.
DIP_DEV int kv4_nibble(uint32_t w, int shift) {
  return (int)kv4_rotl(w, (28 - shift) & 31) >> 28;
}

// Max over aligned groups of W lanes (4 or 16) of whole numbers.
template <int W>
DIP_DEV uint32_t group_umax(uint32_t v) {
  static_assert(W == 4 || W == 16, "W");
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
  if (W == 4) return v;
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
}

// The larger magnitude of a bf16 pair, as the fp32 bits that order like it.
DIP_DEV uint32_t kv4_abs_max(uint32_t pair) {
  return max((pair << 16) & 0x7FFFFFFFu, pair & 0x7FFF0000u);
}

// A group's scale, as fp32 bits (the low 16 are 0), from its largest magnitude.
DIP_DEV uint32_t kv4_scale_bits(uint32_t a) {
  const uint32_t s = __float_as_uint(__uint_as_float(a) / 7.0f) & 0xFFF80000u;
  if (a >= 0x7F800000u) return 0x7FC00000u;  // an infinity or a NaN in the group
  return s < 0x0D800000u ? 0u : s;           // below 2^-100
}

// x's number in a group of that scale, as a nibble.
DIP_DEV uint32_t kv4_number(float x, uint32_t scale_bits) {
  const float s = __uint_as_float(scale_bits);
  const float q = s > 0.f ? rintf(x / s) : 0.f;
  return (uint32_t)(int)fminf(fmaxf(q, -7.f), 7.f) & 15u;
}

// The attention kernels' arguments (dip_kv4_attn.hip, dip_kv4_prompt.hip).
struct Kv4AttnArgs {
  const uint16_t* q;  // [tokens, nkv * group, 128]
  const uint32_t* kc;
  const uint32_t* vc;
  const uint16_t* sc;
  const int64_t* pos;  // the first token's position, or null: `start`
  float* part;         // [tiles, nkv, splits, columns of a tile, kKvPart]
  uint16_t* out;       // [tokens, nkv * group, 128]
  int64_t start;
  int tokens, nkv, group, max_len, splits;
  float scale;
};

// Whether the cache has the rows first .. first + tokens - 1 (tokens >= 0), for any
// first: a position on the device may hold the type's ends.
__host__ DIP_DEV bool rows_in_cache(int64_t first, int tokens, int max_len) {
  return first >= 0 && first <= (int64_t)max_len - tokens;
}

// A prompt's attention over the cache expanded to bf16 (dip_kv4_prompt.hip).
int launch_kv4_prompt_tiles(const Kv4AttnArgs& a, void* workspace, hipStream_t stream);

}  // namespace dip
