// dip_head_rope.h — RMSNorm of a head of 128 values and its rotary embedding, by 16
// lanes with 8 values each: what the writers of the quantised caches share.
#pragma once

#include "dip_common.h"

namespace dip {

constexpr int kKvHeadDim = 128;

// A sum over 16 lanes in 64 bits.
template <int CTRL>
DIP_DEV double dpp_mov64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xF, 0xF, true);
  const uint32_t hi =
      (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
DIP_DEV double sum16_64(double v) {
  v += dpp_mov64<0xB1>(v);   // the lanes of group_sum<16>
  v += dpp_mov64<0x4E>(v);
  v += dpp_mov64<0x141>(v);
  return v + dpp_mov64<0x140>(v);
}

// 1 / sqrt(x) in 64 bits, x normal, or 0, infinite or NaN (inf, 0, NaN): two Newton
// steps on the hardware's estimate (2^-26 or better), which is the result itself
// where x is infinite and the steps would make inf * 0 of it.
DIP_DEV double rsqrt64(double x) {
  const double e = __builtin_amdgcn_rsq(x);
  double r = fma(e * 0.5, fma(-x * e, e, 1.0), e);
  r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
  return x > 0.0 && x < INFINITY ? r : e;
}

// x: values 8 i .. 8 i + 7 (bf16 pairs) of a head that 16 neighbouring lanes hold, i
// = 0 .. 15 each of them; afterwards the head normed, times `weight`, and turned by
// row `row` of the tables.
//
// The norm's mean and root are taken in 64 bits, and x * r is the 64-bit
// product's fp32 rounding (r in two parts): a key next to a border between two of
// a cache's numbers falls to the same side whatever the order of the sum.  The other
// roundings are those of qk_rope_cache_kernel (dip_decode.hip).
DIP_DEV void head_norm_rope(uint32_t (&x)[4], const uint16_t* weight, const uint16_t* cos_t,
                            const uint16_t* sin_t, int64_t row, int i, float eps) {
  const uint4 wv = reinterpret_cast<const uint4*>(weight)[i];
  const uint4 cv = reinterpret_cast<const uint4*>(cos_t)[row * 16 + i];
  const uint4 sv = reinterpret_cast<const uint4*>(sin_t)[row * 16 + i];
  const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w}, cs[4] = {cv.x, cv.y, cv.z, cv.w};
  const uint32_t sn[4] = {sv.x, sv.y, sv.z, sv.w};
  auto lo = [](uint32_t v) { return __uint_as_float(v << 16); };
  auto hi = [](uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); };
  auto pack = [](float u, float v) { return cvt_bf16x2(u, v); };
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const double u = lo(x[e]), v = hi(x[e]);
    ss = fma(u, u, ss);
    ss = fma(v, v, ss);
  }
  double r = rsqrt64(fma(sum16_64(ss), 1.0 / kKvHeadDim, (double)eps));
  if (__builtin_expect(__any(r > 0x1p100), 0)) {
    // without an eps, subnormal numbers alone take r past fp32's range
    const float up = r > 0x1p100 ? 0x1p64f : 1.f;
    r = r > 0x1p100 ? r * 0x1p-64 : r;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = pack(lo(x[e]) * up, hi(x[e]) * up);
  }
  const float r0 = (float)r, r1 = (float)(r - (double)r0);
  uint32_t y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t n = pack(fmaf(lo(x[e]), r0, lo(x[e]) * r1), fmaf(hi(x[e]), r0, hi(x[e]) * r1));
    y[e] = pack(lo(w[e]) * lo(n), hi(w[e]) * hi(n));
  }
  // rotate_half: dims [0, 64) take -y[d + 64], dims [64, 128) take y[d - 64]
  const uint32_t flip = i < 8 ? 0x80008000u : 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t h = (uint32_t)__builtin_amdgcn_mov_dpp((int)y[e], 0x128, 0xF, 0xF, true);
    const uint32_t s = sn[e] ^ flip;
    const uint32_t u = pack(lo(y[e]) * lo(cs[e]), hi(y[e]) * hi(cs[e]));
    const uint32_t v = pack(lo(h) * lo(s), hi(h) * hi(s));
    x[e] = pack(lo(u) + lo(v), hi(u) + hi(v));
  }
}

}  // namespace dip
