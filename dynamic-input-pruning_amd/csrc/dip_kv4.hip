// dip_kv4.hip — writing and reading the 4-bit key/value cache (dip_kv4.h has
// its layout): q/k RMSNorm + rotary embedding + quantisation of a token's or a
// prompt's q | k | v into the cache, the quantisation alone of given keys and
// values, and the cache's rows as the bf16 numbers they stand for.
#include "dip_kv4.h"

namespace dip {
namespace {

constexpr int kWriteWaves = 4;  // waves of a workgroup, each with a task of its own

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

struct Kv4WriteArgs {
  const uint16_t* k;  // [tokens] rows, strides in values (kNorm: the q | k | v rows)
  const uint16_t* v;
  int64_t k_tok, k_head, v_tok, v_head;
  const uint16_t* q_w;  // kNorm only, from here on
  const uint16_t* k_w;
  const uint16_t* cos_t;
  const uint16_t* sin_t;
  uint16_t* q_out;
  const int64_t* pos;  // the row of the first token, or null: `start`
  uint32_t* kc;
  uint32_t* vc;
  uint16_t* sc;
  int64_t start;
  int tokens, nh, nkv, max_len, vblocks;
  int k_vec;  // not kNorm: every head of k starts at a multiple of 16 bytes
  float eps;
};

// One wave per task: first the values, a task per (block of 32 rows, lane
// quarter, kv head), which is the 8 rows that share words, so no two waves write
// one word; then the q and k heads, a task per four heads of a token.  Words whose
// rows lie partly outside the written ones keep those rows' nibbles.
//
// A values' task: lane l holds dimensions 2 l and 2 l + 1 of each row, a scale
// group is 16 lanes.  A heads' task: 16 lanes per head, lane i the dimensions
// 8 i .. 8 i + 7 (one 16-byte load), which are one word of a key; a scale group is
// four lanes, and rotate_half's partner dimension is in lane i ^ 8.
//
// Memory bounds a prompt's: 4099 tokens of 64 / 8 heads move 158 MB in 41 us, 3.9
// TB/s.  (A wave per head, two dimensions per lane and the sum by lane shuffles:
// 133 us.)  One token's 3.2 us are the launch and three waits for memory.
//
// The norm's mean and root are taken in 64 bits, and x * r is the 64-bit
// product's fp32 rounding (r in two parts): a key next to a border between two of
// the cache's numbers falls to the same side whatever the order of the sum, so a
// cache row is a function of its token alone.  The other roundings are those of
// qk_rope_cache_kernel (dip_decode.hip).
template <bool kNorm>
__global__ __launch_bounds__(64 * kWriteWaves) void kv4_write_kernel(Kv4WriteArgs a) {
  const int l = threadIdx.x & 63;
  const int64_t task = (int64_t)blockIdx.x * kWriteWaves + (threadIdx.x >> 6);
  const int64_t first = a.pos ? *a.pos : a.start;
  const bool ok = rows_in_cache(first, a.tokens, a.max_len);  // (a.pos may lie outside)
  const int64_t vtasks = (int64_t)a.vblocks * 4 * a.nkv;
  if (task < vtasks) {
    if (!ok) return;
    const int head = (int)(task % a.nkv), c = (int)(task / a.nkv % 4);
    const int64_t block = first / kKvBlock + task / (4 * a.nkv);
    uint32_t word[2] = {0u, 0u}, mask = 0u, pair[8];
    bool in[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t row = block * kKvBlock + 16 * (j >> 2) + 4 * c + (j & 3);
      in[j] = row >= first && row < first + a.tokens;
      pair[j] = 0u;
      if (in[j])
        pair[j] = *reinterpret_cast<const uint32_t*>(a.v + (row - first) * a.v_tok +
                                                     head * a.v_head + 2 * l);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!in[j]) continue;
      const int64_t row = block * kKvBlock + 16 * (j >> 2) + 4 * c + (j & 3);
      const float x0 = bf16_to_f32(pair[j] & 0xFFFFu);
      const float x1 = __uint_as_float(pair[j] & 0xFFFF0000u);
      const uint32_t sb = kv4_scale_bits(group_umax<16>(kv4_abs_max(pair[j])));
      word[0] |= kv4_rotl(kv4_number(x0, sb), kv4_shift(j));
      word[1] |= kv4_rotl(kv4_number(x1, sb), kv4_shift(j));
      mask |= kv4_rotl(15u, kv4_shift(j));
      if ((l & 15) == 0)
        a.sc[((size_t)head * a.max_len + row) * kKvScaleVals + kKvGroups + (l >> 4)] =
            (uint16_t)(sb >> 16);
    }
    if (mask == 0u) return;
    uint32_t* blk = a.vc + ((size_t)head * (a.max_len / kKvBlock) + block) * kKvBlockWords;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t* w = blk + kv4_value_word(2 * l + e, c);
      *w = mask == 0xFFFFFFFFu ? word[e] : (*w & ~mask) | word[e];
    }
    return;
  }
  const int heads = kNorm ? a.nh + a.nkv : a.nkv, quads = (heads + 3) / 4;
  const int64_t t = (task - vtasks) / quads;
  const int head = (int)((task - vtasks) % quads) * 4 + (l >> 4), i = l & 15;
  if (t >= a.tokens) return;
  const bool on = head < heads;
  const int64_t row = ok ? first + t : 0;
  uint32_t x[4] = {0u, 0u, 0u, 0u};
  if (on) {
    const uint16_t* p = a.k + t * a.k_tok + (int64_t)head * a.k_head + 8 * i;
    if (kNorm || a.k_vec) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = reinterpret_cast<const uint32_t*>(p)[e];
    }
  }
  const bool is_q = kNorm && head < a.nh;
  if (kNorm) {
    const uint4 wv = reinterpret_cast<const uint4*>(is_q ? a.q_w : a.k_w)[i];
    const uint4 cv = reinterpret_cast<const uint4*>(a.cos_t)[row * 16 + i];
    const uint4 sv = reinterpret_cast<const uint4*>(a.sin_t)[row * 16 + i];
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
    double r = rsqrt64(fma(sum16_64(ss), 1.0 / kKvHeadDim, (double)a.eps));
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
    if (is_q) {
      reinterpret_cast<uint4*>(a.q_out)[(t * a.nh + head) * 16 + i] =
          make_uint4(x[0], x[1], x[2], x[3]);
      return;
    }
  }
  if (!ok || !on) return;
  const int kvh = kNorm ? head - a.nh : head;
  uint32_t m = 0u, word = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max(m, kv4_abs_max(x[e]));
  const uint32_t sb = kv4_scale_bits(group_umax<4>(m));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    word |= kv4_rotl(kv4_number(__uint_as_float(x[e] << 16), sb), kv4_shift(2 * e));
    word |= kv4_rotl(kv4_number(__uint_as_float(x[e] & 0xFFFF0000u), sb), kv4_shift(2 * e + 1));
  }
  const size_t at = (size_t)kvh * a.max_len + row;
  a.kc[at * (kKvKeyBytes / 4) + 4 * (i & 3) + (i >> 2)] = word;
  if ((i & 3) == 0) a.sc[at * kKvScaleVals + (i >> 2)] = (uint16_t)(sb >> 16);
}

// Rows start .. start + rows - 1 as bf16 [rows, nkv, 128]: a wave per (block,
// lane quarter, kv head), 8 rows each, as the values are written.  (4099 rows of 8
// heads, 4.7 MB read and 16.8 written: 8.4 us.)
__global__ __launch_bounds__(64 * kWriteWaves) void kv4_read_kernel(
    const uint32_t* __restrict__ kc, const uint32_t* __restrict__ vc,
    const uint16_t* __restrict__ sc, uint32_t* __restrict__ k_out, uint32_t* __restrict__ v_out,
    int64_t start, int rows, int nkv, int max_len, int blocks) {
  const int l = threadIdx.x & 63;
  const int64_t task = (int64_t)blockIdx.x * kWriteWaves + (threadIdx.x >> 6);
  if (task >= (int64_t)blocks * 4 * nkv) return;
  const int head = (int)(task % nkv), c = (int)(task / nkv % 4);
  const int64_t block = start / kKvBlock + task / (4 * nkv);
  const uint32_t* blk = vc + ((size_t)head * (max_len / kKvBlock) + block) * kKvBlockWords;
  const uint32_t v0 = blk[kv4_value_word(2 * l, c)], v1 = blk[kv4_value_word(2 * l + 1, c)];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t row = block * kKvBlock + 16 * (j >> 2) + 4 * c + (j & 3);
    if (row < start || row >= start + rows) continue;
    const size_t at = (size_t)head * max_len + row;
    const uint32_t kw = kc[at * (kKvKeyBytes / 4) + 4 * ((l >> 2) & 3) + (l >> 4)];
    const float ks = bf16_to_f32(sc[at * kKvScaleVals + (l >> 4)]);
    const float vs = bf16_to_f32(sc[at * kKvScaleVals + kKvGroups + (l >> 4)]);
    const int sh = kv4_shift(2 * (l & 3));
    const size_t o = ((size_t)(row - start) * nkv + head) * 64 + l;
    k_out[o] = f32_to_bf16((float)kv4_nibble(kw, sh) * ks) |
               (f32_to_bf16((float)kv4_nibble(kw, sh + 16) * ks) << 16);
    v_out[o] = f32_to_bf16((float)kv4_nibble(v0, kv4_shift(j)) * vs) |
               (f32_to_bf16((float)kv4_nibble(v1, kv4_shift(j)) * vs) << 16);
  }
}

int check_cache(const void* kc, const void* vc, const void* sc, int64_t nkv, int64_t max_len) {
  if (!kc || !vc || !sc) return DIP_ERR_NULL;
  if (nkv <= 0 || nkv > 4096 || max_len <= 0 || max_len % kKvBlock != 0 || max_len > (1 << 30))
    return DIP_ERR_SHAPE;
  if (!aligned16(kc) || !aligned16(vc) || !aligned16(sc)) return DIP_ERR_ALIGN;
  return DIP_OK;
}

// The blocks of 32 rows that rows start .. start + n - 1 touch.
inline int64_t touched(int64_t start, int64_t n) {
  return (start + n - 1) / kKvBlock - start / kKvBlock + 1;
}

template <bool kNorm>
int launch_write(Kv4WriteArgs a, hipStream_t stream) {
  // a token at a position on the device is in one block, whichever it is
  a.vblocks = a.pos ? 1 : (int)touched(a.start, a.tokens);
  const int64_t tasks = (int64_t)a.vblocks * 4 * a.nkv +
                        (int64_t)a.tokens * (((kNorm ? a.nh + a.nkv : a.nkv) + 3) / 4);
  const int64_t grid = (tasks + kWriteWaves - 1) / kWriteWaves;
  if (!launch_fits(grid, 64 * kWriteWaves)) return DIP_ERR_SHAPE;
  hipLaunchKernelGGL((kv4_write_kernel<kNorm>), dim3((unsigned)grid), dim3(64 * kWriteWaves), 0,
                     stream, a);
  return hip_status(hipGetLastError());
}

int norm_rope(const uint16_t* qkv, const uint16_t* q_norm_w, const uint16_t* k_norm_w,
              const uint16_t* cos_table, const uint16_t* sin_table, const int64_t* pos,
              int64_t start, uint16_t* q_out, int8_t* k_cache, int8_t* v_cache,
              uint16_t* kv_scales, int64_t tokens, int64_t n_heads, int64_t n_kv_heads,
              int64_t head_dim, int64_t max_len, float eps, void* stream) {
  if (!qkv || !q_norm_w || !k_norm_w || !cos_table || !sin_table || !q_out) return DIP_ERR_NULL;
  if (head_dim != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (int st = check_cache(k_cache, v_cache, kv_scales, n_kv_heads, max_len)) return st;
  if (n_heads <= 0 || n_heads > 4096 || tokens < 0 || start < 0 || start > max_len ||
      tokens > max_len - start)
    return DIP_ERR_SHAPE;
  if (!(eps >= 0.f)) return DIP_ERR_ARG;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(cos_table) || !aligned16(sin_table) ||
      !aligned16(q_norm_w) || !aligned16(k_norm_w))
    return DIP_ERR_ALIGN;
  if (tokens == 0) return DIP_OK;
  const int64_t width = (n_heads + 2 * n_kv_heads) * kKvHeadDim;
  Kv4WriteArgs a{};
  a.k = qkv;
  a.v = qkv + (n_heads + n_kv_heads) * kKvHeadDim;
  a.k_tok = a.v_tok = width;
  a.k_head = a.v_head = kKvHeadDim;
  a.q_w = q_norm_w;
  a.k_w = k_norm_w;
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.q_out = q_out;
  a.pos = pos;
  a.start = start;
  a.kc = reinterpret_cast<uint32_t*>(k_cache);
  a.vc = reinterpret_cast<uint32_t*>(v_cache);
  a.sc = kv_scales;
  a.tokens = (int)tokens;
  a.nh = (int)n_heads;
  a.nkv = (int)n_kv_heads;
  a.max_len = (int)max_len;
  a.eps = eps;
  return launch_write<true>(a, (hipStream_t)stream);
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" int dip_kv4_write(const uint16_t* k, const uint16_t* v, int64_t k_tok_stride,
                             int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride,
                             int8_t* k_cache, int8_t* v_cache, uint16_t* kv_scales, int64_t start,
                             int64_t tokens, int64_t n_kv_heads, int64_t head_dim, int64_t max_len,
                             void* stream) {
  if (head_dim != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (int st = check_cache(k_cache, v_cache, kv_scales, n_kv_heads, max_len)) return st;
  if (tokens < 0 || start < 0 || start > max_len || tokens > max_len - start) return DIP_ERR_SHAPE;
  if (tokens == 0) return DIP_OK;
  if (!k || !v) return DIP_ERR_NULL;
  if (k_tok_stride < 0 || k_head_stride < 0 || v_tok_stride < 0 || v_head_stride < 0)
    return DIP_ERR_SHAPE;
  // pairs of values are loaded together
  if ((k_tok_stride | k_head_stride | v_tok_stride | v_head_stride) & 1 ||
      (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 3)
    return DIP_ERR_ALIGN;
  Kv4WriteArgs a{};
  a.k = k;
  a.v = v;
  a.k_tok = k_tok_stride;
  a.k_head = k_head_stride;
  a.v_tok = v_tok_stride;
  a.v_head = v_head_stride;
  a.k_vec = aligned16(k) && (k_tok_stride | k_head_stride) % 8 == 0;
  a.start = start;
  a.kc = reinterpret_cast<uint32_t*>(k_cache);
  a.vc = reinterpret_cast<uint32_t*>(v_cache);
  a.sc = kv_scales;
  a.tokens = (int)tokens;
  a.nkv = (int)n_kv_heads;
  a.max_len = (int)max_len;
  return launch_write<false>(a, (hipStream_t)stream);
}

extern "C" int dip_kv4_read(const int8_t* k_cache, const int8_t* v_cache,
                            const uint16_t* kv_scales, uint16_t* k_out, uint16_t* v_out,
                            int64_t start, int64_t rows, int64_t n_kv_heads, int64_t head_dim,
                            int64_t max_len, void* stream) {
  if (head_dim != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (int st = check_cache(k_cache, v_cache, kv_scales, n_kv_heads, max_len)) return st;
  if (rows < 0 || start < 0 || start > max_len || rows > max_len - start) return DIP_ERR_SHAPE;
  if (rows == 0) return DIP_OK;
  if (!k_out || !v_out) return DIP_ERR_NULL;
  if (!aligned16(k_out) || !aligned16(v_out)) return DIP_ERR_ALIGN;
  const int64_t blocks = touched(start, rows);
  const int64_t grid = blocks * n_kv_heads;  // four tasks of a block and head to a workgroup
  if (!launch_fits(grid, 64 * kWriteWaves)) return DIP_ERR_SHAPE;
  hipLaunchKernelGGL(kv4_read_kernel, dim3((unsigned)grid), dim3(64 * kWriteWaves), 0,
                     (hipStream_t)stream, reinterpret_cast<const uint32_t*>(k_cache),
                     reinterpret_cast<const uint32_t*>(v_cache), kv_scales,
                     reinterpret_cast<uint32_t*>(k_out), reinterpret_cast<uint32_t*>(v_out), start,
                     (int)rows, (int)n_kv_heads, (int)max_len, (int)blocks);
  return hip_status(hipGetLastError());
}

extern "C" int dip_qk_norm_rope_kv4(const uint16_t* qkv, const uint16_t* q_norm_w,
                                    const uint16_t* k_norm_w, const uint16_t* cos_table,
                                    const uint16_t* sin_table, const int64_t* pos,
                                    uint16_t* q_out, int8_t* k_cache, int8_t* v_cache,
                                    uint16_t* kv_scales, int64_t n_heads, int64_t n_kv_heads,
                                    int64_t head_dim, int64_t max_len, float eps, void* stream) {
  if (!pos) return DIP_ERR_NULL;
  return norm_rope(qkv, q_norm_w, k_norm_w, cos_table, sin_table, pos, 0, q_out, k_cache, v_cache,
                   kv_scales, 1, n_heads, n_kv_heads, head_dim, max_len, eps, stream);
}

extern "C" int dip_qk_norm_rope_kv4_rows(const uint16_t* qkv, const uint16_t* q_norm_w,
                                         const uint16_t* k_norm_w, const uint16_t* cos_table,
                                         const uint16_t* sin_table, int64_t start,
                                         uint16_t* q_out, int8_t* k_cache, int8_t* v_cache,
                                         uint16_t* kv_scales, int64_t tokens, int64_t n_heads,
                                         int64_t n_kv_heads, int64_t head_dim, int64_t max_len,
                                         float eps, void* stream) {
  return norm_rope(qkv, q_norm_w, k_norm_w, cos_table, sin_table, nullptr, start, q_out, k_cache,
                   v_cache, kv_scales, tokens, n_heads, n_kv_heads, head_dim, max_len, eps, stream);
}
