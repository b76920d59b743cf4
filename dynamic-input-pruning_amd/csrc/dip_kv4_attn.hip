// dip_kv4_attn.hip — grouped-query attention over the 4-bit key/value cache
// (dip_kv4.h): of one token at a position on the device, and of a prompt's
// tokens.
#include "dip_kv4.h"

#include <type_traits>

namespace dip {
namespace {

constexpr int kCols = 16;                  // (token, query head) pairs of a tile: MFMA columns
constexpr int kPart = kKvPart;
constexpr int kMaxSplits = 256;

// The tile's last token's rows, and the blocks of 32 rows that a wave of `waves`
// takes of them.
DIP_DEV int tile_rows(const Kv4AttnArgs& a, int64_t first, int tile) {
  const int last = min((tile * kCols + kCols - 1) / a.group, a.tokens - 1);
  return rows_at(first + last, a.max_len);
}
DIP_DEV int blocks_per_wave(int rows, int waves) {
  const int blocks = (rows + kKvBlock - 1) / kKvBlock;
  return max(1, (blocks + waves - 1) / waves);
}

DIP_DEV float scale_lo(uint32_t w) { return __uint_as_float(w << 16); }
DIP_DEV float scale_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// A tile of 16 columns, each a (token, query head) of one kv head, over the
// rows of one split, cut over the W waves of the workgroup.  Per block of 32
// rows a wave computes, all in registers:
//   scores^T: A = 16 keys as (1.5 + q / 16) / 256, B = the columns' queries, one MFMA
//     per group of 32 dimensions with -1.5 / 256 * (sum of the query's group) as its
//     start, so the result is (1 / 4096) sum q x exactly as numbers go; the group's
//     scale multiplies it, and the sum over the four groups is a score.  Lane (c, col)
//     ends up with the scores of rows 4 c + r and 16 + 4 c + r;
//   softmax against a base that follows the running maximum (the columns' lanes
//     agree on it by two lane swaps) in fp32;
//   values^T: B = bf16(weight * the row's value scale) of the group, where the
//     score is; A = 16 dimensions of the 32 rows as 1.5 + q / 16, and ones, whose
//     product is the sum that the 1.5 must not add.  (Rounding weight * scale to
//     bf16 is off by 2^-9 of itself, as any bf16 weight is.)
// Rows past a column's last get weight and scale 0, so what they hold, NaN
// scales too, does not count.
// A long cache is bound by memory: 131071 rows of 8 kv heads, 151 MB, 33 us (4.6
// TB/s, 93 % of a copy's rate).  Shorter ones by what comes before and after their
// few blocks of a wave: 20011 rows, 23 MB, 11 us; 701 rows in one launch, 16 blocks
// of rows to 8 waves, 9 us.  (With the MFMAs' sums in the accumulator half of the
// registers and every block masked 45 us at 131071 rows.)
template <int W>
__global__ __launch_bounds__(W * 64) void kv4_attn_kernel(Kv4AttnArgs a) {
  __shared__ float wm[W][kCols], wl[W][kCols];
  __shared__ __align__(16) float wacc[W][kCols][kKvHeadDim + 4];
  const int split = blockIdx.x % a.splits, kvh = blockIdx.x / a.splits % a.nkv;
  const int tile = blockIdx.x / a.splits / a.nkv;
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int l16 = l & 15, c = l >> 4;
  const int64_t first = a.pos ? *a.pos : a.start;
  const int rows = tile_rows(a, first, tile);
  const int bpw = blocks_per_wave(rows, a.splits * W);
  const int blocks = (rows + kKvBlock - 1) / kKvBlock;
  const bool direct = a.splits == 1;
  if (!direct && split * W * bpw >= blocks) return;
  const int b0 = min((split * W + wave) * bpw, blocks), b1 = min(b0 + bpw, blocks);

  const int col = tile * kCols + l16;
  const int tok = col / a.group, head = kvh * a.group + col % a.group;
  const bool on = tok < a.tokens;
  const int limit = on ? rows_at(first + tok, a.max_len) : 0;
  // rows that every column of the tile attends (columns without a token, whose
  // queries are 0, take them too: nothing reads their sums)
  const int sure = rows_at(first + tile * kCols / a.group, a.max_len);
  bf16x8_t bq[kKvGroups];
  float qs[kKvGroups];
  {
    const uint4* qp = reinterpret_cast<const uint4*>(
        a.q + ((size_t)tok * a.nkv * a.group + head) * kKvHeadDim);
#pragma unroll
    for (int g = 0; g < kKvGroups; ++g) {
      const uint4 w = on ? qp[4 * g + c] : make_uint4(0, 0, 0, 0);
      bq[g] = __builtin_bit_cast(bf16x8_t, u32x4_t{w.x, w.y, w.z, w.w});
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s = fmaf(scale_hi(x[e]), kKeyUnit, fmaf(scale_lo(x[e]), kKeyUnit, s));
      qs[g] = -kPairBias * row_pair_sum32(row_pair_sum16(s));
    }
  }
  const float sc2 = a.scale * kLog2e * (kPairScale / kKeyUnit);
  const uint32_t* kc = a.kc + (size_t)kvh * a.max_len * (kKvKeyBytes / 4);
  const uint32_t* vc = a.vc + (size_t)kvh * (a.max_len / kKvBlock) * kKvBlockWords;
  const uint4* sc = reinterpret_cast<const uint4*>(a.sc + (size_t)kvh * a.max_len * kKvScaleVals);
  const bf16x8_t ones = __builtin_bit_cast(
      bf16x8_t, u32x4_t{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});

  floatx4 acc[8], bias[kKvGroups];
#pragma unroll
  for (int t = 0; t < 8; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < kKvGroups; ++g) bias[g] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, den = 0.f;  // m: the base; den: this lane's rows only

  struct Raw {
    uint4 kw[2], vw[2], sw[2][4];
  };
  auto load = [&](Raw& x, int b) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x.kw[t] = reinterpret_cast<const uint4*>(kc)[(size_t)(b * kKvBlock + 16 * t + l16) * 4 + c];
      x.vw[t] = reinterpret_cast<const uint4*>(vc)[(size_t)b * (kKvBlockWords / 4) + 64 * t + l];
#pragma unroll
      for (int r = 0; r < 4; ++r) x.sw[t][r] = sc[b * kKvBlock + 16 * t + 4 * c + r];
    }
  };
  auto block = [&](const Raw& x, int b, auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
    const uint4(&kw)[2] = x.kw, (&vw)[2] = x.vw;
    const uint4(&sw)[2][4] = x.sw;
    float s[2][4];
    bool ok[2][4];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t w[4] = {kw[t].x, kw[t].y, kw[t].z, kw[t].w};
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < kKvGroups; ++g) {
        const floatx4 d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            kv4_biased<kKeyLower>(w[g]), bq[g], floatx4{qs[g], qs[g], qs[g], qs[g]}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t z = g < 2 ? sw[t][r].x : sw[t][r].y;
          v[r] = fmaf(g & 1 ? scale_hi(z) : scale_lo(z), d[r], v[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ok[t][r] = !kMasked || b * kKvBlock + 16 * t + 4 * c + r < limit;
        s[t][r] = ok[t][r] ? v[r] * sc2 : -INFINITY;
        mx = fmaxf(mx, s[t][r]);
      }
    }
    mx = fmaxf(m, row_pair_max32(row_pair_max16(mx)) + kDown);
    if (__any(mx > m + kSlack)) {
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - mx);  // what the sums so far are worth
      den *= f;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][r] *= f;
#pragma unroll
      for (int g = 0; g < kKvGroups; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) bias[g][r] *= f;
      m = mx;
    }
    float p[2][4];
    const float base = m == -INFINITY ? 0.f : m;  // (no score above -inf yet: weights 0, or NaN)
    {
      // Not one multiply-add from v: the base comes from the rounded scores, and beyond
      // 2^31 the rounding alone is further than weights reach.
#pragma clang fp contract(off)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[t][r] = ok[t][r] ? fast_exp2(s[t][r] - base) : 0.f;
          den += p[t][r];
        }
    }
    bf16x8_t va[8];
    {
      const uint32_t w[8] = {vw[0].x, vw[0].y, vw[0].z, vw[0].w,
                             vw[1].x, vw[1].y, vw[1].z, vw[1].w};
#pragma unroll
      for (int t = 0; t < 8; ++t) va[t] = kv4_biased(w[t]);
    }
#pragma unroll
    for (int g = 0; g < kKvGroups; ++g) {
      float ps[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t z = g < 2 ? sw[t][r].z : sw[t][r].w;
          const float v = g & 1 ? scale_hi(z) : scale_lo(z);
          ps[t][r] = ok[t][r] ? p[t][r] * v : 0.f;
        }
      const bf16x8_t bp = __builtin_bit_cast(
          bf16x8_t, u32x4_t{cvt_bf16x2(ps[0][0], ps[0][1]),
                            cvt_bf16x2(ps[0][2], ps[0][3]),
                            cvt_bf16x2(ps[1][0], ps[1][1]),
                            cvt_bf16x2(ps[1][2], ps[1][3])});
#pragma unroll
      for (int t = 2 * g; t < 2 * g + 2; ++t)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[t], bp, acc[t], 0, 0, 0);
      bias[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, bp, bias[g], 0, 0, 0);
    }
  };
  // two blocks in turn, the next one's loads in flight behind this one's work
  // (clamped, so that none is behind a branch and waited for with the others)
  if (b0 < b1) {
    const int full = min(b1, max(b0, sure / kKvBlock));  // blocks before it need no mask
    Raw x, y;
    load(x, b0);
    int b = b0;
    for (; b + 2 <= full; b += 2) {
      load(y, b + 1);
      block(x, b, std::false_type{});
      load(x, min(b + 2, b1 - 1));
      block(y, b + 1, std::false_type{});
    }
    for (; b < b1; ++b) {
      load(y, min(b + 1, b1 - 1));
      block(x, b, std::true_type{});
      x = y;
    }
  }

  // the waves' sums: lane (c, col) has dimensions 16 t + 4 c + r of column l16
  den = row_pair_sum32(row_pair_sum16(den));
  if (c == 0) {
    wm[wave][l16] = m;
    wl[wave][l16] = den;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    float4 o;
    o.x = kPairScale * fmaf(-kPairBias, bias[t >> 1][0], acc[t][0]);
    o.y = kPairScale * fmaf(-kPairBias, bias[t >> 1][1], acc[t][1]);
    o.z = kPairScale * fmaf(-kPairBias, bias[t >> 1][2], acc[t][2]);
    o.w = kPairScale * fmaf(-kPairBias, bias[t >> 1][3], acc[t][3]);
    *reinterpret_cast<float4*>(&wacc[wave][l16][16 * t + 4 * c]) = o;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kCols * kKvHeadDim / 2; e += W * 64) {
    const int cl = e / (kKvHeadDim / 2), d = e % (kKvHeadDim / 2) * 2;
    const int cc = tile * kCols + cl;
    if (cc >= a.tokens * a.group) break;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, wm[w][cl]);
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      // a wave without rows has m = -inf and sums 0; one whose scores are all NaN
      // has m = -inf and NaN sums, which must count
      const float f = wm[w][cl] == -INFINITY ? 1.f : fast_exp2(wm[w][cl] - mx);
      sum = fmaf(f, wl[w][cl], sum);
      o0 = fmaf(f, wacc[w][cl][d], o0);
      o1 = fmaf(f, wacc[w][cl][d + 1], o1);
    }
    if (direct) {
      const float inv = rows == 0 ? 0.f : 1.f / sum;  // (a sum of 0: every score is -inf)
      reinterpret_cast<uint32_t*>(a.out)[((size_t)(cc / a.group) * a.nkv * a.group +
                                          kvh * a.group + cc % a.group) * (kKvHeadDim / 2) +
                                         d / 2] =
          f32_to_bf16(o0 * inv) | (f32_to_bf16(o1 * inv) << 16);
    } else {
      float* o = a.part + ((size_t)blockIdx.x * kCols + cl) * kPart;
      if (d == 0) {
        o[0] = mx;
        o[1] = sum;
      }
      o[2 + d] = o0;
      o[3 + d] = o1;
    }
  }
}

// The splits of one column added up, in a fixed order: one workgroup per (kv
// head, column), kCombine groups of 128 threads, each of which takes every
// kCombine-th split's value sums; its first loads are in flight while the splits'
// weights are worked out.  (20011 rows, 64 columns: 4 us; one group of 128 threads
// over all splits in turn 18 to 22.)
constexpr int kCombine = 8, kAhead = 8;

__global__ __launch_bounds__(kCombine * kKvHeadDim) void kv4_combine_kernel(Kv4AttnArgs a,
                                                                            int waves) {
  __shared__ float wgt[kMaxSplits];
  __shared__ float red[kCombine * kKvHeadDim / 64][2];
  __shared__ float so[kCombine][kKvHeadDim];
  const int kvh = blockIdx.x % a.nkv, cc = blockIdx.x / a.nkv, tid = threadIdx.x;
  const int tile = cc / kCols, cl = cc % kCols, d = tid % kKvHeadDim, p = tid / kKvHeadDim;
  const int64_t first = a.pos ? *a.pos : a.start;
  const int rows = tile_rows(a, first, tile);
  const int per = waves * blocks_per_wave(rows, a.splits * waves);  // blocks of a split
  const int ns = ((rows + kKvBlock - 1) / kKvBlock + per - 1) / per;
  const size_t o = ((size_t)(cc / a.group) * a.nkv * a.group + kvh * a.group + cc % a.group) *
                   kKvHeadDim;
  if (ns == 0) {  // no rows
    if (tid < kKvHeadDim) a.out[o + tid] = 0;
    return;
  }
  const float* base = a.part + ((size_t)(tile * a.nkv + kvh) * a.splits * kCols + cl) * kPart;
  const size_t stride = (size_t)kCols * kPart;
  const float ms = tid < ns ? base[tid * stride] : -INFINITY;
  const float ls = tid < ns ? base[tid * stride + 1] : 0.f;
  float v[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) v[u] = base[min(p + kCombine * u, ns - 1) * stride + 2 + d];
  float mx = group_max<64>(ms);
  if ((tid & 63) == 0) red[tid >> 6][0] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kCombine * kKvHeadDim / 64; ++w) mx = fmaxf(mx, red[w][0]);
  // (a split without a score above -inf has sums of 0, or NaN, which must count)
  const float f = tid >= ns ? 0.f : ms == -INFINITY ? 1.f : fast_exp2(ms - mx);
  if (tid < kMaxSplits) wgt[tid] = f;
  const float part = group_sum<64>(f * ls);
  if ((tid & 63) == 0) red[tid >> 6][1] = part;
  __syncthreads();
  float acc = 0.f;
  for (int s0 = p; s0 < ns; s0 += kCombine * kAhead) {
    if (s0 != p) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) v[u] = base[min(s0 + kCombine * u, ns - 1) * stride + 2 + d];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (s0 + kCombine * u < ns) acc = fmaf(wgt[s0 + kCombine * u], v[u], acc);
  }
  so[p][d] = acc;
  __syncthreads();
  if (tid < kKvHeadDim) {
    float sum = 0.f, r = 0.f;
#pragma unroll
    for (int w = 0; w < kCombine * kKvHeadDim / 64; ++w) sum += red[w][1];
#pragma unroll
    for (int w = 0; w < kCombine; ++w) r += so[w][tid];
    a.out[o + tid] = (uint16_t)f32_to_bf16(r / sum);
  }
}

// How a launch cuts its tiles' rows.  Alone, a workgroup of 8 waves takes a tile's
// and writes the result itself; otherwise twice `pairs` workgroups of 4 waves (two
// to a CU) do, whose sums a second launch adds up.  `us` is about what it takes,
// from measured times: 3 us, 5 us and 1.6 us per block of a wave for each round of
// the workgroups, 6.5 us for the second launch (64 columns of 8 kv heads over 20000
// rows: 26 us, by this 30; 512 columns over 8000 rows: 51, 59; 1024 over 1000: 26,
// 29; 8 over 1000 in one launch 11, in two 13).  (Split tiles with 8 waves: 20011
// rows of 64 / 8 heads 15.2 us for 11.6.)
struct Cut {
  int pairs;
  int64_t us100;
  int waves() const { return pairs == 1 ? 8 : 4; }
  int splits() const { return pairs == 1 ? 1 : 2 * pairs; }
};

inline Cut cut_for(int64_t tiles, int64_t nkv, int64_t max_rows) {
  const int64_t blocks = (max_rows + kKvBlock - 1) / kKvBlock, cus = device_cus();
  const int64_t most = min((blocks + 7) / 8, (int64_t)kMaxSplits / 2);
  Cut best{1, INT64_MAX};
  for (int64_t s = 1; s <= most; s = s < 8 ? s + 1 : s + s / 8) {
    const int64_t rounds = (tiles * nkv * s + cus - 1) / cus;
    const int64_t per = (blocks + 8 * s - 1) / (8 * s);
    const int64_t us = 300 + rounds * (500 + 160 * per) + (s > 1 ? 650 : 0);
    if (us < best.us100) best = Cut{(int)s, us};
  }
  return best;
}

inline int64_t col_tiles(int64_t tokens, int64_t group) {
  return (tokens * group + kCols - 1) / kCols;
}

inline size_t part_bytes(int64_t tiles, int64_t nkv, int splits) {
  return splits == 1 ? 0 : (size_t)tiles * nkv * splits * kCols * kPart * sizeof(float);
}

int check_attn(const void* q, const void* kc, const void* vc, const void* sc, const void* out,
               int64_t tokens, int64_t nh, int64_t nkv, int64_t hd, int64_t max_len) {
  if (hd != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (!kc || !vc || !sc) return DIP_ERR_NULL;
  if (nkv <= 0 || nh <= 0 || nh % nkv != 0 || nh > 4096 || max_len <= 0 ||
      max_len % kKvBlock != 0 || max_len > (1 << 30) || tokens < 0 || tokens > max_len)
    return DIP_ERR_SHAPE;
  if (tokens > 0 && (!q || !out)) return DIP_ERR_NULL;
  if (!aligned16(q) || !aligned16(kc) || !aligned16(vc) || !aligned16(sc) || !aligned16(out))
    return DIP_ERR_ALIGN;
  return DIP_OK;
}

int launch_attn(Kv4AttnArgs a, int64_t tiles, Cut cut, hipStream_t stream) {
  a.splits = cut.splits();
  const int64_t grid = tiles * a.nkv * a.splits;
  const int64_t cols = (int64_t)a.tokens * a.group * a.nkv;
  if (!launch_fits(grid, 64 * cut.waves()) || cols > INT32_MAX ||
      (a.splits > 1 && !launch_fits(cols, kCombine * kKvHeadDim)))
    return DIP_ERR_SHAPE;
  if (cut.waves() == 8)
    hipLaunchKernelGGL((kv4_attn_kernel<8>), dim3((unsigned)grid), dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((kv4_attn_kernel<4>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(kv4_combine_kernel, dim3((unsigned)cols), dim3(kCombine * kKvHeadDim), 0,
                       stream, a, cut.waves());
  return hip_status(hipGetLastError());
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" size_t dip_kv4_decode_attention_workspace_size(int64_t n_heads, int64_t n_kv_heads,
                                                          int64_t head_dim, int64_t max_len) {
  if (head_dim != kKvHeadDim || n_heads <= 0 || n_heads > 4096 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || max_len <= 0 || max_len > (1 << 30))
    return 0;
  const int64_t tiles = col_tiles(1, n_heads / n_kv_heads);
  return part_bytes(tiles, n_kv_heads, cut_for(tiles, n_kv_heads, max_len).splits());
}

extern "C" int dip_kv4_decode_attention(const uint16_t* q, const int8_t* k_cache,
                                        const int8_t* v_cache, const uint16_t* kv_scales,
                                        const int64_t* pos, uint16_t* out, int64_t n_heads,
                                        int64_t n_kv_heads, int64_t head_dim, int64_t max_len,
                                        float scale, void* workspace, size_t ws_bytes,
                                        void* stream) {
  if (!pos) return DIP_ERR_NULL;
  if (int st = check_attn(q, k_cache, v_cache, kv_scales, out, 1, n_heads, n_kv_heads, head_dim,
                          max_len))
    return st;
  const int64_t group = n_heads / n_kv_heads, tiles = col_tiles(1, group);
  Kv4AttnArgs a{q, reinterpret_cast<const uint32_t*>(k_cache),
                reinterpret_cast<const uint32_t*>(v_cache), kv_scales, pos,
                static_cast<float*>(workspace), out, 0, 1, (int)n_kv_heads, (int)group,
                (int)max_len, 0, scale};
  const Cut cut = cut_for(tiles, n_kv_heads, max_len);
  const size_t need = part_bytes(tiles, n_kv_heads, cut.splits());
  if (need && (!workspace || ws_bytes < need)) return DIP_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return DIP_ERR_ALIGN;
  return launch_attn(a, tiles, cut, (hipStream_t)stream);
}

namespace {
// Whether a prompt goes over the cache expanded to bf16, in tiles of 128 columns,
// or through the token's kernel, 16 columns to a tile: the one that takes less by
// the two estimates (8 kv heads: from 2000 columns on over 300 rows, 800 over 3000,
// 200 over 20000).
inline bool by_tiles(int64_t tokens, int64_t start, int64_t nkv, int64_t group) {
  return prompt_tiles_us100(tokens, start, nkv, group) <
         cut_for(col_tiles(tokens, group), nkv, start + tokens).us100;
}
}  // namespace

extern "C" size_t dip_kv4_prompt_attention_workspace_size(int64_t tokens, int64_t start,
                                                          int64_t n_heads, int64_t n_kv_heads,
                                                          int64_t head_dim) {
  if (head_dim != kKvHeadDim || n_heads <= 0 || n_heads > 4096 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || tokens <= 0 || start < 0 || start > (1 << 30) || tokens > (1 << 30))
    return 0;
  const int64_t group = n_heads / n_kv_heads;
  if (by_tiles(tokens, start, n_kv_heads, group))
    return prompt_tiles_workspace(tokens, start, n_kv_heads, group);
  const int64_t tiles = col_tiles(tokens, group);
  return part_bytes(tiles, n_kv_heads, cut_for(tiles, n_kv_heads, start + tokens).splits());
}

extern "C" int dip_kv4_prompt_attention(const uint16_t* q, const int8_t* k_cache,
                                        const int8_t* v_cache, const uint16_t* kv_scales,
                                        int64_t start, uint16_t* out, int64_t tokens,
                                        int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                        int64_t max_len, float scale, void* workspace,
                                        size_t ws_bytes, void* stream) {
  if (int st = check_attn(q, k_cache, v_cache, kv_scales, out, tokens, n_heads, n_kv_heads,
                          head_dim, max_len))
    return st;
  if (start < 0 || start > max_len - tokens) return DIP_ERR_SHAPE;
  if (tokens == 0) return DIP_OK;
  const int64_t group = n_heads / n_kv_heads, tiles = col_tiles(tokens, group);
  Kv4AttnArgs a{q, reinterpret_cast<const uint32_t*>(k_cache),
                reinterpret_cast<const uint32_t*>(v_cache), kv_scales, nullptr,
                static_cast<float*>(workspace), out, start, (int)tokens, (int)n_kv_heads,
                (int)group, (int)max_len, 0, scale};
  const size_t need =
      dip_kv4_prompt_attention_workspace_size(tokens, start, n_heads, n_kv_heads, head_dim);
  if (need && (!workspace || ws_bytes < need)) return DIP_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return DIP_ERR_ALIGN;
  if (by_tiles(tokens, start, n_kv_heads, group))
    return launch_prompt_tiles(a, workspace, (hipStream_t)stream);
  return launch_attn(a, tiles, cut_for(tiles, n_kv_heads, start + tokens), (hipStream_t)stream);
}
