// dip_kv8_attn.hip — grouped-query attention over the paged 8-bit key/value cache
// (dip_kv8.h): of one or a few tokens of each of several sequences, at positions on
// the device, and of a prompt's tokens.
#include "dip_kv8.h"

namespace dip {
namespace {

struct Kv8AttnArgs {
  const uint16_t* q;  // [seqs, tokens, nkv * group, 128]
  Kv8Pages c;
  const int32_t* table;  // [seqs, width]
  const int64_t* pos;    // [seqs] first token's position, or null: `start`
  float* part;           // [seqs, tiles, nkv, splits, columns of a tile, kKvPart]
  uint16_t* out;         // [seqs, tokens, nkv * group, 128]
  int64_t start;
  int seqs, tokens, group, width;
  int tiles;   // of columns
  int per;     // pages of a split
  int splits;
  float scale;
};

// The first token's position of sequence s (behind every row: far, but no overflow).
DIP_DEV int64_t first_of(const Kv8AttnArgs& a, int s) {
  return a.pos ? min(a.pos[s], (int64_t)1 << 40) : a.start;
}
// The pages that the last token of a tile of `cols` columns attends.
DIP_DEV int tile_pages(const Kv8AttnArgs& a, int64_t first, int tile, int cols) {
  const int last = min((tile * cols + cols - 1) / a.group, a.tokens - 1);
  // (no token before row 0 is one: a sequence without a position has no rows)
  const int rows = first < 0 ? 0 : rows_at(first + last, a.width * kPageRows);
  return (rows + kPageRows - 1) / kPageRows;
}

// A tile of 16 CT columns, each a (token, query head) of one kv head of a sequence,
// over the pages of one split, in turn by the W waves of the workgroup.  Per page a
// wave computes, all in registers:
//   scores^T: A = 16 keys, B = the columns' queries, 16x16x32 MFMAs; lane (c, col) ends
//     up with the scores of rows 16 t + 4 c + r;
//   softmax against a base that follows the running maximum (the columns' lanes agree
//     on it by two lane swaps) in fp32;
//   values^T: A = 16 dimensions of 32 rows, B = the weights rounded to bf16 (off by
//     2^-8 of each at most) where the scores are.
// Keys and values become bf16 times their page's scale on the way, two to an
// instruction.
template <int W, int CT>
__global__ __launch_bounds__(W * 64) void kv8_attn_kernel(Kv8AttnArgs a) {
  constexpr int kCols = 16 * CT;
  __shared__ float wm[W][kCols], wl[W][kCols];
  __shared__ __align__(16) float wacc[W][kCols][kKvHeadDim + 4];
  const int nkv = a.c.nkv;
  const int split = blockIdx.x % a.splits, kvh = blockIdx.x / a.splits % nkv;
  const int tile = blockIdx.x / a.splits / nkv % a.tiles;
  const int seq = blockIdx.x / a.splits / nkv / a.tiles;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  const int l16 = l & 15, c = l >> 4;
  const int64_t first = first_of(a, seq);
  const int pages = tile_pages(a, first, tile, kCols);
  const bool direct = a.splits == 1;
  if (!direct && split * a.per >= pages) return;
  const int p0 = split * a.per + wave, p1 = min(split * a.per + a.per, pages);

  bf16x8_t bq[CT][4];
  int limit[CT];  // rows that the lane's columns attend
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = tile * kCols + 16 * ct + l16;
    const int tok = col / a.group, head = kvh * a.group + col % a.group;
    const bool on = tok < a.tokens && first >= 0;
    limit[ct] = on ? rows_at(first + tok, a.width * kPageRows) : 0;
    const uint4* qp = reinterpret_cast<const uint4*>(
        a.q + (((size_t)seq * a.tokens + tok) * nkv * a.group + head) * kKvHeadDim);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint4 w = on ? qp[8 * (g >> 1) + 2 * c + (g & 1)] : make_uint4(0, 0, 0, 0);
      bq[ct][g] = __builtin_bit_cast(bf16x8_t, u32x4_t{w.x, w.y, w.z, w.w});
    }
  }
  // rows that every column of the tile attends (columns without a token, whose
  // queries are 0, take them too: nothing reads their sums)
  const int sure = rows_at(first + tile * kCols / a.group, a.width * kPageRows);
  const float sc2 = a.scale * kLog2e;
  const int32_t* table = a.table + (size_t)seq * a.width;

  floatx4 acc[CT][8];
  float m[CT], den[CT];  // m: the base; den: this lane's rows only
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    den[ct] = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[ct][t] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  struct Raw {
    uint4 k[8], v[8];
    float2 scale;
  };
  auto load = [&](Raw& x, int id) {
    const size_t at = (size_t)max(id, 0) * nkv + kvh;
    const uint4* kp = reinterpret_cast<const uint4*>(a.c.k + at * kPageBytes) + 8 * l16 + c;
    const uint4* vp = reinterpret_cast<const uint4*>(a.c.v + at * kPageBytes) + 4 * l16 + c;
#pragma unroll
    for (int t = 0; t < 8; ++t) x.k[t] = kp[128 * (t >> 1) + 4 * (t & 1)];
#pragma unroll
    for (int t = 0; t < 8; ++t) x.v[t] = vp[64 * t];
    x.scale = *reinterpret_cast<const float2*>(a.c.scales + 2 * at);
  };
  auto number = [&](int p) {
    return __builtin_amdgcn_readfirstlane(page_number(table, min(p, p1 - 1), a.c.pages));
  };
  auto page = [&](Raw& x, int id, int p) {
    if (id < 0) {  // rows of no page: zeros
#pragma unroll
      for (int t = 0; t < 8; ++t) x.k[t] = x.v[t] = make_uint4(0, 0, 0, 0);
    }
    float s[CT][4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint4 lo = x.k[2 * t], hi = x.k[2 * t + 1];
      const bf16x8_t ka[4] = {
          kv8_operand(lo.x, lo.y, x.scale.x), kv8_operand(lo.z, lo.w, x.scale.x),
          kv8_operand(hi.x, hi.y, x.scale.x), kv8_operand(hi.z, hi.w, x.scale.x)};
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        floatx4 d{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < 4; ++g)
          d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[g], bq[ct][g], d, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[ct][t][r] = d[r] * sc2;
      }
    }
    const bool masked = (p + 1) * kPageRows > sure;
    const int row = p * kPageRows + 4 * c;  // of s[..][0][0]
    if (masked) {
      asm volatile("");  // a branch: comparisons and selections that most pages skip
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (row + 16 * (e >> 2) + (e & 3) >= limit[ct]) s[ct][e >> 2][e & 3] = -INFINITY;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[ct][e >> 2][e & 3]);
      mx = fmaxf(m[ct], row_pair_max32(row_pair_max16(mx)) + kDown);
      if (__any(mx > m[ct] + kSlack)) {
        // what the sums so far are worth
        const float f = m[ct] == -INFINITY ? 0.f : fast_exp2(m[ct] - mx);
        den[ct] *= f;
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[ct][t][r] *= f;
        m[ct] = mx;
      }
      // (no score above -inf yet: weights 0, or NaN)
      const float base = m[ct] == -INFINITY ? 0.f : m[ct];
      {
        // Not one multiply-add from the sum: the base comes from the rounded scores, and
        // beyond 2^31 the rounding alone is further than weights reach.
#pragma clang fp contract(off)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[ct][e >> 2][e & 3] = fast_exp2(s[ct][e >> 2][e & 3] - base);
      }
    }
    if (masked) {
      asm volatile("");
      uint32_t some = 0u;
      // weights of 0, whatever a base of +inf or NaN made of them
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (row + 16 * (e >> 2) + (e & 3) >= limit[ct]) s[ct][e >> 2][e & 3] = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t)
        some |= kv8_nan_bytes(x.v[t].x) | kv8_nan_bytes(x.v[t].y) | kv8_nan_bytes(x.v[t].z) |
                kv8_nan_bytes(x.v[t].w);
      if (__any(some != 0u)) {
        // A NaN counts for the columns that attend its row alone: it is taken out of the
        // values, and a product of ones where NaN is with ones where a column attends
        // says which sums it belongs to.
        bf16x8_t there[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4_t w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = row + 32 * h + 16 * (e >> 1) + 2 * (e & 1);
              w[e] = (r < limit[ct] ? 0x3F80u : 0u) | (r + 1 < limit[ct] ? 0x3F800000u : 0u);
            }
            there[ct][h] = __builtin_bit_cast(bf16x8_t, w);
          }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const uint4 w = x.v[t];
          const uint4 n = make_uint4(kv8_nan_bytes(w.x), kv8_nan_bytes(w.y), kv8_nan_bytes(w.z),
                                     kv8_nan_bytes(w.w));
          x.v[t] = make_uint4(w.x & ~n.x, w.y & ~n.y, w.z & ~n.z, w.w & ~n.w);
          const uint32_t one = 0x38383838u;  // 1.0
          const bf16x8_t a0 = kv8_operand(n.x & one, n.y & one, 1.f);
          const bf16x8_t a1 = kv8_operand(n.z & one, n.w & one, 1.f);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            floatx4 d{0.f, 0.f, 0.f, 0.f};
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, there[ct][0], d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, there[ct][1], d, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[ct][t][r] = d[r] > 0.f ? NAN : acc[ct][t][r];
          }
        }
      }
    }
    bf16x8_t bp[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float(&p)[4] = s[ct][2 * h], (&q)[4] = s[ct][2 * h + 1];
#pragma unroll
        for (int r = 0; r < 4; ++r) den[ct] += p[r] + q[r];
        bp[ct][h] = __builtin_bit_cast(
            bf16x8_t, u32x4_t{cvt_bf16x2(p[0], p[1]), cvt_bf16x2(p[2], p[3]),
                              cvt_bf16x2(q[0], q[1]), cvt_bf16x2(q[2], q[3])});
      }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const bf16x8_t a0 = kv8_operand(x.v[t].x, x.v[t].y, x.scale.y);
      const bf16x8_t a1 = kv8_operand(x.v[t].z, x.v[t].w, x.scale.y);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        acc[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, bp[ct][0], acc[ct][t], 0, 0, 0);
        acc[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, bp[ct][1], acc[ct][t], 0, 0, 0);
      }
    }
  };
  // the next page's loads in flight behind this one's work, its number read before
  if (p0 < p1) {
    Raw x, y;
    int id = number(p0), next = number(p0 + W), p = p0;
    load(x, id);
    for (; p + W < p1; p += W) {
      load(y, next);
      const int after = number(p + 2 * W);
      page(x, id, p);
      x = y;
      id = next;
      next = after;
    }
    page(x, id, p);
  }

  // the waves' sums: lane (c, col) has dimensions 16 t + 4 c + r of its columns
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float sum = row_pair_sum32(row_pair_sum16(den[ct]));
    if (c == 0) {
      wm[wave][16 * ct + l16] = m[ct];
      wl[wave][16 * ct + l16] = sum;
    }
#pragma unroll
    for (int t = 0; t < 8; ++t)
      *reinterpret_cast<float4*>(&wacc[wave][16 * ct + l16][16 * t + 4 * c]) =
          make_float4(acc[ct][t][0], acc[ct][t][1], acc[ct][t][2], acc[ct][t][3]);
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
      const float inv = pages == 0 ? 0.f : 1.f / sum;  // (a sum of 0: every score is -inf)
      reinterpret_cast<uint32_t*>(
          a.out)[(((size_t)seq * a.tokens + cc / a.group) * nkv * a.group + kvh * a.group +
                  cc % a.group) * (kKvHeadDim / 2) + d / 2] =
          f32_to_bf16(o0 * inv) | (f32_to_bf16(o1 * inv) << 16);
    } else {
      float* o = a.part + ((size_t)blockIdx.x * kCols + cl) * kKvPart;
      if (d == 0) {
        o[0] = mx;
        o[1] = sum;
      }
      o[2 + d] = o0;
      o[3 + d] = o1;
    }
  }
}

// The splits of a column added up: a workgroup per (sequence, column, kv head).
__global__ __launch_bounds__(kCombine * kKvHeadDim) void kv8_combine_kernel(Kv8AttnArgs a,
                                                                            int cols) {
  const int nkv = a.c.nkv, all = a.tokens * a.group;
  const int kvh = blockIdx.x % nkv, cc = blockIdx.x / nkv % all, seq = blockIdx.x / nkv / all;
  const int tile = cc / cols, cl = cc % cols;
  const int pages = tile_pages(a, first_of(a, seq), tile, cols);
  combine_splits(
      a.part + ((((size_t)seq * a.tiles + tile) * nkv + kvh) * a.splits * cols + cl) * kKvPart,
      (size_t)cols * kKvPart, (pages + a.per - 1) / a.per,
      a.out + (((size_t)seq * a.tokens + cc / a.group) * nkv * a.group + kvh * a.group +
               cc % a.group) * kKvHeadDim);
}

// A page of a head expanded for a prompt (dip_attn.h), two blocks of 32 rows: a
// workgroup per (kv head, page).  The keys by (8 dimensions, row), the values by
// dimension, of which a thread has all 64 rows.
__global__ __launch_bounds__(256) void kv8_expand_kernel(Kv8Pages a, const int32_t* table,
                                                         int width, uint4* work, uint32_t* bad,
                                                         int pages) {
  const int page = blockIdx.x % pages, kvh = blockIdx.x / pages, tid = threadIdx.x;
  const int id = page < width ? page_number(table, page, a.pages) : -1;
  uint4* out = work + (size_t)blockIdx.x * 2 * kBlockVecs;
  if (id < 0) {
    for (int i = tid; i < 2 * kBlockVecs; i += 256) out[i] = make_uint4(0, 0, 0, 0);
    if (tid < 2) bad[2 * blockIdx.x + tid] = ~0u;
    return;
  }
  const size_t at = (size_t)id * a.nkv + kvh;
  const float2 sc = *reinterpret_cast<const float2*>(a.scales + 2 * at);
  auto put = [](uint4* p, bf16x8_t v) {
    const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
    *p = make_uint4(w.x, w.y, w.z, w.w);
  };
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = tid & 63, u = 4 * n + (tid >> 6);
    const uint2 w = *reinterpret_cast<const uint2*>(a.k + at * kPageBytes + row * kKvHeadDim + 8 * u);
    put(out + (row >> 5) * kBlockVecs + u * 32 + (row & 31), kv8_operand(w.x, w.y, sc.x));
  }
  const int d = tid & 127, b = tid >> 7;  // dimension, block
  uint2 w[4];                             // rows 16 t + 4 c + 0 .. 3 of the block at t = 0, 1
#pragma unroll
  for (int c = 0; c < 4; ++c)
    w[c] = *reinterpret_cast<const uint2*>(a.v + at * kPageBytes + d * kPageRows + 16 * c + 8 * b);
  uint32_t first = 255u;  // row with a NaN
#pragma unroll
  for (int c = 3; c >= 0; --c) {
#pragma unroll
    for (int t = 1; t >= 0; --t) {
      uint32_t& x = t ? w[c].y : w[c].x;
      const uint32_t n = kv8_nan_bytes(x);
      if (n) first = min(first, (uint32_t)(16 * t + 4 * c) + ((uint32_t)__builtin_ctz(n) >> 3));
      x &= ~n;
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      put(out + b * kBlockVecs + 512 + (2 * t + h) * 128 + d,
          kv8_operand(t ? w[h].y : w[h].x, t ? w[2 + h].y : w[2 + h].x, sc.y));
  // a group's dimensions have their NaNs in the same rows
  const uint32_t byte = first << (8 * ((d >> 5) & 3));
  __shared__ uint32_t found[2][4];
  if ((d & 31) == 0) found[b][d >> 5] = byte;
  __syncthreads();
  if (tid < 2)
    bad[2 * blockIdx.x + tid] = found[tid][0] | found[tid][1] | found[tid][2] | found[tid][3];
}

// How a launch cuts its work: columns in tiles of 16 ct, a sequence's pages into
// splits of `per`.
struct Cut {
  int ct, tiles, per, splits;
  size_t part_bytes(int64_t seqs, int64_t nkv) const {
    return splits == 1 ? 0
                       : (size_t)seqs * tiles * nkv * splits * 16 * ct * kKvPart * sizeof(float);
  }
};

inline Cut cut_for(int64_t seqs, int64_t tokens, int64_t nkv, int64_t group, int64_t width) {
  Cut c;
  const int64_t cols = tokens * group;
  c.ct = cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
  c.tiles = (int)((cols + 16 * c.ct - 1) / (16 * c.ct));
  const int64_t heads = seqs * c.tiles * nkv;
  int64_t per = (width * heads + 1023) / 1024;
  per = max(min(per, (int64_t)64), (int64_t)4);
  per = max(per, (width + kMaxSplits - 1) / kMaxSplits);
  if (width <= 16) per = width;
  c.per = (int)per;
  c.splits = (int)((width + per - 1) / per);
  return c;
}

int check_attn(const void* q, const void* out, int64_t seqs, int64_t tokens, int64_t nh,
               int64_t nkv, int64_t hd) {
  if (hd != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (nkv <= 0 || nh <= 0 || nh % nkv != 0 || nh > 4096 || seqs < 0 || seqs > (1 << 24) ||
      tokens < 0 || tokens > (1 << 30) || seqs * tokens * nh > INT32_MAX)
    return DIP_ERR_SHAPE;
  if (!aligned16(q) || !aligned16(out)) return DIP_ERR_ALIGN;
  return DIP_OK;
}

template <int W, int CT>
void launch_tiles(const Kv8AttnArgs& a, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((kv8_attn_kernel<W, CT>), dim3((unsigned)grid), dim3(64 * W), 0, stream, a);
}

int launch_attn(Kv8AttnArgs a, const Cut& cut, hipStream_t stream) {
  a.tiles = cut.tiles;
  a.per = cut.per;
  a.splits = cut.splits;
  const int64_t grid = (int64_t)a.seqs * cut.tiles * a.c.nkv * cut.splits;
  const int64_t cols = (int64_t)a.seqs * a.tokens * a.group * a.c.nkv;
  if (!launch_fits(grid, 512) ||
      (cut.splits > 1 && !launch_fits(cols, kCombine * kKvHeadDim)))
    return DIP_ERR_SHAPE;
  if (cut.ct == 1 && cut.splits == 1)
    launch_tiles<8, 1>(a, grid, stream);
  else if (cut.ct == 1)
    launch_tiles<4, 1>(a, grid, stream);
  else if (cut.ct == 2)
    launch_tiles<4, 2>(a, grid, stream);
  else
    launch_tiles<4, 4>(a, grid, stream);
  if (cut.splits > 1)
    hipLaunchKernelGGL(kv8_combine_kernel, dim3((unsigned)cols), dim3(kCombine * kKvHeadDim), 0,
                       stream, a, 16 * cut.ct);
  return hip_status(hipGetLastError());
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" size_t dip_kv8_decode_attention_workspace_size(int64_t seqs, int64_t tokens,
                                                          int64_t n_heads, int64_t n_kv_heads,
                                                          int64_t head_dim, int64_t table_width) {
  if (head_dim != kKvHeadDim || n_heads <= 0 || n_heads > 4096 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || seqs <= 0 || seqs > (1 << 24) || tokens <= 0 ||
      tokens > (1 << 30) || seqs * tokens * n_heads > INT32_MAX || table_width <= 0 ||
      table_width > (1 << 24))
    return 0;
  return cut_for(seqs, tokens, n_kv_heads, n_heads / n_kv_heads, table_width)
      .part_bytes(seqs, n_kv_heads);
}

extern "C" int dip_kv8_decode_attention(const uint16_t* q, const uint8_t* k_cache,
                                        const uint8_t* v_cache, const float* kv_scales,
                                        int64_t pages, const int32_t* table, int64_t table_width,
                                        const int64_t* pos, uint16_t* out, int64_t seqs,
                                        int64_t tokens, int64_t n_heads, int64_t n_kv_heads,
                                        int64_t head_dim, float scale, void* workspace,
                                        size_t ws_bytes, void* stream) {
  if (int st = check_attn(q, out, seqs, tokens, n_heads, n_kv_heads, head_dim)) return st;
  if (int st = check_pages(k_cache, v_cache, kv_scales, pages, n_kv_heads, table, seqs,
                           table_width))
    return st;
  if (tokens == 0 || seqs == 0) return DIP_OK;
  if (!q || !out || !pos) return DIP_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(pos) & 7) return DIP_ERR_ALIGN;
  const int64_t group = n_heads / n_kv_heads;
  const Cut cut = cut_for(seqs, tokens, n_kv_heads, group, table_width);
  const size_t need = cut.part_bytes(seqs, n_kv_heads);
  if (need && (!workspace || ws_bytes < need)) return DIP_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return DIP_ERR_ALIGN;
  const Kv8AttnArgs a{q,
                      Kv8Pages{const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache),
                               const_cast<float*>(kv_scales), (int)pages, (int)n_kv_heads},
                      table, pos, static_cast<float*>(workspace), out, 0, (int)seqs, (int)tokens,
                      (int)group, (int)table_width, 0, 0, 0, scale};
  return launch_attn(a, cut, (hipStream_t)stream);
}

namespace {
// Whether a prompt goes over the cache expanded to bf16, in tiles of 128 columns.
inline bool by_tiles(int64_t tokens, int64_t group) { return tokens * group > 256; }
}  // namespace

extern "C" size_t dip_kv8_prompt_attention_workspace_size(int64_t tokens, int64_t start,
                                                          int64_t n_heads, int64_t n_kv_heads,
                                                          int64_t head_dim) {
  if (head_dim != kKvHeadDim || n_heads <= 0 || n_heads > 4096 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || tokens <= 0 || start < 0 || start > (1 << 30) ||
      tokens * n_heads > INT32_MAX)
    return 0;
  const int64_t group = n_heads / n_kv_heads;
  if (by_tiles(tokens, group)) return prompt_tiles_workspace(tokens, start, n_kv_heads, group);
  return cut_for(1, tokens, n_kv_heads, group, (start + tokens + kPageRows - 1) / kPageRows)
      .part_bytes(1, n_kv_heads);
}

extern "C" int dip_kv8_prompt_attention(const uint16_t* q, const uint8_t* k_cache,
                                        const uint8_t* v_cache, const float* kv_scales,
                                        int64_t pages, const int32_t* table, int64_t table_width,
                                        int64_t start, uint16_t* out, int64_t tokens,
                                        int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                        float scale, void* workspace, size_t ws_bytes,
                                        void* stream) {
  if (int st = check_attn(q, out, 1, tokens, n_heads, n_kv_heads, head_dim)) return st;
  if (int st = check_pages(k_cache, v_cache, kv_scales, pages, n_kv_heads, table, 1, table_width))
    return st;
  if (start < 0 || start > table_width * kPageRows - tokens) return DIP_ERR_SHAPE;
  if (tokens == 0) return DIP_OK;
  if (!q || !out) return DIP_ERR_NULL;
  const int64_t group = n_heads / n_kv_heads;
  const int64_t used = (start + tokens + kPageRows - 1) / kPageRows;
  const size_t need =
      dip_kv8_prompt_attention_workspace_size(tokens, start, n_heads, n_kv_heads, head_dim);
  if (need && (!workspace || ws_bytes < need)) return DIP_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return DIP_ERR_ALIGN;
  const Kv8Pages c{const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache),
                   const_cast<float*>(kv_scales), (int)pages, (int)n_kv_heads};
  hipStream_t s = (hipStream_t)stream;
  if (by_tiles(tokens, group)) {
    PromptArgs p{q, out, start, (int)tokens, (int)n_kv_heads, (int)group, scale};
    if (int st = prompt_tiles_plan(p, workspace)) return st;
    hipLaunchKernelGGL(kv8_expand_kernel, dim3((unsigned)(n_kv_heads * (p.blocks / 2))), dim3(256),
                       0, s, c, table, (int)table_width, const_cast<uint4*>(p.work),
                       const_cast<uint32_t*>(p.bad), p.blocks / 2);
    return launch_prompt_tiles(p, s);
  }
  const Kv8AttnArgs a{q, c, table, nullptr, static_cast<float*>(workspace), out, start, 1,
                      (int)tokens, (int)group, (int)used, 0, 0, 0, scale};
  return launch_attn(a, cut_for(1, tokens, n_kv_heads, group, used), s);
}
