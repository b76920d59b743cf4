// dip_kv8_attn.hip — grouped-query attention over the paged 8-bit key/value cache
// (dip_kv8.h): of one or a few tokens of each of several sequences, at positions on
// the device, and of a prompt's tokens.
#include "dip_kv8.h"

#include <type_traits>

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
  int per;     // pages of a split, at least
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

// The pages of a split of a sequence that has `pages`.
DIP_DEV int pages_per_split(const Kv8AttnArgs& a, int pages) {
  return max(a.per, (pages + a.splits - 1) / a.splits);
}

// A workgroup's share.  Workgroups go to the 8 XCDs in turn: the heads of a split come
// one after the other, so that an XCD gets all splits alike, of which the later ones have
// less to do where lengths differ.  (By splits first, 32 sequences of up to 16384 rows,
// four splits: 138 us.)
struct Task {
  int split, kvh, tile, seq;
  DIP_DEV explicit Task(const Kv8AttnArgs& a) {
    const int heads = a.seqs * a.tiles * a.c.nkv, head = blockIdx.x % heads;
    split = blockIdx.x / heads;
    kvh = head % a.c.nkv;
    tile = head / a.c.nkv % a.tiles;
    seq = head / a.c.nkv / a.tiles;
  }
  DIP_DEV size_t part(const Kv8AttnArgs& a) const {
    return (((size_t)seq * a.tiles + tile) * a.c.nkv + kvh) * a.splits + split;
  }
};

// What a wave has of 16 columns, each a (token, query head) of one kv head of a
// sequence: lane (c, l16) of column l16 the queries' operand, the sums of dimensions 16 t
// + 4 c + r, and the softmax's base and sum.
//
// kFine: the weights in two bf16 parts, off by 2^-17 of each, for a second product of
// each 32 rows; else in one, off by 2^-8 of each at most.  Where memory bounds the kernel
// the second product is hidden: 1 token over 701 rows 9.6 us for 9.3, of 32 sequences of up
// to 16384 118.7 for 118.1, over 131071 57.4 for 56.7, and the results are those of 32-bit
// weights but for some of the result's own roundings.  Where the products and the softmax
// bound it it is not: 5 tokens of 6 sequences of up to 20011 47.9 for 43.1, a prompt of
// 4096 379 for 284, 509 tokens behind 16003 386 for 292.  Those keep one part, as the
// attention over the 4-bit cache does.
template <bool kFine>
struct Columns {
  bf16x8_t q[4];
  floatx4 acc[8];
  float m, den;  // m: the base; den: this lane's rows only
  int limit;     // rows that the column attends
  int sure;      // rows that every column attends
  float scale2;  // to scores in powers of 2

  DIP_DEV Columns(const Kv8AttnArgs& a, int seq, int kvh, int64_t first, int col0, int l16, int c) {
    const int nkv = a.c.nkv, col = col0 + l16, tok = col / a.group;
    const int head = kvh * a.group + col % a.group;
    const bool on = tok < a.tokens && first >= 0;
    limit = on ? rows_at(first + tok, a.width * kPageRows) : 0;
    // (columns without a token, whose queries are 0, take them too: nothing reads
    // their sums)
    sure = rows_at(first + col0 / a.group, a.width * kPageRows);
    scale2 = a.scale * kLog2e;
    const uint4* qp = reinterpret_cast<const uint4*>(
        a.q + (((size_t)seq * a.tokens + tok) * nkv * a.group + head) * kKvHeadDim);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint4 w = on ? qp[8 * (g >> 1) + 2 * c + (g & 1)] : make_uint4(0, 0, 0, 0);
      q[g] = __builtin_bit_cast(bf16x8_t, u32x4_t{w.x, w.y, w.z, w.w});
    }
    m = -INFINITY;
    den = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  // Whether some column of the wave does not attend all of a page.
  DIP_DEV bool masks(int page) const { return (page + 1) * kPageRows > sure; }

  // Adds a page's rows, kMasked if it masks some.  keys(t, i) and values(t): the lane's 16
  // bytes of the page, of row 16 t + l16 from dimension 64 i + 16 c on, and of dimension
  // 16 t + l16.
  //   scores^T: A = 16 keys, B = the columns' queries, 16x16x32 MFMAs; lane (c, col) ends
  //     up with the scores of rows 16 t + 4 c + r;
  //   softmax against a base that follows the running maximum (the columns' lanes agree
  //     on it by two lane swaps) in fp32;
  //   values^T: A = 16 dimensions of 32 rows, B = the weights in bf16 parts where the
  //     scores are.
  // Keys and values become bf16 times their page's scale on the way, two to an
  // instruction.
  template <bool kMasked, typename K, typename V>
  DIP_DEV void add(K keys, V values, float2 scale, int page, int c) {
    float s[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint4 lo = keys(t, 0), hi = keys(t, 1);
      floatx4 d{0.f, 0.f, 0.f, 0.f};
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand(lo.x, lo.y, scale.x), q[0], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand(lo.z, lo.w, scale.x), q[1], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand(hi.x, hi.y, scale.x), q[2], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand(hi.z, hi.w, scale.x), q[3], d, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][r] = d[r] * scale2;
    }
    const int row = page * kPageRows + 4 * c;  // of s[0][0]
    if (kMasked) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (row + 16 * (e >> 2) + (e & 3) >= limit) s[e >> 2][e & 3] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
    mx = fmaxf(m, row_pair_max32(row_pair_max16(mx)) + kDown);
    if (__any(mx > m + kSlack)) {
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - mx);  // what the sums so far are worth
      den *= f;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][r] *= f;
      m = mx;
    }
    const float base = m == -INFINITY ? 0.f : m;  // (no score above -inf yet: weights 0, or NaN)
    {
      // Not one multiply-add from the sum: the base comes from the rounded scores, and
      // beyond 2^31 the rounding alone is further than weights reach.
#pragma clang fp contract(off)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e >> 2][e & 3] = fast_exp2(s[e >> 2][e & 3] - base);
    }
    if (kMasked) {
      // weights of 0, whatever a base of +inf or NaN made of them
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (row + 16 * (e >> 2) + (e & 3) >= limit) s[e >> 2][e & 3] = 0.f;
    }
    bf16x8_t p[2], rest[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float(&x)[4] = s[2 * h], (&y)[4] = s[2 * h + 1];
#pragma unroll
      for (int r = 0; r < 4; ++r) den += x[r] + y[r];
      const u32x4_t w{cvt_bf16x2(x[0], x[1]), cvt_bf16x2(x[2], x[3]), cvt_bf16x2(y[0], y[1]),
                      cvt_bf16x2(y[2], y[3])};
      p[h] = __builtin_bit_cast(bf16x8_t, w);
      if (kFine)
        rest[h] = __builtin_bit_cast(bf16x8_t,
                                     u32x4_t{left_of(x[0], x[1], w[0]), left_of(x[2], x[3], w[1]),
                                             left_of(y[0], y[1], w[2]), left_of(y[2], y[3], w[3])});
    }
    if (!kMasked) {
#pragma unroll
      for (int t = 0; t < 8; ++t) product(t, values(t), p, rest, scale.y);
      return;
    }
    // A NaN counts for the columns that attend its row alone: it is taken out of the values,
    // and a product of ones where NaN is with ones where a column attends says which sums
    // it belongs to.
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const uint4 w = values(t), n = nans(w);
      product(t, make_uint4(w.x & ~n.x, w.y & ~n.y, w.z & ~n.z, w.w & ~n.w), p, rest, scale.y);
      if (!__any((n.x | n.y | n.z | n.w) != 0u)) continue;
      bf16x8_t there[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4_t o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = row + 32 * h + 16 * (e >> 1) + 2 * (e & 1);
          o[e] = (r < limit ? 0x3F80u : 0u) | (r + 1 < limit ? 0x3F800000u : 0u);
        }
        there[h] = __builtin_bit_cast(bf16x8_t, o);
      }
      constexpr uint32_t kOne = 0x38383838u;
      floatx4 d{0.f, 0.f, 0.f, 0.f};
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand(n.x & kOne, n.y & kOne, 1.f),
                                                  there[0], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand(n.z & kOne, n.w & kOne, 1.f),
                                                  there[1], d, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[t][r] = d[r] > 0.f ? NAN : acc[t][r];
    }
  }

  DIP_DEV static uint4 nans(uint4 w) {
    return make_uint4(kv8_nan_bytes(w.x), kv8_nan_bytes(w.y), kv8_nan_bytes(w.z),
                      kv8_nan_bytes(w.w));
  }
  // What rounding to bf16 (a pair, in w) leaves of x and y, as bf16 too.
  DIP_DEV static uint32_t left_of(float x, float y, uint32_t w) {
    return cvt_bf16x2(x - __uint_as_float(w << 16), y - __uint_as_float(w & 0xFFFF0000u));
  }
  DIP_DEV void product(int t, uint4 w, const bf16x8_t (&p)[2], const bf16x8_t (&rest)[2],
                       float scale) {
    const bf16x8_t lo = kv8_operand(w.x, w.y, scale), hi = kv8_operand(w.z, w.w, scale);
    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, p[0], acc[t], 0, 0, 0);
    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, p[1], acc[t], 0, 0, 0);
    if (!kFine) return;
    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, rest[0], acc[t], 0, 0, 0);
    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, rest[1], acc[t], 0, 0, 0);
  }
};

// The 16-byte pieces of a page's keys (of values behind them) that an operand takes.
DIP_DEV int key_piece(int t, int i, int l16, int c) { return (16 * t + l16) * 8 + 4 * i + c; }
DIP_DEV int value_piece(int t, int l16, int c) { return (16 * t + l16) * 4 + c; }
constexpr int kPagePieces = kPageBytes / 16;

constexpr int kRawBuffer = 0x00027000;  // a buffer of bytes, bounds checked
DIP_DEV uint4 buffer_piece(__amdgpu_buffer_rsrc_t b, int piece) {
  const u32x4_t w =
      __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(b, 16 * piece, 0, 0));
  return make_uint4(w.x, w.y, w.z, w.w);
}

// Up to 16 columns: a workgroup of W waves takes a split's pages in turn, each wave
// with all columns, from memory into registers, 32 KB of a wave in flight.  Bound by
// memory: 32 sequences of up to 16384 rows (547 MB) 113 us, 4.9 TB/s, MFMA 12 % and VALU 35
// % busy; one of 131071 (268 MB) 53, 5.1 TB/s.  One of 701 rows, in one launch of 8 waves:
// 9.6 us of waits in a row.
template <int W>
__global__ __launch_bounds__(W * 64) void kv8_attn_kernel(Kv8AttnArgs a) {
  __shared__ float wm[W][16], wl[W][16];
  __shared__ __align__(16) float wacc[W][16][kKvHeadDim + 4];
  const int nkv = a.c.nkv;
  const Task task(a);
  const int split = task.split, kvh = task.kvh, seq = task.seq;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  const int l16 = l & 15, c = l >> 4;
  const int64_t first = first_of(a, seq);
  const int pages = tile_pages(a, first, 0, 16);
  const bool direct = a.splits == 1;
  const int per = pages_per_split(a, pages);
  if (!direct && split * per >= pages) return;
  const int p0 = split * per + wave, p1 = min(split * per + per, pages);
  const int32_t* table = a.table + (size_t)seq * a.width;
  Columns<true> x(a, seq, kvh, first, 0, l16, c);

  struct Raw {
    uint4 k[8], v[8];
    float2 scale;
  };
  // Page number id, or zeros where that is negative: the bounds of the buffer say so,
  // so the loads are behind no branch, which would have them all waited for where it ends.
  auto load = [&](Raw& r, int id) {
    const size_t at = (size_t)max(id, 0) * nkv + kvh;
    const int bytes = id < 0 ? 0 : kPageBytes;
    const auto kp = __builtin_amdgcn_make_buffer_rsrc(a.c.k + at * kPageBytes, 0, bytes, kRawBuffer);
    const auto vp = __builtin_amdgcn_make_buffer_rsrc(a.c.v + at * kPageBytes, 0, bytes, kRawBuffer);
#pragma unroll
    for (int t = 0; t < 8; ++t) r.k[t] = buffer_piece(kp, key_piece(t >> 1, t & 1, l16, c));
#pragma unroll
    for (int t = 0; t < 8; ++t) r.v[t] = buffer_piece(vp, value_piece(t, l16, c));
    r.scale = *reinterpret_cast<const float2*>(a.c.scales + 2 * at);
  };
  auto number = [&](int p) {
    const int id = page_number(table, min(p, p1 - 1), a.c.pages);
    return __builtin_amdgcn_readfirstlane(p < p1 ? id : -1);
  };
  // the next page's loads in flight behind this one's work, its number read before
  if (p0 < p1) {
    Raw r, s;
    int next = number(p0 + W), p = p0;
    load(r, number(p0));
    auto key = [&](int t, int i) { return r.k[2 * t + i]; };
    auto value = [&](int t) { return r.v[t]; };
    for (; p < p1 && !x.masks(p); p += W) {
      load(s, next);
      next = number(p + 2 * W);
      x.add<false>(key, value, r.scale, p, c);
      r = s;
    }
    for (; p < p1; p += W) {
      load(s, next);
      next = number(p + 2 * W);
      x.add<true>(key, value, r.scale, p, c);
      r = s;
    }
  }

  // the waves' sums
  const float sum = row_pair_sum32(row_pair_sum16(x.den));
  if (c == 0) {
    wm[wave][l16] = x.m;
    wl[wave][l16] = sum;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t)
    *reinterpret_cast<float4*>(&wacc[wave][l16][16 * t + 4 * c]) =
        make_float4(x.acc[t][0], x.acc[t][1], x.acc[t][2], x.acc[t][3]);
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * kKvHeadDim / 2; e += W * 64) {
    const int cl = e / (kKvHeadDim / 2), d = e % (kKvHeadDim / 2) * 2;
    if (cl >= a.tokens * a.group) break;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, wm[w][cl]);
    float all = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      // a wave without rows has m = -inf and sums 0; one whose scores are all NaN
      // has m = -inf and NaN sums, which must count
      const float f = wm[w][cl] == -INFINITY ? 1.f : fast_exp2(wm[w][cl] - mx);
      all = fmaf(f, wl[w][cl], all);
      o0 = fmaf(f, wacc[w][cl][d], o0);
      o1 = fmaf(f, wacc[w][cl][d + 1], o1);
    }
    if (direct) {
      const float inv = pages == 0 ? 0.f : 1.f / all;  // (a sum of 0: every score is -inf)
      reinterpret_cast<uint32_t*>(
          a.out)[(((size_t)seq * a.tokens + cl / a.group) * nkv * a.group + kvh * a.group +
                  cl % a.group) * (kKvHeadDim / 2) + d / 2] =
          f32_to_bf16(o0 * inv) | (f32_to_bf16(o1 * inv) << 16);
    } else {
      float* o = a.part + (task.part(a) * 16 + cl) * kKvPart;
      if (d == 0) {
        o[0] = mx;
        o[1] = all;
      }
      o[2 + d] = o0;
      o[3 + d] = o1;
    }
  }
}

constexpr int kWideWaves = 3;  // waves of a SIMD
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// More columns: a workgroup of W waves takes a split's pages one after the other, each
// wave with 16 columns of its own.  A page goes straight from memory to LDS, the next one
// while this one is worked on; its 16-byte pieces lie there in an order in which eight
// neighbouring lanes' are in different banks.  6 sequences of up to 20011 rows with 40
// columns (135 MB): 37 us, 3.8 TB/s, VALU 53 % and MFMA 18 % busy: the conversion and the
// softmax, and the wait for a page, of which three or four workgroups of a CU have one each
// under way.  (Each wave with all 40 columns, padded to
// 64, in registers: 68 us; masked pages and others in one loop, which spills: 39, a
// whole call 49 for 43; two pages under way, whose three buffers leave room for fewer
// workgroups: 10 more.)
template <int W>
__global__ __launch_bounds__(W * 64, kWideWaves) void kv8_wide_kernel(Kv8AttnArgs a) {
  __shared__ uint4 buf_a[2 * kPagePieces], buf_b[2 * kPagePieces];
  const int nkv = a.c.nkv;
  const Task task(a);
  const int split = task.split, kvh = task.kvh, tile = task.tile, seq = task.seq;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
  const int l16 = l & 15, c = l >> 4;
  const int64_t first = first_of(a, seq);
  const int pages = tile_pages(a, first, tile, 16 * W);
  const bool direct = a.splits == 1;
  const int per = pages_per_split(a, pages);
  const int p0 = split * per, p1 = min(p0 + per, pages);
  if (!direct && p0 >= pages) return;
  const int32_t* table = a.table + (size_t)seq * a.width;
  const int col0 = tile * 16 * W + 16 * wave;
  Columns<false> x(a, seq, kvh, first, col0, l16, c);

  // piece s of a buffer: keys of row s / 8, then values of dimension (s - 512) / 4
  constexpr int kLoads = (2 * kPagePieces / 64 + W - 1) / W;  // of a wave
  auto fetch = [&](uint4* buf, int id) {
    const size_t at = (size_t)max(id, 0) * nkv + kvh;
    const uint4* kp = reinterpret_cast<const uint4*>(a.c.k + at * kPageBytes);
    const uint4* vp = reinterpret_cast<const uint4*>(a.c.v + at * kPageBytes);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int at64 = min(n * W + wave, 2 * kPagePieces / 64 - 1);  // (the last one more than once)
      const int s = at64 * 64 + l;
      const uint4* src = at64 < kPagePieces / 64
                             ? kp + (s & ~7) + ((s ^ (s >> 3)) & 7)
                             : vp + ((s & ~3) - kPagePieces) + ((s ^ (s >> 3)) & 3);
      __builtin_amdgcn_global_load_lds((global_void*)src, (lds_void*)(buf + at64 * 64), 16, 0, 0);
    }
  };
  auto number = [&](int p) {
    return __builtin_amdgcn_readfirstlane(page_number(table, min(p, p1 - 1), a.c.pages));
  };
  auto scales = [&](int id) {
    return id < 0 ? make_float2(0.f, 0.f)
                  : *reinterpret_cast<const float2*>(a.c.scales + 2 * ((size_t)id * nkv + kvh));
  };
  auto add = [&](auto masked, const uint4* buf, int id, float2 scale, int p) {
    auto key = [&](int t, int i) {
      const int s = key_piece(t, i, l16, c);
      return buf[(s & ~7) + ((s ^ (s >> 3)) & 7)];
    };
    auto value = [&](int t) {
      const int s = kPagePieces + value_piece(t, l16, c);
      return buf[(s & ~3) + ((s ^ (s >> 3)) & 3)];
    };
    if constexpr (decltype(masked)::value) {
      const uint32_t there = id < 0 ? 0u : ~0u;  // (rows of no page: zeros)
      auto kept = [&](uint4 w) {
        return make_uint4(w.x & there, w.y & there, w.z & there, w.w & there);
      };
      x.add<true>([&](int t, int i) { return kept(key(t, i)); },
                  [&](int t) { return kept(value(t)); }, scale, p, c);
    } else {
      x.add<false>(key, value, scale, p, c);
    }
  };
  // this wave's pieces have landed, then everybody's, and the other buffer's readers
  // are through
  auto landed = [&] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  if (p0 < p1) {
    int id = number(p0), next = number(p0 + 1);
    float2 scale = scales(id);
    fetch(buf_a, id);
    int p = p0, at = 0;  // a page, and the buffer that it is in
    auto turn = [&](auto masked, const uint4* cur, uint4* free) {
      if (p >= p1 || (!decltype(masked)::value && (x.masks(p) || id < 0))) return false;
      landed();
      const float2 after = scales(next);
      const int then = number(p + 2);
      if (p + 1 < p1) fetch(free, next);
      add(masked, cur, id, scale, p);
      id = next, next = then, scale = after;
      ++p;
      return true;
    };
    // The pages that all of the wave's columns attend, then the others.  (A wave changes
    // loops by itself: each meets the others once a page in both.)
    while (turn(std::false_type{}, buf_a, buf_b) && (at = 1, turn(std::false_type{}, buf_b, buf_a)))
      at = 0;
    for (; p < p1; at ^= 1) {
      if (at == 0)
        turn(std::true_type{}, buf_a, buf_b);
      else
        turn(std::true_type{}, buf_b, buf_a);
    }
  }

  const float sum = row_pair_sum32(row_pair_sum16(x.den));
  const int cc = col0 + l16;
  if (cc >= a.tokens * a.group) return;
  if (direct) {
    const float inv = pages == 0 ? 0.f : 1.f / sum;  // (a sum of 0: every score is -inf)
    uint2* o = reinterpret_cast<uint2*>(
        a.out + (((size_t)seq * a.tokens + cc / a.group) * nkv * a.group + kvh * a.group +
                 cc % a.group) * kKvHeadDim);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      o[4 * t + c] = make_uint2(cvt_bf16x2(x.acc[t][0] * inv, x.acc[t][1] * inv),
                                cvt_bf16x2(x.acc[t][2] * inv, x.acc[t][3] * inv));
    return;
  }
  float* o = a.part + (task.part(a) * 16 * W + 16 * wave + l16) * kKvPart;
  if (c == 0) {
    o[0] = x.m;
    o[1] = sum;
  }
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2*>(o + 2 + 16 * t + 4 * c + 2 * r) =
          make_float2(x.acc[t][2 * r], x.acc[t][2 * r + 1]);
}

// The splits of a column (of a sequence and kv head) added up: by a wave where there are
// few of them, by four, or by a workgroup of 16, which fewer splits are worth where all of
// these run at once, two to a CU.  (1920 columns of 21 splits: 6.4 us by four waves each,
// 9.3 by one, 17 by 16; 40 of 64: 10 by four, 6 by 16; 64 of 16: 9.1 by one, 4.7 by 16; a
// whole call with 512 of 4: 14.8 by one, 16 by 16.)
template <int kWaves>
__global__ __launch_bounds__(kWaves == 16 ? 1024 : 256) void kv8_combine_kernel(Kv8AttnArgs a,
                                                                                int cols) {
  __shared__ float2 red[kWaves == 4 ? 4 : 1][64];
  const int nkv = a.c.nkv, all = a.tokens * a.group;
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int64_t at = kWaves == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
  if (kWaves == 1 && at >= (int64_t)a.seqs * all * nkv) return;
  const int kvh = (int)(at % nkv), cc = (int)(at / nkv % all), seq = (int)(at / nkv / all);
  const int tile = cc / cols, cl = cc % cols;
  const int pages = tile_pages(a, first_of(a, seq), tile, cols), per = pages_per_split(a, pages);
  const int ns = (pages + per - 1) / per;
  const float* base =
      a.part + ((((size_t)seq * a.tiles + tile) * nkv + kvh) * a.splits * cols + cl) * kKvPart;
  uint16_t* out = a.out + (((size_t)seq * a.tokens + cc / a.group) * nkv * a.group +
                           kvh * a.group + cc % a.group) * kKvHeadDim;
  const size_t stride = (size_t)cols * kKvPart;
  if (kWaves == 16)
    combine_splits(base, stride, ns, out);
  else
    combine_splits_waves<kWaves == 16 ? 4 : kWaves>(base, stride, ns, kWaves == 1 ? 0 : wave, l,
                                                    red, out);
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

// How a launch cuts its work: columns in tiles of 16 `waves` (0: up to 16 columns, with
// the waves taking pages in turn), a sequence's pages into splits of `per` at least.
//
// A single sequence's splits are one round of the workgroups that run at once, each with
// an even share of the pages there are.  Of several sequences, whose lengths only the
// device knows, a split is a share of the table's width that makes half as many
// workgroups again as run at once (narrow ones: three times as many), of which those
// behind a sequence's end leave at once.  In a graph, states in turn: 32 of up to 16384
// rows 120 us, with one round 134, with a round and a third 118, with two 130; 6 of up to
// 20011 with 5 tokens each 46, with one round 53, a third more 49, with two 67; with 3
// tokens each 41, 42, 44 and 57 (of two waves' workgroups five fit a CU, four are counted:
// with five 56).  Where the table is wider than the longest sequence's pages splits are
// longer and more workgroups leave: four times as wide the first takes 137 us for 120,
// the second 82 for 42 (one state).
// A split has a page for each wave at least, of several sequences 8: 4000 rows of one 10.8
// us with 4 for 14.0 with 8, 20011 rows 17.3 for 19.4; 8 sequences of 2000 15.8 for 13.9.
struct Cut {
  int waves, tiles, per, splits;
  int cols() const { return waves ? 16 * waves : 16; }
  size_t part_bytes(int64_t seqs, int64_t nkv) const {
    return splits == 1 ? 0
                       : (size_t)seqs * tiles * nkv * splits * cols() * kKvPart * sizeof(float);
  }
};

// More waves share a page's fetch, and fewer such workgroups fit a CU and wait for pages
// by turns: of 4 waves at most, and of 8, 80 columns of 1 sequence of 20000 rows of 64 / 8
// heads 33 us and 35, 128 35 and 33, 256 50 and 54; of 6 sequences of up to 20000 rows 79 and
// 90, 80 and 91, 142 and 174; of 32 of up to 6000 119 and 136, 127 and 143, 193 and 197; of
// 16 / 2 heads 6 sequences 35 and 47, 40 and 46, 50 and 87.  (Of 3 at most 64 columns 70 for
// 51 and 96 for 70 in the second and third.)
constexpr int kMaxWide = 4;

inline Cut cut_for(int64_t seqs, int64_t tokens, int64_t nkv, int64_t group, int64_t width) {
  Cut c;
  const int64_t cols = tokens * group;
  c.waves = cols <= 16 ? 0 : (int)min((cols + 15) / 16, (int64_t)kMaxWide);
  c.tiles = (int)((cols + c.cols() - 1) / c.cols());
  const int64_t heads = seqs * c.tiles * nkv;
  const int64_t cus = device_cus();
  // workgroups that run at once
  const int64_t slots = cus * (c.waves ? min(4 * kWideWaves / c.waves, 4) : 2);
  int64_t per = c.waves || seqs == 1 ? 4 : 8, splits;
  if (seqs == 1) {
    splits = min(max(slots / heads, (int64_t)1), (width + per - 1) / per);
  } else {
    const int64_t want = c.waves ? slots * 3 / 2 : 6 * cus;
    per = max((width * heads + want - 1) / want, per);
    splits = (width + per - 1) / per;
  }
  splits = min(splits, (int64_t)kMaxSplits);
  if (width <= 16) splits = 1;
  c.per = (int)per;
  c.splits = (int)splits;
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

int launch_attn(Kv8AttnArgs a, const Cut& cut, hipStream_t stream) {
  a.tiles = cut.tiles;
  a.per = cut.per;
  a.splits = cut.splits;
  const int64_t grid = (int64_t)a.seqs * cut.tiles * a.c.nkv * cut.splits;
  const int64_t cols = (int64_t)a.seqs * a.tokens * a.group * a.c.nkv;
  if (!launch_fits(grid, 512) || (cut.splits > 1 && !launch_fits(cols, kCombine * kKvHeadDim)))
    return DIP_ERR_SHAPE;
  const dim3 g((unsigned)grid);
  switch (cut.waves) {
    case 0:
      if (cut.splits == 1)
        hipLaunchKernelGGL(kv8_attn_kernel<8>, g, dim3(512), 0, stream, a);
      else
        hipLaunchKernelGGL(kv8_attn_kernel<4>, g, dim3(256), 0, stream, a);
      break;
    case 2: hipLaunchKernelGGL(kv8_wide_kernel<2>, g, dim3(128), 0, stream, a); break;
    case 3: hipLaunchKernelGGL(kv8_wide_kernel<3>, g, dim3(192), 0, stream, a); break;
    default: hipLaunchKernelGGL(kv8_wide_kernel<4>, g, dim3(256), 0, stream, a);
  }
  if (cut.splits > 32 || (cut.splits > 8 && cols <= 2 * device_cus()))
    hipLaunchKernelGGL(kv8_combine_kernel<16>, dim3((unsigned)cols), dim3(1024), 0, stream, a,
                       cut.cols());
  else if (cut.splits > 16)
    hipLaunchKernelGGL(kv8_combine_kernel<4>, dim3((unsigned)cols), dim3(256), 0, stream, a,
                       cut.cols());
  else if (cut.splits > 1)
    hipLaunchKernelGGL(kv8_combine_kernel<1>, dim3((unsigned)((cols + 3) / 4)), dim3(256), 0,
                       stream, a, cut.cols());
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
// Whether a prompt goes over the cache expanded to bf16, in tiles of 128 columns: where
// the columns of a kv head are worth the expansion of all rows before, which the kernels
// above do without.  Those take a page again for every 64 columns, but cut it into splits
// that fill the card from fewer columns where there are fewer heads.  Columns of a kv
// head, us by pages and by tiles, in a row:
//   64 / 8 heads, 16000 rows before  256 42 59, 512 67 71, 640 83 77, 1024 117 99
//                 6000               256 27 37, 512 40 42, 640 46 43, 1024 57 52
//                 500                128 19 17, 512 19 21, 1024 21 26 (none 7 10, 7 10, 8 12)
//   32 / 32       6000               256 57 73, 512 101 100, 640 142 114
//   32 / 4        16000              512 43 50, 768 55 56, 1024 67 62, 1536 92 76
//   16 / 2        16000              512 34 45, 1024 42 46, 1536 55 52, 2048 68 58
//   8 / 1         16000              512 23 39, 1024 34 43, 2048 43 45, 4096 68 56
inline bool by_tiles(int64_t tokens, int64_t group, int64_t nkv) {
  return tokens * group > max((int64_t)512, min(4096 / nkv, (int64_t)1536));
}
}  // namespace

extern "C" size_t dip_kv8_prompt_attention_workspace_size(int64_t tokens, int64_t start,
                                                          int64_t n_heads, int64_t n_kv_heads,
                                                          int64_t head_dim) {
  if (head_dim != kKvHeadDim || n_heads <= 0 || n_heads > 4096 || n_kv_heads <= 0 ||
      n_heads % n_kv_heads != 0 || tokens <= 0 || start < 0 || start > (1 << 30) ||
      tokens * n_heads > INT32_MAX)
    return 0;
  const int64_t group = n_heads / n_kv_heads;
  if (by_tiles(tokens, group, n_kv_heads))
    return prompt_tiles_workspace(tokens, start, n_kv_heads, group);
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
  if (by_tiles(tokens, group, n_kv_heads)) {
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
