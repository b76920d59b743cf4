// dip_kv4_prompt.hip — a prompt's attention over the 4-bit key/value cache
// (dip_kv4.h): the rows expanded once to bf16 in the order the matrix
// instructions read them, then attention in tiles of 128 (token, query head)
// columns.
//
// Every tile of columns reads every earlier row, so unpacking in the tiles would
// be done tokens * group / 128 times; once costs two passes over 512 bytes per row
// and kv head, a few per cent of the products' time from some hundred columns on
// (4096 rows of 8 heads 8 us).
#include "dip_kv4.h"

namespace dip {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kTileCols = 128;   // columns of a workgroup, 32 to a wave
constexpr int kPromptWaves = 4;
constexpr int kMinWgs = 2;
constexpr int kStepBlocks = 2;   // blocks of 32 cache rows of a step
constexpr int kTileRows = 32 * kStepBlocks;
constexpr int kBlockVecs = 1024; // 16-byte pieces of an expanded block: 512 of keys, 512 of values

// The largest scale of finite values: bf16's largest over 7, cut to 5 bits.  (Times 7
// it is still a bf16 number.)
constexpr float kMaxScale = 0x1.2p125f;

// The expanded cache: per kv head and block of 32 rows
//   keys   [16][32 rows] pieces: piece (u, row) holds dimensions 8 u .. 8 u + 7;
//   values [2][2][128 dims] pieces: piece (c, h, d) holds dimension d of rows
//          16 c + 4 h + 0 .. 3 and 16 c + 8 + 4 h + 0 .. 3,
// each the order in which the lanes of a 32x32x16 MFMA take their operand.  Blocks
// in pairs; what lies behind the cache's end is 0.  bad[kv head][block]: a byte per
// value group, the first row of the block whose group is not finite (255: none).
// Those values are 0 here, and a number of -8, which nobody writes, is -7: whatever
// the rows that nobody has written hold, a weight of 0 makes 0 of it.
__global__ __launch_bounds__(256) void kv4_expand_kernel(
    const uint32_t* __restrict__ kc, const uint32_t* __restrict__ vc,
    const uint16_t* __restrict__ sc, uint4* __restrict__ work, uint32_t* __restrict__ bad,
    int max_len, int blocks) {
  __shared__ uint32_t scales[kKvBlock][4];  // pairs: keys (g 0, 1), (2, 3), values
  const int b = blockIdx.x % blocks, kvh = blockIdx.x / blocks, tid = threadIdx.x;
  uint4* out = work + (size_t)blockIdx.x * kBlockVecs;
  if (b * kKvBlock >= max_len) {
    for (int i = tid; i < kBlockVecs; i += 256) out[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) bad[blockIdx.x] = 0xFFFFFFFFu;
    return;
  }
  const size_t row0 = (size_t)kvh * max_len + b * kKvBlock;
  if (tid < 128)
    scales[tid >> 2][tid & 3] = reinterpret_cast<const uint32_t*>(sc + row0 * kKvScaleVals)[tid];
  __syncthreads();
  auto scale = [&](int row, int g) {  // g 0 .. 3 keys, 4 .. 7 values
    const uint32_t w = scales[row][g >> 1];
    return __uint_as_float(g & 1 ? w & 0xFFFF0000u : w << 16);
  };
  if (tid < 128) {
    const int row = tid & 31, c = tid >> 5;
    const uint4 w = reinterpret_cast<const uint4*>(kc + (row0 + row) * (kKvKeyBytes / 4))[c];
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float s = scale(row, g);
      uint32_t o[4];
#pragma unroll
      for (int m = 0; m < 4; ++m)
        o[m] = cvt_bf16x2((float)kv4_nibble(x[g], kv4_shift(2 * m)) * s,
                          (float)kv4_nibble(x[g], kv4_shift(2 * m + 1)) * s);
      out[(4 * g + c) * 32 + row] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else if (tid < 132) {
    const int g = tid - 128;
    uint32_t first = 255;
    for (int r = kKvBlock - 1; r >= 0; --r)
      if (!(fabsf(scale(r, 4 + g)) <= kMaxScale)) first = r;
    const uint32_t w = first << (8 * g);
    uint32_t all = w;
    all |= __shfl_xor(all, 1, 64);
    all |= __shfl_xor(all, 2, 64);
    if (g == 0) bad[blockIdx.x] = all;
  }
  {
    const int d = tid & 127, h = tid >> 7, g = 4 + (d >> 5);
    const uint32_t* blk = vc + ((size_t)kvh * (max_len / kKvBlock) + b) * kKvBlockWords;
    const uint32_t lo = blk[kv4_value_word(d, h)], hi = blk[kv4_value_word(d, 2 + h)];
    auto value = [&](uint32_t w, int row, int j) {
      const float s = scale(row, g);
      const float v = (float)max(kv4_nibble(w, kv4_shift(j)), -7) * s;
      return fabsf(s) <= kMaxScale ? v : 0.f;
    };
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t o[4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int r = 16 * c + 4 * h + 2 * m, j = 4 * c + 2 * m;
        o[m] = cvt_bf16x2(value(lo, r, j), value(lo, r + 1, j + 1));
        o[2 + m] = cvt_bf16x2(value(hi, r + 8, j), value(hi, r + 9, j + 1));
      }
      out[512 + (c * 2 + h) * 128 + d] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// The steps of 64 rows that a split takes of a tile's.
DIP_DEV int steps_per_split(int rows, int splits) {
  const int steps = (rows + kTileRows - 1) / kTileRows;
  return (steps + splits - 1) / splits;
}
DIP_DEV int tile_end(const Kv4AttnArgs& a, int tile) {
  const int last = min((tile * kTileCols + kTileCols - 1) / a.group, a.tokens - 1);
  return (int)(a.start + last + 1);
}

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// Attention of a tile's 128 columns, 32 to a wave, over the rows of a split, 64 to
// a step; a step's expanded rows (32 KB) go straight from memory to LDS while the
// step before is worked on.  Per step and wave, with the lane's column l % 32 and
// h = l / 32:
//   scores^T = K Q^T: 32x32x16 MFMAs, the queries' operand held in registers for
//     good; lane (h, column) gets the scores of rows 8 i + 4 h + 0 .. 3;
//   softmax in fp32 against a base that follows the running maximum (lanes l and
//     l ^ 32 share a column);
//   out^T += V^T P^T, the weights rounded to bf16 in place: they are the operand
//     as they lie.  (Off by 2^-8 of itself at most, as any bf16 weight is.)
// 4096 tokens of 64 / 8 heads, 275 GFLOP without the masked half: 294 us a call, the
// expansion's 8 with it, 0.94 PFLOP/s, where a large product of matrices reaches 1.15
// to 1.37 (a trace of 30 calls alone has this launch at 297 to 334).  The MFMAs are busy
// 49 % of the time and the VALU, the softmax mostly, 56 %; without the fetch it took 240
// us, without the exponentials 336, without the second product 290 (of 350).  (8 waves to a workgroup 341 of then 352, but 72 for 43 at 1024 tokens; three
// buffers 353; rows through registers into LDS 493; 32 rows to a step and three
// workgroups to a CU 340 to 346.)
template <bool kSplit>
__global__ __launch_bounds__(kPromptWaves * 64, kMinWgs) void kv4_prompt_kernel(
    Kv4AttnArgs a, const uint4* work, const uint32_t* bad, int blocks, int tiles) {
  __shared__ uint4 buf_a[kStepBlocks * kBlockVecs], buf_b[kStepBlocks * kBlockVecs];
  __shared__ int bad_row[kKvGroups];
  const int kvh = blockIdx.x % a.nkv, rest = blockIdx.x / a.nkv;
  const int split = kSplit ? rest % a.splits : 0;
  const int tile = tiles - 1 - (kSplit ? rest / a.splits : rest);  // the longest first
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = threadIdx.x & 63, l32 = l & 31, h = l >> 5;
  const int rows = tile_end(a, tile);
  const int steps = (rows + kTileRows - 1) / kTileRows;
  const int per = steps_per_split(rows, kSplit ? a.splits : 1);
  const int t0 = split * per, t1 = min(t0 + per, steps);
  if (kSplit && t0 >= t1) return;

  const int col = tile * kTileCols + wave * 32 + l32;
  const int tok = min(col / a.group, a.tokens - 1), head = kvh * a.group + col % a.group;
  const bool on = col < a.tokens * a.group;
  const int limit = (int)a.start + tok + 1;
  const int sure = (int)a.start + min((tile * kTileCols + wave * 32) / a.group, a.tokens - 1) + 1;
  const int most = (int)a.start + min((tile * kTileCols + wave * 32 + 31) / a.group,
                                      a.tokens - 1) + 1;  // of this wave's columns
  bf16x8_t bq[8];
  {
    const uint4* qp = reinterpret_cast<const uint4*>(
        a.q + ((size_t)tok * a.nkv * a.group + head) * kKvHeadDim);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint4 w = qp[2 * k + h];
      const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
      w.x ^= sign, w.y ^= sign, w.z ^= sign, w.w ^= sign;
      bq[k] = __builtin_bit_cast(bf16x8_t, u32x4_t{w.x, w.y, w.z, w.w});
    }
  }
  if (threadIdx.x < kKvGroups) bad_row[threadIdx.x] = INT32_MAX;

  const uint4* src = work + (size_t)kvh * blocks * kBlockVecs;
  auto fetch = [&](uint4* buf, int t) {
#pragma unroll
    for (int i = 0; i < kStepBlocks * kBlockVecs / 256; ++i) {
      const int at = i * 256 + wave * 64;
      __builtin_amdgcn_global_load_lds(
          (global_void*)(src + (size_t)t * kStepBlocks * kBlockVecs + at + l),
          (lds_void*)(buf + at), 16, 0, 0);
    }
  };

  const float c2 = fabsf(a.scale) * kLog2e;  // (its sign is in the queries)
  floatx16 acc[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  float m = -INFINITY, den = 0.f;  // m: the base; den: this lane's rows only

  auto step = [&](const uint4* buf, int t) {
    if (t * kTileRows >= most) return;  // every row lies behind this wave's columns
    auto frag = [&](int i) {
      const uint4 w = buf[i];
      return __builtin_bit_cast(bf16x8_t, u32x4_t{w.x, w.y, w.z, w.w});
    };
    floatx16 s[kStepBlocks];
#pragma unroll
    for (int b = 0; b < kStepBlocks; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            frag(b * kBlockVecs + (2 * k + h) * 32 + l32), bq[k], s[b], 0, 0, 0);
    }
    const bool masked = (t + 1) * kTileRows > sure;
    // this lane's row of value r of block b, from the column's first row that it
    // does not attend
    const int behind = t * kTileRows + 4 * h - limit;
    if (masked) {
      asm volatile("");  // a branch: 64 comparisons and selections that most steps skip
#pragma unroll
      for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (behind + 32 * b + 8 * (r >> 2) + (r & 3) >= 0) s[b][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
    {
#pragma clang fp contract(off)
      mx = fmaxf(m, row_pair_max32(mx) * c2 + kDown);
    }
    // kSlack: with 32 columns to a wave some column has a new maximum in most steps, and
    // the sums' 64 products are a quarter of a step's instructions (4096 tokens of 64 / 8
    // heads 350 us for 343)
    if (__any(mx > m + kSlack)) {
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - mx);
      den *= f;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= f;
      m = mx;
    }
    const float base = m == -INFINITY ? 0.f : m;
    // The base comes from a rounded product: where its rounding is not small all are
    // taken rounded, as the distance from it may be further than weights reach.  (A
    // branch; 4096 tokens of 64 / 8 heads 295.4 us for 294.6, 509 behind 16003 rows 307
    // for 302.4.)
    const bool far = __any(fabsf(base) > 0x1p24f);
    if (__builtin_expect(far, 0)) {
      asm volatile("");
#pragma unroll
      for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] *= c2;
    }
    const float by = far ? 1.f : c2;
#pragma unroll
    for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = fast_exp2(fmaf(s[b][r], by, -base));
    if (masked) {  // weights of 0, whatever a base of +inf or NaN made of them
      asm volatile("");
#pragma unroll
      for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (behind + 32 * b + 8 * (r >> 2) + (r & 3) >= 0) s[b][r] = 0.f;
    }
#pragma unroll
    for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) den += s[b][r];
#pragma unroll
    for (int b = 0; b < kStepBlocks; ++b)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bf16x8_t p = __builtin_bit_cast(
            bf16x8_t, u32x4_t{cvt_bf16x2(s[b][8 * c], s[b][8 * c + 1]),
                              cvt_bf16x2(s[b][8 * c + 2], s[b][8 * c + 3]),
                              cvt_bf16x2(s[b][8 * c + 4], s[b][8 * c + 5]),
                              cvt_bf16x2(s[b][8 * c + 6], s[b][8 * c + 7])});
#pragma unroll
        for (int d = 0; d < 4; ++d)
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              frag(b * kBlockVecs + 512 + (c * 2 + h) * 128 + d * 32 + l32), p, acc[d], 0, 0, 0);
      }
  };
  // this wave's pieces have landed, then everybody's, and the other buffer's
  // readers are through
  auto landed = [&] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  fetch(buf_a, t0);
  for (int t = t0; t < t1; t += 2) {
    landed();
    if (t + 1 < t1) fetch(buf_b, t + 1);
    step(buf_a, t);
    if (t + 1 >= t1) break;
    landed();
    if (t + 2 < t1) fetch(buf_a, t + 2);
    step(buf_b, t + 1);
  }

  // the first row of each group of values that is not finite
  __syncthreads();
  for (int b = kStepBlocks * t0 + (int)threadIdx.x; b < kStepBlocks * t1; b += kPromptWaves * 64) {
    const uint32_t w = bad[(size_t)kvh * blocks + b];
    if (w == 0xFFFFFFFFu) continue;
    for (int g = 0; g < kKvGroups; ++g)
      if (((w >> (8 * g)) & 255u) != 255u)
        atomicMin(&bad_row[g], b * kKvBlock + (int)((w >> (8 * g)) & 255u));
  }
  __syncthreads();
  den = row_pair_sum32(den);
  if (!on) return;
  if (kSplit) {
    float* o = a.part + (((size_t)(tile * a.nkv + kvh) * a.splits + split) * kTileCols +
                         wave * 32 + l32) * kKvPart;
    if (h == 0) {
      o[0] = m;
      o[1] = den;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const bool nan = bad_row[d] < limit;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        o[2 + 32 * d + 8 * (r >> 2) + 4 * h + (r & 3)] = nan ? NAN : acc[d][r];
    }
    return;
  }
  const float inv = 1.f / den;  // (a sum of 0: every score is -inf, which makes NaN)
  uint2* o = reinterpret_cast<uint2*>(a.out + ((size_t)tok * a.nkv * a.group + head) * kKvHeadDim);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const float f = bad_row[d] < limit ? NAN : inv;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[8 * d + 2 * i + h] = make_uint2(cvt_bf16x2(acc[d][4 * i] * f, acc[d][4 * i + 1] * f),
                                        cvt_bf16x2(acc[d][4 * i + 2] * f, acc[d][4 * i + 3] * f));
  }
}

// The splits of a column added up in their order: a wave per (kv head, column).
__global__ __launch_bounds__(256) void kv4_prompt_combine_kernel(Kv4AttnArgs a) {
  const int l = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= (int64_t)a.tokens * a.group * a.nkv) return;
  const int kvh = (int)(at % a.nkv), cc = (int)(at / a.nkv);
  const int tile = cc / kTileCols, rows = tile_end(a, tile);
  const int per = steps_per_split(rows, a.splits);
  const int ns = ((rows + kTileRows - 1) / kTileRows + per - 1) / per;
  const float* base = a.part + ((size_t)(tile * a.nkv + kvh) * a.splits * kTileCols +
                                cc % kTileCols) * kKvPart;
  const size_t stride = (size_t)kTileCols * kKvPart;
  // lane s the weight of split s (64 at most), then 8 splits' sums in flight
  const float2 ml = l < ns ? *reinterpret_cast<const float2*>(base + l * stride)
                           : make_float2(-INFINITY, 0.f);
  const float mx = group_max<64>(ml.x);
  const float f = l >= ns ? 0.f : ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - mx);
  const float sum = group_sum<64>(f * ml.y);
  float o0 = 0.f, o1 = 0.f;
  for (int s0 = 0; s0 < ns; s0 += 8) {
    float2 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = *reinterpret_cast<const float2*>(base + min(s0 + u, ns - 1) * stride + 2 + 2 * l);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s0 + u >= ns) break;
      const float w = __shfl(f, s0 + u, 64);
      o0 = fmaf(w, v[u].x, o0);
      o1 = fmaf(w, v[u].y, o1);
    }
  }
  const float inv = 1.f / sum;
  reinterpret_cast<uint32_t*>(a.out)[((size_t)(cc / a.group) * a.nkv * a.group +
                                      kvh * a.group + cc % a.group) * 64 + l] =
      cvt_bf16x2(o0 * inv, o1 * inv);
}

struct Plan {
  int64_t tiles, blocks;
  int splits;
  size_t work, bad, part;  // bytes
  int64_t us100;           // about what the launches take, in hundredths of a microsecond
};

// The splits of a tile's rows that take least, by estimates from measured times: 10
// us, 0.12 ns per row and kv head to expand, and for a step of 64 rows 2.6 us where
// a CU has one workgroup and 3 us where it has two; splits add 7 us and 0.12 ns for
// each column's sums, which are written and read again.  (512 tokens of 64 / 8
// heads: 2 splits 39 us, 1 split 23; 32 tokens behind 20010 rows: 32 splits 69 us, 16
// splits 87.)
Plan plan_for(int64_t tokens, int64_t start, int64_t nkv, int64_t group) {
  Plan p;
  p.tiles = (tokens * group + kTileCols - 1) / kTileCols;
  p.blocks = (start + tokens + kTileRows - 1) / kTileRows * kStepBlocks;
  const int64_t steps = (start + tokens + kTileRows - 1) / kTileRows, cus = device_cus();
  p.us100 = INT64_MAX;
  for (int64_t s = 1; s <= min((steps + 3) / 4, (int64_t)64); s = s < 8 ? s + 1 : s + s / 8) {
    const int64_t wgs = p.tiles * nkv * s, per = (steps + s - 1) / s;
    const int64_t us = 1000 + (start + tokens) * nkv * 12 / 1000 +
                       per * (wgs <= cus ? 260 : 300 * ((wgs + 2 * cus - 1) / (2 * cus))) +
                       (s == 1 ? 0 : 700 + tokens * group * nkv * s * 12 / 1000);
    if (us < p.us100) {
      p.us100 = us;
      p.splits = (int)s;
    }
  }
  p.work = (size_t)nkv * p.blocks * kBlockVecs * 16;
  p.bad = ((size_t)nkv * p.blocks * 4 + 15) / 16 * 16;
  p.part = p.splits == 1 ? 0
                         : (size_t)p.tiles * nkv * p.splits * kTileCols * kKvPart * sizeof(float);
  return p;
}

}  // namespace

size_t prompt_tiles_workspace(int64_t tokens, int64_t start, int64_t nkv, int64_t group) {
  const Plan p = plan_for(tokens, start, nkv, group);
  return p.work + p.bad + p.part;
}

int64_t prompt_tiles_us100(int64_t tokens, int64_t start, int64_t nkv, int64_t group) {
  return plan_for(tokens, start, nkv, group).us100;
}

int launch_prompt_tiles(Kv4AttnArgs a, void* workspace, hipStream_t stream) {
  const Plan p = plan_for(a.tokens, a.start, a.nkv, a.group);
  const int64_t expand = a.nkv * p.blocks, grid = p.tiles * a.nkv * p.splits;
  const int64_t cols = (int64_t)a.tokens * a.group * a.nkv;
  if (!launch_fits(expand, 256) || !launch_fits(grid, kPromptWaves * 64) || cols > INT32_MAX ||
      !launch_fits((cols + 3) / 4, 256))
    return DIP_ERR_SHAPE;
  char* w = static_cast<char*>(workspace);
  uint4* work = reinterpret_cast<uint4*>(w);
  uint32_t* bad = reinterpret_cast<uint32_t*>(w + p.work);
  a.part = reinterpret_cast<float*>(w + p.work + p.bad);
  a.splits = p.splits;
  hipLaunchKernelGGL(kv4_expand_kernel, dim3((unsigned)expand), dim3(256), 0, stream, a.kc, a.vc,
                     a.sc, work, bad, a.max_len, (int)p.blocks);
  if (p.splits > 1) {
    hipLaunchKernelGGL((kv4_prompt_kernel<true>), dim3((unsigned)grid), dim3(kPromptWaves * 64), 0,
                       stream, a, work, bad, (int)p.blocks, (int)p.tiles);
    hipLaunchKernelGGL(kv4_prompt_combine_kernel, dim3((unsigned)((cols + 3) / 4)), dim3(256), 0,
                       stream, a);
  } else {
    hipLaunchKernelGGL((kv4_prompt_kernel<false>), dim3((unsigned)grid), dim3(kPromptWaves * 64),
                       0, stream, a, work, bad, (int)p.blocks, (int)p.tiles);
  }
  return hip_status(hipGetLastError());
}

}  // namespace dip
