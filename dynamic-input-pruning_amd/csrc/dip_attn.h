// dip_attn.h — what the attention kernels over the quantised caches share.
#pragma once

#include "dip_common.h"
#include "dip_head_rope.h"
#include "dip_internal.h"

namespace dip {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kKvPart = 2 + kKvHeadDim;  // max, sum, value sum of one column
constexpr float kLog2e = 1.44269504088896340736f;

// The attention kernels' weights are 2^(score - base), against a base that follows the
// running maximum: it is raised to kDown above a new one that passes the old by more
// than kSlack (powers of 2; score in them too), so that the sums are seldom taken
// against a new base.  Weights then lie below 2^(kSlack - kDown), and the sums of 2^18
// of them times the largest values within fp32, where with weights of about 1 two
// rows of large values were beyond it.  kDown cancels in the division.  (At the small
// end a weight of 2^-n of the largest rounds coarser in value groups of a scale below
// 2^(n - 100), the least that scales are.)
constexpr float kSlack = 8.f, kDown = 26.f;

// 2^x; results below the normal range are 0.
DIP_DEV float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Cache rows that the token at position pos attends: 0 .. pos.
DIP_DEV int rows_at(int64_t pos, int max_len) {
  return pos < 0 ? 0 : (pos < (int64_t)max_len ? (int)pos + 1 : max_len);
}

// Attention of a prompt's tokens, in tiles of 128 (token, query head) columns over a
// cache's rows expanded to bf16 (dip_kv4_prompt.hip), of which each cache brings its
// own expansion.
//
// Every tile of columns reads every earlier row, so unpacking in the tiles would
// be done tokens * group / 128 times; once costs two passes over 512 bytes per row
// and kv head, a few per cent of the products' time from some hundred columns on.
//
// Expanded, per kv head and block of 32 rows
//   keys   [16][32 rows] pieces: piece (u, row) holds dimensions 8 u .. 8 u + 7;
//   values [2][2][128 dims] pieces: piece (c, h, d) holds dimension d of rows
//          16 c + 4 h + 0 .. 3 and 16 c + 8 + 4 h + 0 .. 3,
// each the order in which the lanes of a 32x32x16 MFMA take their operand.  Blocks
// in pairs; what lies behind the cache's end is 0.  bad[kv head][block]: a byte per
// group of 32 dimensions, the first row of the block whose values of the group are not
// finite (255: none).  Those values are 0 in the expansion, so that a weight of 0 makes
// 0 of every row.
constexpr int kExpandRows = 32;
constexpr int kBlockVecs = 1024;  // 16-byte pieces of an expanded block: 512 of keys, 512 of values

struct PromptArgs {
  const uint16_t* q;  // [tokens, nkv * group, 128]
  uint16_t* out;      // [tokens, nkv * group, 128]
  int64_t start;      // the first token's position
  int tokens, nkv, group;
  float scale;
  // set by the launch
  const uint4* work;    // the expanded rows, [nkv][blocks][kBlockVecs]
  const uint32_t* bad;  // [nkv][blocks]
  float* part;          // [tiles, nkv, splits, columns of a tile, kKvPart]
  int blocks, tiles, splits;
};

size_t prompt_tiles_workspace(int64_t tokens, int64_t start, int64_t nkv, int64_t group);
// About what the launches take, in hundredths of a microsecond.
int64_t prompt_tiles_us100(int64_t tokens, int64_t start, int64_t nkv, int64_t group);
// Lays the workspace out (work, bad, blocks and the rest of `a`); DIP_ERR_SHAPE for
// what cannot be launched.  Then the expansion fills work and bad.
int prompt_tiles_plan(PromptArgs& a, void* workspace);
int launch_prompt_tiles(const PromptArgs& a, hipStream_t stream);

// One column's splits added up, in a fixed order, by a workgroup of kCombine groups
// of 128 threads: split j has its maximum, its sum and its 128 value sums at base + j *
// stride.  Each group takes every kCombine-th split's value sums; its first loads are
// in flight while the splits' weights are worked out.  (20011 rows of the 4-bit cache,
// 64 columns: 4 us; one group of 128 threads over all splits in turn 18 to 22.)
constexpr int kMaxSplits = 256;
constexpr int kCombine = 8, kAhead = 8;

DIP_DEV void combine_splits(const float* base, size_t stride, int ns, uint16_t* out) {
  __shared__ float wgt[kMaxSplits];
  __shared__ float red[kCombine * kKvHeadDim / 64][2];
  __shared__ float so[kCombine][kKvHeadDim];
  const int tid = threadIdx.x, d = tid % kKvHeadDim, p = tid / kKvHeadDim;
  if (ns == 0) {  // no rows
    if (tid < kKvHeadDim) out[tid] = 0;
    return;
  }
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
    out[tid] = (uint16_t)f32_to_bf16(r / sum);
  }
}

// The same of up to 64 splits by kWaves waves (a workgroup's), each of which takes every
// kWaves-th split, lane l dimensions 2 l and 2 l + 1.  `red`: LDS for the waves' sums.
template <int kWaves>
DIP_DEV void combine_splits_waves(const float* base, size_t stride, int ns, int wave, int l,
                                  float2 (*red)[64], uint16_t* out) {
  // lane s the weight of split s, then 16 splits' sums in flight
  const float2 ml = l < ns ? *reinterpret_cast<const float2*>(base + l * stride)
                           : make_float2(-INFINITY, 0.f);
  const float mx = group_max<64>(ml.x);
  // (a split without a score above -inf has sums of 0, or NaN, which must count)
  const float f = l >= ns ? 0.f : ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - mx);
  const float sum = group_sum<64>(f * ml.y);
  float o0 = 0.f, o1 = 0.f;
  for (int s0 = wave; s0 < ns; s0 += 16 * kWaves) {
    float2 v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u)
      v[u] = *reinterpret_cast<const float2*>(base + min(s0 + kWaves * u, ns - 1) * stride + 2 +
                                              2 * l);
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      if (s0 + kWaves * u >= ns) break;
      const float w = __shfl(f, s0 + kWaves * u, 64);
      o0 = fmaf(w, v[u].x, o0);
      o1 = fmaf(w, v[u].y, o1);
    }
  }
  if (kWaves > 1) {
    red[wave][l] = make_float2(o0, o1);
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      o0 += red[w][l].x;
      o1 += red[w][l].y;
    }
  }
  const float inv = ns == 0 ? 0.f : 1.f / sum;  // (no rows: zeros)
  reinterpret_cast<uint32_t*>(out)[l] = cvt_bf16x2(o0 * inv, o1 * inv);
}

}  // namespace dip
