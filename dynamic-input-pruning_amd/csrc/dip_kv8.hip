// dip_kv8.hip — writing and reading the paged 8-bit key/value cache (dip_kv8.h has
// its layout): q/k RMSNorm + rotary embedding + rounding of the tokens' q | k | v of
// several sequences into their pages, the rounding alone of given keys and values,
// and the cache's rows as the bf16 numbers they stand for.
#include "dip_kv8.h"

namespace dip {
namespace {

constexpr int kWriteWaves = 4;

struct Kv8WriteArgs {
  const uint16_t* k;  // token t of sequence s at s * k_seq + t * k_tok (kNorm: q | k | v)
  const uint16_t* v;
  int64_t k_seq, k_tok, k_head, v_seq, v_tok, v_head;
  const uint16_t* q_w;  // kNorm only, to eps
  const uint16_t* k_w;
  const uint16_t* cos_t;
  const uint16_t* sin_t;
  uint16_t* q_out;
  float eps;
  const int64_t* pos;
  const int32_t* table;
  Kv8Pages c;
  int seqs, tokens, nh, width;
  int tiles;     // pages that a sequence's tokens may touch
  int64_t rows;  // positions that tables of both kinds have
  int k_vec, v_vec;  // every head of k, of v starts at a multiple of 16 bytes
};

DIP_DEV void load_head(uint32_t (&x)[4], const uint16_t* p, bool vec) {
  if (vec) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = reinterpret_cast<const uint32_t*>(p)[e];
  }
}

// The largest magnitude of a lane's 8 values (fp32 bits, which order like them), 0 if
// its group of 32 dimensions (four lanes) has a value that is not finite; `bad` then.
DIP_DEV uint32_t finite_most(const uint32_t (&x)[4], bool& bad) {
  uint32_t m = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) m = max(m, max((x[e] << 16) & 0x7FFFFFFFu, x[e] & 0x7FFF0000u));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
  bad = m >= 0x7F800000u;
  return bad ? 0u : m;
}

// The scale (fp32 bits) of values up to a.
DIP_DEV uint32_t scale_bits(uint32_t a) {
  const uint32_t e = a >> 23;
  return a == 0u ? 0u : (max(e, 27u + 7u) - 7u) << 23;
}

// A lane's 8 values as numbers of scale s.
DIP_DEV void numbers_of(const uint32_t (&x)[4], uint32_t s, bool bad, uint32_t& w0, uint32_t& w1) {
  const float inv = s == 0u ? 1.f : __uint_as_float((254u << 23) - s);
  const float cap = s == 247u << 23 ? 240.f : 256.f;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float lo = fminf(fmaxf(__uint_as_float(x[e] << 16) * inv, -cap), cap);
    const float hi = fminf(fmaxf(__uint_as_float(x[e] & 0xFFFF0000u) * inv, -cap), cap);
    w[e >> 1] = e & 1 ? __builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, (int)w[e >> 1], true)
                      : __builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, (int)w[e >> 1], false);
  }
  w0 = bad ? kNanByte4 : w[0];
  w1 = bad ? kNanByte4 : w[1];
}

// Four numbers taken from one scale to another, `by` the first over the second.
DIP_DEV uint32_t rounded_again(uint32_t w, float by) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(lo.x * by, lo.y * by, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi.x * by, hi.y * by, r, true);
}

// The bytes of word t of a quarter's pieces whose rows 16 t + 4 c .. + 3 lie in [lo, hi).
DIP_DEV uint32_t row_bytes(int t, int c, int lo, int hi) {
  uint32_t m = 0u;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int r = 16 * t + 4 * c + g;
    if (r >= lo && r < hi) m |= 0xFFu << (8 * g);
  }
  return m;
}

// First a workgroup for each (sequence, page that its tokens may touch, kv head): wave
// c has the rows 16 t + 4 c + g, t = 0 .. 3, of the page, 16 lanes (g) to a row with 8
// dimensions each, so the four waves' rows are different pieces of the values' layout
// and nothing is exchanged between them but the largest magnitudes.  All of a page's
// rows are in registers before any is written, as they share a scale.  Then, with the
// norm, the q heads, a wave per four heads of a token.
// A prompt of 4099 tokens of 64 / 8 heads: 42 us, 187 MB at 3.7 to 3.9 TB/s, VALU 76 % busy
// with the norm, in 64 bits; 40000 tokens' keys and values without it at 5.8 TB/s.  One
// token: 5.5 us of waits in a row, 5.0 for 4.1 where the page's 63 earlier rows are rounded
// again to a larger scale.
template <bool kNorm>
__global__ __launch_bounds__(64 * kWriteWaves) void kv8_write_kernel(Kv8WriteArgs a) {
  __shared__ uint32_t most[2][kWriteWaves];
  const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
  const int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t kv_wgs = (int64_t)a.seqs * a.tiles * a.c.nkv;
  if (blockIdx.x >= kv_wgs) {
    const int quads = (a.nh + 3) / 4;
    const int64_t task = (blockIdx.x - kv_wgs) * kWriteWaves + c, tok = task / quads;
    const int head = (int)(task % quads) * 4 + g;
    if (tok >= (int64_t)a.seqs * a.tokens) return;
    const int64_t s = tok / a.tokens, t = tok % a.tokens, first = a.pos[s];
    if (first < 0 || first >= a.rows - t) return;
    // (read beside the token's values, for the write behind them)
    const int id = page_number(a.table + s * a.width, (first + t) / kPageRows, a.c.pages);
    uint32_t x[4] = {0u, 0u, 0u, 0u};
    if (head < a.nh) load_head(x, a.k + s * a.k_seq + t * a.k_tok + head * kKvHeadDim + 8 * i, true);
    head_norm_rope(x, a.q_w, a.cos_t, a.sin_t, first + t, i, a.eps);
    if (head < a.nh && id >= 0)
      reinterpret_cast<uint4*>(a.q_out)[(tok * a.nh + head) * 16 + i] =
          make_uint4(x[0], x[1], x[2], x[3]);
    return;
  }
  const int head = (int)(blockIdx.x % a.c.nkv);
  const int64_t s = blockIdx.x / a.c.nkv / a.tiles;
  const int64_t first = a.pos[s];
  if (first < 0 || first >= a.rows) return;
  const int64_t page = first / kPageRows + blockIdx.x / a.c.nkv % a.tiles;
  // the page's rows that are written
  const int lo = (int)max(first - page * kPageRows, (int64_t)0);
  const int hi = (int)min(min(first + a.tokens, a.rows) - page * kPageRows, (int64_t)kPageRows);
  if (hi <= lo) return;
  const int id = page_number(a.table + s * a.width, page, a.c.pages);
  if (id < 0) return;
  const size_t at = (size_t)id * a.c.nkv + head;
  uint8_t* kp = a.c.k + at * kPageBytes;
  uint8_t* vp = a.c.v + at * kPageBytes;
  const uint2 was = lo > 0 ? *reinterpret_cast<const uint2*>(a.c.scales + 2 * at)
                           : make_uint2(0u, 0u);

  uint32_t k[4][4], v[4][4];
  bool k_bad[4], v_bad[4];
  uint32_t k_most = 0u, v_most = 0u;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) k[t][e] = v[t][e] = 0u;
    k_bad[t] = v_bad[t] = false;
    if (16 * t + 4 * c >= hi || 16 * t + 4 * c + 3 < lo) continue;
    const int r = 16 * t + 4 * c + g;
    const bool in = r >= lo && r < hi;
    const int64_t tok = in ? page * kPageRows + r - first : 0;
    if (in) {
      load_head(k[t], a.k + s * a.k_seq + tok * a.k_tok +
                          (kNorm ? a.nh + head : head) * a.k_head + 8 * i, kNorm || a.k_vec);
      load_head(v[t], a.v + s * a.v_seq + tok * a.v_tok + head * a.v_head + 8 * i,
                kNorm || a.v_vec);
    }
    if (kNorm) head_norm_rope(k[t], a.k_w, a.cos_t, a.sin_t, first + tok, i, a.eps);
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = 16 * t + 4 * c + g;
    const bool in = r >= lo && r < hi;
    const uint32_t mk = finite_most(k[t], k_bad[t]), mv = finite_most(v[t], v_bad[t]);
    k_most = max(k_most, in ? mk : 0u);
    v_most = max(v_most, in ? mv : 0u);
  }
#pragma unroll
  for (int m = 4; m < 64; m <<= 1) {
    k_most = max(k_most, (uint32_t)__shfl_xor(k_most, m, 64));
    v_most = max(v_most, (uint32_t)__shfl_xor(v_most, m, 64));
  }
  if (l == 0) {
    most[0][c] = k_most;
    most[1][c] = v_most;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWriteWaves; ++w) {
    k_most = max(k_most, most[0][w]);
    v_most = max(v_most, most[1][w]);
  }
  const uint32_t ks = max(was.x, scale_bits(k_most)), vs = max(was.y, scale_bits(v_most));
  if (threadIdx.x == 0) *reinterpret_cast<uint2*>(a.c.scales + 2 * at) = make_uint2(ks, vs);
  const bool k_up = ks > was.x && lo > 0, v_up = vs > was.y && lo > 0;
  // 1 / the new scale times the old, 0 where no number is left of the earlier ones
  const float k_by = __uint_as_float(was.x) * __uint_as_float((254u << 23) - ks);
  const float v_by = __uint_as_float(was.y) * __uint_as_float((254u << 23) - vs);

  uint32_t col[2][4], mask[4], any = 0u, all = ~0u;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = 16 * t + 4 * c + g;
    uint32_t w0, w1;
    numbers_of(k[t], ks, k_bad[t], w0, w1);
    uint2* kr = reinterpret_cast<uint2*>(kp + r * kKvHeadDim + 8 * i);
    if (r >= lo && r < hi) {
      *kr = make_uint2(w0, w1);
    } else if (k_up && r < lo) {
      const uint2 old = *kr;
      *kr = make_uint2(rounded_again(old.x, k_by), rounded_again(old.y, k_by));
    }
    numbers_of(v[t], vs, v_bad[t], col[0][t], col[1][t]);
    kv8_rows_to_columns(col[0][t], col[1][t]);
    mask[t] = row_bytes(t, c, lo, hi);
    any |= mask[t];
    all &= mask[t];
  }
  if (any == 0u && !v_up) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint4* piece = reinterpret_cast<uint4*>(vp + (8 * i + 2 * g + e) * kPageRows + 16 * c);
    if (all != ~0u) {
      const uint4 old = *piece;
      uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (v_up) o[t] = rounded_again(o[t], v_by);
        col[e][t] = (col[e][t] & mask[t]) | (o[t] & ~mask[t]);
      }
    }
    *piece = make_uint4(col[e][0], col[e][1], col[e][2], col[e][3]);
  }
}

// Rows pos .. of each sequence as bf16 [seqs, tokens, nkv, 128], 0 where it has no
// page: lanes, waves and workgroups as in the write.
__global__ __launch_bounds__(64 * kWriteWaves) void kv8_read_kernel(Kv8Pages a, const int32_t* table,
                                                                    const int64_t* pos,
                                                                    uint4* k_out, uint4* v_out,
                                                                    int tokens, int width,
                                                                    int tiles) {
  const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
  const int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = (int)(blockIdx.x % a.nkv);
  const int64_t s = blockIdx.x / a.nkv / tiles, rows = (int64_t)width * kPageRows;
  const int64_t at_pos = pos[s];
  const bool there = at_pos >= 0 && at_pos < rows;
  const int64_t first = there ? at_pos : 0;
  const int64_t page = first / kPageRows + blockIdx.x / a.nkv % tiles;
  const int id = there && page < width ? page_number(table + s * width, page, a.pages) : -1;
  const size_t at = (size_t)max(id, 0) * a.nkv + head;
  const float2 sc = *reinterpret_cast<const float2*>(a.scales + 2 * at);
  uint4 w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e)
    w[e] = *reinterpret_cast<const uint4*>(a.v + at * kPageBytes + (8 * i + 2 * g + e) * kPageRows +
                                           16 * c);
  const uint32_t w0[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, w1[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = 16 * t + 4 * c + g;
    const int64_t tok = page * kPageRows + r - first;
    const uint2 kw = *reinterpret_cast<const uint2*>(a.k + at * kPageBytes + r * kKvHeadDim + 8 * i);
    uint32_t x = w0[t], y = w1[t];
    kv8_columns_to_rows(x, y);
    u32x4_t ko = __builtin_bit_cast(u32x4_t, kv8_operand(kw.x, kw.y, sc.x));
    u32x4_t vo = __builtin_bit_cast(u32x4_t, kv8_operand(x, y, sc.y));
    if (id < 0) ko = vo = u32x4_t{0u, 0u, 0u, 0u};
    if (tok < 0 || tok >= tokens) continue;
    const size_t o = ((s * tokens + tok) * a.nkv + head) * 16 + i;
    k_out[o] = make_uint4(ko.x, ko.y, ko.z, ko.w);
    v_out[o] = make_uint4(vo.x, vo.y, vo.z, vo.w);
  }
}

// Pages that `tokens` rows at an unknown position may touch.
inline int64_t page_tiles(int64_t tokens) { return (tokens + kPageRows - 2) / kPageRows + 1; }

template <bool kNorm>
int launch_write(Kv8WriteArgs a, hipStream_t stream) {
  const int64_t tiles = min(page_tiles(a.tokens), (int64_t)a.width);
  a.tiles = (int)tiles;
  const int64_t q_tasks = kNorm ? (int64_t)a.seqs * a.tokens * ((a.nh + 3) / 4) : 0;
  const int64_t grid = a.seqs * tiles * a.c.nkv + (q_tasks + kWriteWaves - 1) / kWriteWaves;
  if (!launch_fits(grid, 64 * kWriteWaves)) return DIP_ERR_SHAPE;
  hipLaunchKernelGGL((kv8_write_kernel<kNorm>), dim3((unsigned)grid), dim3(64 * kWriteWaves), 0,
                     stream, a);
  return hip_status(hipGetLastError());
}

inline bool positions_ok(const int64_t* pos) {
  return pos && (reinterpret_cast<uintptr_t>(pos) & 7) == 0;
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" int dip_kv8_write(const uint16_t* k, const uint16_t* v, int64_t k_seq_stride,
                             int64_t k_tok_stride, int64_t k_head_stride, int64_t v_seq_stride,
                             int64_t v_tok_stride, int64_t v_head_stride, uint8_t* k_cache,
                             uint8_t* v_cache, float* kv_scales, int64_t pages,
                             const int32_t* table, int64_t table_width, const int64_t* pos,
                             int64_t seqs, int64_t tokens, int64_t n_kv_heads, int64_t head_dim,
                             void* stream) {
  if (head_dim != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (int st = check_pages(k_cache, v_cache, kv_scales, pages, n_kv_heads, table, seqs,
                           table_width))
    return st;
  if (tokens < 0 || tokens > (1 << 30) || seqs * tokens > INT32_MAX) return DIP_ERR_SHAPE;
  if (tokens == 0 || seqs == 0) return DIP_OK;
  if (!k || !v || !pos) return DIP_ERR_NULL;
  const int64_t ks = k_seq_stride | k_tok_stride | k_head_stride;
  const int64_t vs = v_seq_stride | v_tok_stride | v_head_stride;
  if (ks < 0 || vs < 0) return DIP_ERR_SHAPE;
  // pairs of values are loaded together
  if ((ks | vs) & 1 || (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 3 ||
      !positions_ok(pos))
    return DIP_ERR_ALIGN;
  Kv8WriteArgs a{};
  a.k = k;
  a.v = v;
  a.k_seq = k_seq_stride, a.k_tok = k_tok_stride, a.k_head = k_head_stride;
  a.v_seq = v_seq_stride, a.v_tok = v_tok_stride, a.v_head = v_head_stride;
  a.k_vec = aligned16(k) && ks % 8 == 0;
  a.v_vec = aligned16(v) && vs % 8 == 0;
  a.pos = pos;
  a.table = table;
  a.c = Kv8Pages{k_cache, v_cache, kv_scales, (int)pages, (int)n_kv_heads};
  a.seqs = (int)seqs;
  a.tokens = (int)tokens;
  a.width = (int)table_width;
  a.rows = table_width * kPageRows;
  return launch_write<false>(a, (hipStream_t)stream);
}

extern "C" int dip_kv8_read(const uint8_t* k_cache, const uint8_t* v_cache,
                            const float* kv_scales, int64_t pages, const int32_t* table,
                            int64_t table_width, const int64_t* pos, uint16_t* k_out,
                            uint16_t* v_out, int64_t seqs, int64_t tokens, int64_t n_kv_heads,
                            int64_t head_dim, void* stream) {
  if (head_dim != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (int st = check_pages(k_cache, v_cache, kv_scales, pages, n_kv_heads, table, seqs,
                           table_width))
    return st;
  if (tokens < 0 || tokens > (1 << 30) || seqs * tokens > INT32_MAX) return DIP_ERR_SHAPE;
  if (tokens == 0 || seqs == 0) return DIP_OK;
  if (!k_out || !v_out || !pos) return DIP_ERR_NULL;
  if (!aligned16(k_out) || !aligned16(v_out) || !positions_ok(pos)) return DIP_ERR_ALIGN;
  const int64_t tiles = page_tiles(tokens), grid = seqs * tiles * n_kv_heads;
  if (!launch_fits(grid, 64 * kWriteWaves)) return DIP_ERR_SHAPE;
  const Kv8Pages c{const_cast<uint8_t*>(k_cache), const_cast<uint8_t*>(v_cache),
                   const_cast<float*>(kv_scales), (int)pages, (int)n_kv_heads};
  hipLaunchKernelGGL(kv8_read_kernel, dim3((unsigned)grid), dim3(64 * kWriteWaves), 0,
                     (hipStream_t)stream, c, table, pos, reinterpret_cast<uint4*>(k_out),
                     reinterpret_cast<uint4*>(v_out), (int)tokens, (int)table_width, (int)tiles);
  return hip_status(hipGetLastError());
}

extern "C" int dip_qk_norm_rope_kv8(const uint16_t* qkv, const uint16_t* q_norm_w,
                                    const uint16_t* k_norm_w, const uint16_t* cos_table,
                                    const uint16_t* sin_table, int64_t table_rows,
                                    const int64_t* pos, uint16_t* q_out, uint8_t* k_cache,
                                    uint8_t* v_cache, float* kv_scales, int64_t pages,
                                    const int32_t* table, int64_t table_width, int64_t seqs,
                                    int64_t tokens, int64_t n_heads, int64_t n_kv_heads,
                                    int64_t head_dim, float eps, void* stream) {
  if (head_dim != kKvHeadDim) return DIP_ERR_UNSUPPORTED;
  if (int st = check_pages(k_cache, v_cache, kv_scales, pages, n_kv_heads, table, seqs,
                           table_width))
    return st;
  if (n_heads <= 0 || n_heads > 4096 || tokens < 0 || tokens > (1 << 30) ||
      seqs * tokens > INT32_MAX || table_rows <= 0)
    return DIP_ERR_SHAPE;
  if (!(eps >= 0.f)) return DIP_ERR_ARG;
  if (tokens == 0 || seqs == 0) return DIP_OK;
  if (!qkv || !q_norm_w || !k_norm_w || !cos_table || !sin_table || !pos || !q_out)
    return DIP_ERR_NULL;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(cos_table) || !aligned16(sin_table) ||
      !aligned16(q_norm_w) || !aligned16(k_norm_w) || !positions_ok(pos))
    return DIP_ERR_ALIGN;
  Kv8WriteArgs a{};
  a.k = qkv;
  a.v = qkv + (n_heads + n_kv_heads) * kKvHeadDim;
  a.k_tok = a.v_tok = (n_heads + 2 * n_kv_heads) * kKvHeadDim;
  a.k_seq = a.v_seq = tokens * a.k_tok;
  a.k_head = a.v_head = kKvHeadDim;
  a.q_w = q_norm_w;
  a.k_w = k_norm_w;
  a.cos_t = cos_table;
  a.sin_t = sin_table;
  a.q_out = q_out;
  a.eps = eps;
  a.pos = pos;
  a.table = table;
  a.c = Kv8Pages{k_cache, v_cache, kv_scales, (int)pages, (int)n_kv_heads};
  a.seqs = (int)seqs;
  a.tokens = (int)tokens;
  a.nh = (int)n_heads;
  a.width = (int)table_width;
  a.rows = min(table_width * kPageRows, table_rows);
  return launch_write<true>(a, (hipStream_t)stream);
}
