// dip_sample.h — what drawing a token from logits (dip_sample.hip, which says how) and
// verifying drafted ones (dip_verify.hip) share: the weights of a row's tokens and the
// border of those that the filters keep.
#pragma once

#include "dip_common.h"
#include "dip_internal.h"

#include <hip/hip_fp16.h>
#include <math.h>

namespace dip {

struct SampleArgs {
  const void* logits;
  int64_t vocab, row_bytes;
  const void* more;  // rows rows1 .. of a launch are rows 0 .. of this tensor
  int64_t more_bytes;
  int rows1;
  const float* u;
  double top_p, per_64th, least, least_64ths;  // see Weigher; min-p in 64ths of an octave
  int64_t top_k;
  float per_hi, per_lo;
  int shift;
  int slices;
  int64_t slice_vecs;  // 16-byte pieces of a row that a slice takes
  char* rows;  // row_state(a, r) of each
  int64_t row_ws;
  int64_t* token;
  float* prob;
};

// In dip_sample.hip: the launches that leave every row's plan, list and slices' sums in
// its RowState, and the one that leaves the slices' largest logits there.
void launch_slices(int dtype, const SampleArgs& a, int rows, hipStream_t s);
void launch_slices_max(int dtype, const SampleArgs& a, int rows, hipStream_t s);

namespace {

constexpr int kThreads = 256;  // of a slice's workgroup, and what kN stands at below
// (64 rows of 151936 fp32 logits: 256 threads 13.8 us, 512 10.0, 1024 11.0.)
constexpr int kDrawThreads = 512;
constexpr int kBins = 1024;
constexpr int kListMax = 4096;
constexpr int kRankMax = 512;  // longer lists are sorted, not ranked by comparing all pairs
constexpr int kMaxSlices = 256;
constexpr int kRadixBins = 256;
constexpr uint32_t kKeyMinusInf = 0x007FFFFFu;  // order_key of -inf

// fp32 (no NaN) as a whole number that orders like it, -0 as 0.
DIP_DEV uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
DIP_DEV float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// NaN as -inf.
DIP_DEV float no_nan(float x) { return fmaxf(x, -INFINITY); }

template <int kType>
DIP_DEV float load_logit(const void* row, int64_t i) {
  if (kType == DIP_F32) return no_nan(static_cast<const float*>(row)[i]);
  if (kType == DIP_F16) return no_nan(__half2float(static_cast<const __half*>(row)[i]));
  return no_nan(bf16_to_f32(static_cast<const uint16_t*>(row)[i]));
}

// Where the histogram says that the borders lie, and the row's ends.
struct Plan {
  uint32_t top, least;        // order_keys of the largest logit and the smallest above -inf
  int lo, hi;                 // the bins to list; lo = kBins: none
  int by_k, ranked;           // top-k cuts tokens; its or top-p's border is in the list
  uint64_t above_n, above_w;  // tokens and weights of the bins before lo
  uint64_t total;             // weights of all bins
};

// A row's workspace, followed by the slices' histograms (kBins weights each).
struct RowState {
  Plan plan;
  uint64_t best[kMaxSlices];            // per slice: order_key << 32 | ~index of its largest
  uint32_t least[kMaxSlices];           // smallest order_key above -inf
  unsigned long long sure[kMaxSlices];  // weights before the bins of the list
  unsigned long long hw[kBins];         // histogram: weights, tokens
  uint32_t hn[kBins];
  uint32_t listed, pad[3];
  uint64_t list[kListMax];              // order_key << 32 | ~index
};
static_assert(sizeof(RowState) % 16 == 0, "rows of the workspace stay aligned");

DIP_DEV RowState& row_state(const SampleArgs& a, int r) {
  return *reinterpret_cast<RowState*>(a.rows + r * a.row_ws);
}
DIP_DEV unsigned long long* slice_hist(const SampleArgs& a, int r, int s) {
  return reinterpret_cast<unsigned long long*>(a.rows + r * a.row_ws + sizeof(RowState)) +
         (size_t)s * kBins;
}
DIP_DEV const char* row_of(const SampleArgs& a, int r) {
  return r < a.rows1 ? static_cast<const char*>(a.logits) + (int64_t)r * a.row_bytes
                     : static_cast<const char*>(a.more) + (int64_t)(r - a.rows1) * a.more_bytes;
}

// The 16-byte piece v of a row.  Pieces lie where memory has them; one that reaches
// over an end of the row is not loaded here, but token by token by its visitor.
template <int kType>
struct Piece {
  static constexpr int kSize = kType == DIP_F32 ? 4 : 2, kVec = 16 / kSize;
  int64_t first;  // its first token
  bool inside;
  uint4 w;

  DIP_DEV Piece() {}
  DIP_DEV Piece(const char* row, int64_t vocab, int64_t v) {
    first = v * kVec - (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize;
    inside = first >= 0 && first + kVec <= vocab;
    w = make_uint4(0, 0, 0, 0);
    if (inside) w = *reinterpret_cast<const uint4*>(row + first * kSize);
  }
  // f(index, logit) of its tokens, NaN as -inf.
  template <typename F>
  DIP_DEV void tokens(const char* row, int64_t vocab, F f) const {
    if (inside) {
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t b = kSize == 4 ? x[i] : (x[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
        const float l = kType == DIP_F32   ? __uint_as_float(b)
                        : kType == DIP_F16 ? __half2float(__ushort_as_half((unsigned short)b))
                                           : bf16_to_f32(b);
        f(first + i, no_nan(l));
      }
    } else {
      for (int i = 0; i < kVec; ++i)
        if (first + i >= 0 && first + i < vocab)
          f(first + i, load_logit<kType>(row, first + i));
    }
  }
  // f(index, logit of p's row, logit of q's row) of two rows' pieces at the same place.
  template <typename F>
  DIP_DEV static void pairs(const Piece& p, const Piece& q, const char* row, const char* other,
                            int64_t vocab, F f) {
    if (p.inside) {
      float y[kVec];
      q.tokens(other, vocab, [&](int64_t i, float v) { y[i - q.first] = v; });
      p.tokens(row, vocab, [&](int64_t i, float x) { f(i, x, y[i - p.first]); });
    } else {
      p.tokens(row, vocab, [&](int64_t i, float x) { f(i, x, load_logit<kType>(other, i)); });
    }
  }
};

// f(index, logit) of the tokens in the pieces [v0, v1) by the workgroup's threads,
// `head` being this thread's first one (loaded before what the caller waits for).
// (2, 4 or 8 pieces of a thread loaded together: 64 rows of 151936 fp32 logits 31, 33
// and 38 us unfiltered for 31, one bf16 row 12, 12 and 13 for 11.5.)
template <int kType, int kN = kThreads, typename F>
DIP_DEV void each_token(Piece<kType> head, const char* row, int64_t vocab, int64_t v0, int64_t v1,
                        F f) {
  for (int64_t v = v0 + threadIdx.x; v < v1;) {
    head.tokens(row, vocab, f);
    v += kN;
    if (v < v1) head = Piece<kType>(row, vocab, v);
  }
}
template <int kType, int kN = kThreads, typename F>
DIP_DEV void each_token(const char* row, int64_t vocab, int64_t v0, int64_t v1, F f) {
  each_token<kType, kN>(Piece<kType>(row, vocab, v0 + threadIdx.x), row, vocab, v0, v1, f);
}

template <int kType>
DIP_DEV int64_t row_vecs(const char* row, int64_t vocab) {
  constexpr int kSize = kType == DIP_F32 ? 4 : 2;
  return ((reinterpret_cast<uintptr_t>(row) & 15) + vocab * kSize + 15) / 16;
}

// 2^-(j / 64), j = 0 .. 63, from the series of exp.
struct Roots {
  double v[64];
  constexpr Roots() : v() {
    for (int j = 0; j < 64; ++j) {
      const double x = -0.69314718055994530942 * j / 64;
      double term = 1.0, sum = 1.0;
      for (int i = 1; i < 24; ++i) {
        term *= x / i;
        sum += term;
      }
      v[j] = sum;
    }
  }
};
__device__ const Roots kRoots = Roots();

// What a row's largest logit makes of the others.  A weight is 2^-(n / 64) exp(z)
// with n - 64 z / ln 2 = 64 (max - logit) / (temperature ln 2), |z| < 0.0055: a table
// of 64 roots in 64 bits, and z and exp(z) - 1 = z + z^2 / 2 + z^3 / 6 in 32, with the
// roundings of the difference and of its product carried along.  That is off by
// 4e-10 of the weight, at random; a running sum over n tokens by 4e-10 / sqrt(n) of
// itself.  (All in 64 bits, whose conversions run at a quarter of the rate: 250
// rows of 32003 15.7 us in the launch that adds the weights up.)
struct Weigher {
  float most, per_hi, per_lo;  // 64ths of an octave per logit, in two parts
  bool inf;                    // the largest is +inf, and only its equals count
  double least;                // min-p * 2^shift
  float cap;                   // 61 octaves of weight, in the logit
  float bins_per_logit;
  const double* roots;         // 2^(shift - j / 64), in LDS

  // The workgroup's `lds` gets the roots; a barrier must follow before their use.
  DIP_DEV Weigher(const SampleArgs& a, uint32_t top_key, uint32_t least_key, double* lds)
      : Weigher(a, put_roots(a, lds), top_key, least_key) {}
  DIP_DEV static const double* put_roots(const SampleArgs& a, double* lds) {
    if (threadIdx.x < 64)
      lds[threadIdx.x] = __builtin_amdgcn_ldexp(kRoots.v[threadIdx.x], a.shift);
    return lds;
  }
  // `lds` has the roots.
  DIP_DEV Weigher(const SampleArgs& a, const double* lds, uint32_t top_key, uint32_t least_key)
      : per_hi(a.per_hi), per_lo(a.per_lo), least(a.least), roots(lds) {
    most = key_value(top_key);
    inf = most == INFINITY;
    if (inf) most = 0.f;
    cap = 64.f * 61 / per_hi;
    // bins reach down to the smallest logit, or to the weight that counts as 0
    const float range = fminf(most - key_value(least_key), 64.f * (a.shift + 1) / per_hi);
    bins_per_logit = range > 0.f && !inf ? fminf(kBins / range, 3e38f) : 0.f;
  }
  // The logits that the other functions take.
  DIP_DEV float value(float x) const {
    return !inf ? x : x == INFINITY ? 0.f : -INFINITY;
  }
  // w * 2^shift; less than 1 / 2, a whole number of 0, beyond `cap` and for -inf.
  DIP_DEV double scaled(float x) const {
    // most - x = hi + lo exactly.  (Of 16-bit numbers, too: they may lie as far apart in
    // magnitude as fp32's.  Without it their weights are off by up to 2e-6, and 250 rows
    // of 32003 bf16 logits take 17.0 us for 17.8.)
    const float hi = most - x, part = hi - most;
    const float low = ((most - (hi - part)) - (x + part)) * per_hi;
    const bool far = !(hi <= cap);
    constexpr float kRound = 12582912.f;  // 1.5 * 2^23: the sum's low bits are n
    const float t = fmaf(hi, per_hi, kRound), n = t - kRound;
    const float f = fmaf(-hi, per_lo, fmaf(-hi, per_hi, n)) - low;
    constexpr float c = 0.69314718055994530942f / 64;
    const float q = f * fmaf(f, fmaf(f, c * c * c / 6, c * c / 2), c);
    const uint32_t i = __float_as_uint(t);
    const double r = roots[i & 63];
    // the octaves off the exponent (a root's is 2^shift or less, 2^-14 at the least)
    const uint64_t w = __builtin_bit_cast(uint64_t, fma(r, (double)q, r));
    const uint32_t top = (uint32_t)(w >> 32) - ((i << 14) & 0xFFF00000u);
    const uint64_t v = (uint64_t)top << 32 | (uint32_t)w;
    return far ? 0.0 : __builtin_bit_cast(double, v);
  }
  // Rounded to a whole number: below 2^52, so the sum's low bits are it.
  DIP_DEV static unsigned long long whole(double w) {
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
  DIP_DEV unsigned long long whole_of(float x) const {
    return whole(scaled(x));
  }
  // The weight if min-p keeps it, else 0.
  DIP_DEV unsigned long long kept_whole(float x) const {
    const double w = scaled(x);
    return w >= least ? whole(w) : 0ull;
  }
  // Never lower for a smaller logit.
  DIP_DEV int bin(float x) const {
    return (int)fminf((most - x) * bins_per_logit, (float)(kBins - 1));
  }
  // The same of logits as they are, given by their keys.
  DIP_DEV double key_scaled(uint32_t k) const { return scaled(value(key_value(k))); }
  DIP_DEV unsigned long long key_whole(uint32_t k) const { return whole(key_scaled(k)); }
  DIP_DEV unsigned long long key_kept(uint32_t k) const {
    const double w = key_scaled(k);
    return w >= least ? whole(w) : 0ull;
  }
};

struct Cut {  // the last kept token of the order
  uint32_t key;
  int64_t index;
  DIP_DEV bool keeps(uint32_t k, int64_t i) const { return k > key || (k == key && i <= index); }
};

template <int kN = kThreads, typename T, typename F>
DIP_DEV T block_reduce(T v, F f, T* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = f(v, (T)__shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int i = 1; i < kN / 64; ++i) v = f(v, lds[i]);
  return v;
}

// The sum of the threads before this one; `total`: of all.
template <int kN = kThreads>
DIP_DEV uint64_t block_exclusive(uint64_t v, uint64_t* lds, uint64_t& total) {
  uint64_t run = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = __shfl_up(run, m, 64);
    if ((int)(threadIdx.x & 63) >= m) run += o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = run;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kN / 64; ++i) {
    if (i == (int)(threadIdx.x >> 6)) before = total;
    total += lds[i];
  }
  return before + run - v;
}

template <int kN>
constexpr int lds_words = 2 * (kN / 64) + 4;  // of the calls above and below
constexpr int kLdsWords = lds_words<kThreads>;

// The row's largest (order_key << 32 | ~index) and smallest logits, from the slices'.
DIP_DEV void row_ends(const SampleArgs& a, const RowState& st, uint64_t* lds, uint64_t& best,
                      uint32_t& least) {
  uint64_t b = 0;
  uint32_t l = 0xFFFFFFFFu;
  for (int s = threadIdx.x; s < a.slices; s += kThreads) {
    b = max(b, st.best[s]);
    l = min(l, st.least[s]);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    b = max(b, (uint64_t)__shfl_xor(b, m, 64));
    l = min(l, (uint32_t)__shfl_xor(l, m, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[2 * (threadIdx.x >> 6)] = b;
    lds[2 * (threadIdx.x >> 6) + 1] = l;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    b = max(b, lds[2 * i]);
    l = min(l, (uint32_t)lds[2 * i + 1]);
  }
  best = b;
  least = l;
}

template <int kN = kThreads, typename W>
DIP_DEV Plan make_plan(const SampleArgs& a, const uint32_t* hn, const unsigned long long* hw,
                       const W& wt, Plan p, uint64_t* lds) {
  constexpr int kPer = kBins / kN;
  uint64_t* sh = lds + 2 * (kN / 64);
  const int b0 = threadIdx.x * kPer;
  const bool some_k = a.top_k > 0 && a.top_k < a.vocab;  // else nobody counted the tokens
  uint64_t n[kPer], w[kPer], sn = 0, sw = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    n[i] = some_k ? hn[b0 + i] : 0;
    w[i] = hw[b0 + i];
    sn += n[i];
    sw += w[i];
  }
  uint64_t tokens = 0;
  const uint64_t bn = some_k ? block_exclusive<kN>(sn, lds, tokens) : 0;
  const uint64_t bw = block_exclusive<kN>(sw, lds, p.total);
  // the first bin at which `test(tokens, weights up to and with it)` holds, and
  // what lies before it, in sh[0 .. 2]
  auto first = [&](auto test) {
    __syncthreads();
    if (threadIdx.x == 0) sh[0] = kBins;
    __syncthreads();
    uint64_t cn = bn, cw = bw;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (!test(cn, cw) && test(cn + n[i], cw + w[i])) {
        sh[0] = (uint64_t)(b0 + i);
        sh[1] = cn;
        sh[2] = cw;
      }
      cn += n[i];
      cw += w[i];
    }
    __syncthreads();
  };
  p.by_k = some_k && (uint64_t)a.top_k < tokens;
  p.lo = p.hi = kBins;
  p.above_n = p.above_w = 0;
  uint64_t base = p.total;  // what top-p takes its share of, at least
  if (p.by_k) {
    first([&](uint64_t cn, uint64_t) { return cn >= (uint64_t)a.top_k; });
    p.lo = p.hi = (int)sh[0];
    p.above_n = sh[1];
    base = p.above_w = sh[2];
  }
  if (a.top_p < 1) {
    const double mass = a.top_p * (double)base;
    first([&](uint64_t, uint64_t cw) { return (double)cw >= mass && cw > 0; });
    if ((int)sh[0] < p.lo) {
      p.lo = (int)sh[0];
      p.above_n = sh[1];
      p.above_w = sh[2];
      if (!p.by_k) p.hi = p.lo;
    }
  }
  p.ranked = p.lo < kBins;
  // min-p's border: surely in the bins m .. m + 2.  If nothing is to be looked for
  // before their end, they alone are listed; if they begin before lo, from there on.
  if (a.least > 0) {
    const double bin = a.least_64ths / a.per_64th * wt.bins_per_logit;
    const int m = max(0, (bin < kBins ? (int)bin : kBins) - 1);
    if (m < p.lo && m < kBins) {
      if (m + 2 < p.lo) {
        p.ranked = 0;
        p.hi = m + 2;
      }
      p.lo = m;
      __syncthreads();
      if (b0 <= m && m < b0 + kPer) {
        uint64_t cn = bn, cw = bw;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (b0 + i < m) cn += n[i], cw += w[i];
        sh[1] = cn;
        sh[2] = cw;
      }
      __syncthreads();
      p.above_n = sh[1];
      p.above_w = sh[2];
    }
  }
  __syncthreads();
  return p;
}

// The border of the first `count` tokens (mass < 0), or of the fewest whose
// weights reach `mass`, among those that `kept` keeps: the key from its highest
// byte down, then the index among the tokens of that key.  A workgroup-wide call,
// for rows that the list cannot hold.
template <int kType, int kN = kThreads, typename W, typename K>
DIP_DEV Cut search_bits(const SampleArgs& a, const char* row, const W& wt, K kept,
                        uint64_t count, double mass, uint32_t* hn, unsigned long long* hw,
                        uint64_t* lds) {
  uint64_t* sh = lds + 2 * (kN / 64);
  const int tid = threadIdx.x;
  const bool by_mass = mass >= 0;
  const int64_t vecs = row_vecs<kType>(row, a.vocab);
  uint32_t prefix = 0;
  uint64_t above_n = 0, above_w = 0, ties = 0;
  for (int level = 24; level >= 0; level -= 8) {
    for (int b = tid; b < kRadixBins; b += kN) hn[b] = 0, hw[b] = 0;
    __syncthreads();
    each_token<kType, kN>(row, a.vocab, 0, vecs, [&](int64_t i, float x) {
      const uint32_t k = order_key(x);
      if (!kept(k, i) || (level < 24 && (k >> (level + 8)) != (prefix >> (level + 8)))) return;
      const unsigned long long w = wt.key_whole(k);
      if (w == 0) return;
      atomicAdd(&hn[(k >> level) & 255], 1u);
      atomicAdd(&hw[(k >> level) & 255], w);
    });
    __syncthreads();
    if (tid == 0) {
      uint64_t n = above_n, w = above_w;
      int b = kRadixBins - 1, last = 0;
      for (; b >= 0; --b) {
        if (hn[b]) {
          if (by_mass ? (double)(w + hw[b]) >= mass : n + hn[b] >= count) break;
          last = b;
        }
        n += hn[b];
        w += hw[b];
      }
      if (b < 0) {  // the sum falls short by its rounding: the last token there is
        b = last;
        n -= hn[b];
        w -= hw[b];
      }
      sh[0] = (uint64_t)b;
      sh[1] = n;
      sh[2] = w;
      sh[3] = hn[b];
    }
    __syncthreads();
    prefix |= (uint32_t)sh[0] << level;
    above_n = sh[1];
    above_w = sh[2];
    ties = sh[3];
    __syncthreads();
  }
  uint64_t need = count - above_n;
  if (by_mass) {
    const double n = ceil((mass - (double)above_w) / (double)wt.key_whole(prefix));
    need = n < 1.0 ? 1 : (n < (double)ties ? (uint64_t)n : ties);
  }
  // the index of the need-th token of that key
  const int64_t per = (a.vocab + kN - 1) / kN;
  const int64_t lo = min(tid * per, a.vocab), end = min(lo + per, a.vocab);
  uint64_t mine = 0, all;
  for (int64_t i = lo; i < end; ++i) mine += order_key(load_logit<kType>(row, i)) == prefix;
  const uint64_t before = block_exclusive<kN>(mine, lds, all);
  if (before < need && need <= before + mine) {
    uint64_t left = need - before;
    for (int64_t i = lo; i < end; ++i)
      if (order_key(load_logit<kType>(row, i)) == prefix && --left == 0) {
        sh[0] = (uint64_t)i;
        break;
      }
  }
  __syncthreads();
  const Cut c{prefix, (int64_t)sh[0]};
  __syncthreads();
  return c;
}

// v[0 .. n) in descending order (its values differ), `out` of as many words.
template <int kN = kThreads>
DIP_DEV void order_list(uint64_t* v, uint64_t* out, int n) {
  if (n <= kRankMax) {  // each one's place is the number of larger ones
    for (int i = threadIdx.x; i < n; i += kN) {
      const uint64_t x = v[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += v[j] > x;
      out[rank] = x;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kN) v[i] = out[i];
    __syncthreads();
    return;
  }
  int size = 2 * kRankMax;
  while (size < n) size *= 2;
  for (int i = n + (int)threadIdx.x; i < size; i += kN) v[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int step = run / 2; step > 0; step /= 2) {
      for (int t = threadIdx.x; t < size / 2; t += kN) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const bool down = (i & run) == 0;
        const uint64_t x = v[i], y = v[j];
        if (down ? x < y : x > y) {
          v[i] = y;
          v[j] = x;
        }
      }
      __syncthreads();
    }
}

// The last of the ordered list that top-k and top-p keep.
template <int kN, typename W>
DIP_DEV int last_kept(const SampleArgs& a, const Plan& p, const W& wt, const uint64_t* list,
                      int n, uint64_t* lds) {
  uint64_t* sh = lds + 2 * (kN / 64);
  int last = n - 1;
  if (!p.ranked) return last;
  // a run of `per` neighbours per thread, and the weights before it
  const int per = (n + kN - 1) / kN, i0 = min((int)threadIdx.x * per, n), i1 = min(i0 + per, n);
  uint64_t mine = 0, all;
  for (int i = i0; i < i1; ++i) mine += wt.key_whole((uint32_t)(list[i] >> 32));
  const uint64_t before = p.above_w + block_exclusive<kN>(mine, lds, all);
  if (p.by_k) last = (int)min((uint64_t)n, (uint64_t)a.top_k - p.above_n) - 1;
  if (a.top_p < 1) {
    if (threadIdx.x == 0) sh[1] = (uint64_t)last;
    uint64_t run = before;
    if (p.by_k) {  // the sum that top-p takes its share of
      for (int i = i0; i < i1; ++i) {
        run += wt.key_whole((uint32_t)(list[i] >> 32));
        if (i == last) sh[0] = run;
      }
    } else if (threadIdx.x == 0) {
      sh[0] = p.total;
    }
    __syncthreads();
    const double mass = a.top_p * (double)sh[0];
    run = before;
    for (int i = i0; i < i1; ++i) {
      const bool was = (double)run >= mass;
      run += wt.key_whole((uint32_t)(list[i] >> 32));
      if (i <= last && !was && (double)run >= mass) sh[1] = (uint64_t)i;
    }
    __syncthreads();
    last = (int)sh[1];
  }
  return last;
}

// The border that the bits give, for a row whose list overflows.
template <int kType, int kN = kThreads, typename W>
DIP_DEV Cut search_row(const SampleArgs& a, const Plan& p, const char* row, const W& wt,
                       uint32_t* hn, unsigned long long* hw, uint64_t* lds) {
  Cut cut{0u, a.vocab};
  auto kept = [&](uint32_t k, int64_t i) { return cut.keeps(k, i); };
  if (p.by_k)
    cut = search_bits<kType, kN>(a, row, wt, kept, (uint64_t)a.top_k, -1.0, hn, hw, lds);
  if (a.top_p < 1) {
    uint64_t w = 0;
    each_token<kType, kN>(row, a.vocab, 0, row_vecs<kType>(row, a.vocab), [&](int64_t i, float x) {
      const uint32_t k = order_key(x);
      if (kept(k, i)) w += wt.key_whole(k);
    });
    w = block_reduce<kN>(w, [](uint64_t x, uint64_t y) { return x + y; }, lds);
    cut = search_bits<kType, kN>(a, row, wt, kept, 0, a.top_p * (double)w, hn, hw, lds);
  }
  return cut;
}

// u's place among `total`; u beyond 1 or NaN: the last.
DIP_DEV uint64_t goal_of(double u, uint64_t total) {
  const double t = u * (double)total;
  return min(t < 0 ? 0 : t < (double)total ? (uint64_t)t : total - 1, total - 1);
}

// The border of a row that was looked through in slices, n of its tokens listed, and
// in `sums` (the weights that each slice is sure of) the slices' kept weights.
template <int kType, bool kHist>
DIP_DEV Cut cut_of_slices(const SampleArgs& a, const Plan& p, const char* row, const Weigher& wt,
                          int n, uint64_t* list, uint64_t* spare, unsigned long long* sums,
                          uint32_t* hn, unsigned long long* hw, uint64_t* lds) {
  const int tid = threadIdx.x;
  constexpr int kSize = kType == DIP_F32 ? 4 : 2, kVec = 16 / kSize;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize;
  auto slice_of = [&](int64_t i) { return (int)((i + off) / kVec / a.slice_vecs); };
  Cut cut{0u, a.vocab};
  if (kHist && n > kListMax) {
    cut = search_row<kType, kDrawThreads>(a, p, row, wt, hn, hw, lds);
    if (tid < a.slices) sums[tid] = 0;
    __syncthreads();
    each_token<kType, kDrawThreads>(
        row, a.vocab, 0, row_vecs<kType>(row, a.vocab), [&](int64_t i, float x) {
          const uint32_t k = order_key(x);
          if (!cut.keeps(k, i)) return;
          const unsigned long long w = wt.key_kept(k);
          if (w) atomicAdd(&sums[slice_of(i)], w);
        });
  } else if (kHist && n > 0) {
    order_list<kDrawThreads>(list, spare, n);
    const int last = last_kept<kDrawThreads>(a, p, wt, list, n, lds);
    const int per = (n + kDrawThreads - 1) / kDrawThreads;
    const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
    cut.key = (uint32_t)(list[last] >> 32);
    cut.index = (int64_t)(uint32_t)~(uint32_t)list[last];
    for (int i = i0; i < i1 && i <= last; ++i) {
      const unsigned long long x = wt.key_kept((uint32_t)(list[i] >> 32));
      if (x) atomicAdd(&sums[slice_of((int64_t)(uint32_t)~(uint32_t)list[i])], x);
    }
  }
  __syncthreads();
  return cut;
}

// Rows of up to kRowPieces pieces per thread are held in a workgroup's registers: thread
// t has the neighbouring pieces from t * per on, and `mine` visits its tokens.
constexpr int kRowPieces = 4;

// The border of such a row; hn and hw zero, *listed too.
template <int kType, int kN, typename M>
DIP_DEV Cut cut_of_row(const SampleArgs& a, Plan plan, const char* row, const Weigher& wt, M mine,
                       uint64_t* list, uint64_t* spare, uint32_t* listed, uint32_t* hn,
                       unsigned long long* hw, uint64_t* lds) {
  mine([&](int64_t, float x) {
    const float y = wt.value(x);
    const unsigned long long w = wt.whole_of(y);
    if (w == 0) return;
    const int b = wt.bin(y);
    atomicAdd(&hn[b], 1u);
    atomicAdd(&hw[b], w);
  });
  __syncthreads();
  plan = make_plan<kN>(a, hn, hw, wt, plan, lds);
  if (plan.lo < kBins) {
    mine([&](int64_t i, float x) {
      const float y = wt.value(x);
      const int b = wt.bin(y);
      if (b < plan.lo || b > plan.hi || wt.whole_of(y) == 0) return;
      const uint32_t to = atomicAdd(listed, 1u);
      if (to < kListMax) list[to] = (uint64_t)order_key(x) << 32 | (uint32_t)~(uint32_t)i;
    });
    __syncthreads();
    const int n = (int)min(*listed, (uint32_t)kListMax + 1);
    if (n > kListMax) {
      __syncthreads();
      return search_row<kType, kN>(a, plan, row, wt, hn, hw, lds);
    } else if (n > 0) {
      order_list<kN>(list, spare, n);
      const int last = last_kept<kN>(a, plan, wt, list, n, lds);
      return Cut{(uint32_t)(list[last] >> 32), (int64_t)(uint32_t)~(uint32_t)list[last]};
    }
  }
  return Cut{0u, a.vocab};
}

// Which rows are drawn in one launch: those of up to kOneLaunch pieces, and up to
// the most that the launch takes where there are many rows or nothing to count: a
// workgroup alone takes longer over a long row's histogram than slices do, and slices
// are more work.  Rows of 32003 bf16 logits in one launch and in slices, us, top-k 20
// and top-p 0.9: 1 row 31 for 21, 37 for 24; 48 rows 32 for 32, 39 for 33; 64 rows 32
// for 35, 39 for 35; 96 rows 32 for 41, 39 for 41; 256 rows 33 for 48, 40 for 51.  (Of
// 20001 they cross at 48 rows, of 9001 fp32 logits from the first.)  Without a filter
// 17 for 17 and, of 250 rows, 18 for 28.  256 threads while they have two pieces each
// at most, 1024 beyond (4000 bf16 logits 15 and 17 us, 8000 20 and 18).
constexpr int64_t kSmallRow = 512;
constexpr int64_t kOneLaunch = 2048;
constexpr int64_t kMostPieces = 1024 * kRowPieces;
constexpr int64_t kManyRows = 64;

inline bool counts(const SampleArgs& a) {
  return a.per_64th > 0 && ((a.top_k > 0 && a.top_k < a.vocab) || a.top_p < 1);
}

// The threads of the one workgroup that takes a row, 0: it goes in slices.
inline int row_threads(const SampleArgs& a, int64_t rows, int64_t vecs) {
  if (vecs <= kSmallRow) return kThreads;
  return vecs <= kOneLaunch || (vecs <= kMostPieces && (rows >= kManyRows || !counts(a))) ? 1024
                                                                                         : 0;
}

// Slices of a row: about a thousand workgroups in all, of 256 pieces at least; two
// thousand while these have ten pieces to a thread, as a slice's histogram costs the
// others' launches about as much as four.  (176 rows of 151936 fp32 logits with their
// draft's, verified with top-p and min-p, 96 us for 110, drawn from with min-p 250 rows
// 83 for 99; with two thousand in any case 64 rows with top-p 66 for 59.)
inline int slices_for(int64_t rows, int64_t vecs) {
  const int64_t want = max(max((int64_t)1, 1024 / rows), min(2048 / rows, vecs / 2560));
  const int64_t most = (vecs + 255) / 256;
  return (int)max((int64_t)1, min(min(want, most), (int64_t)kMaxSlices));
}
inline int64_t max_vecs(int64_t vocab, int size) { return (vocab * size + 15) / 16 + 1; }

// The filters and the slices of rows of `vocab` logits of a type, `size` bytes each.
inline SampleArgs sample_args(int64_t rows, int64_t vocab, int size, double temperature,
                              int64_t top_k, double top_p, double min_p) {
  int shift = 62;
  for (int64_t n = 1; n < vocab; n *= 2) --shift;
  shift = min(shift, 51);
  const int64_t vecs = max_vecs(vocab, size);
  SampleArgs a{};
  a.vocab = vocab;
  a.rows1 = (int)rows;
  a.top_p = top_p;
  // 0: greedy, which top-k 1 is at any temperature (one row of 151936 bf16 logits 25
  // us by way of its weights, 5 greedily); temperatures beyond 1e-30 and 1e30 count as these
  a.per_64th = temperature > 0 && top_k != 1
                   ? 64 * 1.4426950408889634074 / fmin(fmax(temperature, 1e-30), 1e30)
                   : 0;
  a.per_hi = (float)a.per_64th;
  a.per_lo = (float)(a.per_64th - a.per_hi);
  a.least = min_p * (double)(1ull << shift);
  a.least_64ths = min_p > 0 ? -log2(min_p) * 64 : 0;
  a.top_k = top_k;
  a.shift = shift;
  a.slices = slices_for(rows, vecs);
  a.slice_vecs = (vecs + a.slices - 1) / a.slices;
  a.row_ws = (int64_t)(sizeof(RowState) + (size_t)a.slices * kBins * sizeof(uint64_t));
  return a;
}

// Whether the library takes the logits' type and the filters.
inline int check_sampling(int dtype, int64_t vocab, double temperature, int64_t top_k,
                          double top_p, double min_p) {
  if (dtype != DIP_BF16 && dtype != DIP_F16 && dtype != DIP_F32) return DIP_ERR_UNSUPPORTED;
  if (vocab <= 0 || vocab > (1 << 30)) return DIP_ERR_SHAPE;
  if (!(temperature >= 0) || temperature > 1e300 || top_k < 0 || !(top_p > 0 && top_p <= 1) ||
      !(min_p >= 0 && min_p <= 1))
    return DIP_ERR_ARG;
  return DIP_OK;
}


}  // namespace
}  // namespace dip
