// dip_sample.hip — drawing the next token from logits: temperature, top-k,
// top-p and min-p, then the inverse of the distribution at a given number.
//
// With the tokens in the order (logit descending, index ascending) and weights
// w = exp((logit - max) / temperature), a prefix of that order is kept:
//   top-k  the first k tokens;
//   top-p  of those, the fewest whose weights reach p times their sum;
//   min-p  of those, the ones with w >= min_p.
// The token is the first one, by index, at which the running sum of the kept
// weights exceeds u times their sum.  The border of the kept prefix is a pair
// (logit, index), so ties are cut by index and the row is never sorted.
//
// A weight is a whole number, w * 2^shift rounded (shift such that a row's sum
// stays below 2^63; w in 64 bits): sums are exact, in any order and by any
// atomics, so the token does not depend on how a row is split.  In 32 bits a sum
// over 150000 tokens is off by more than an unlikely token's weight.  Weights
// below 2^-shift / 2 (2^-45 at 150000 tokens) are 0 and never drawn.
//
// Each row is cut into slices, one workgroup each, in up to four launches:
//   max     the largest logit of each slice (with its index), and the smallest;
//   hist    tokens and their weights counted in kBins bins of even width in the
//           logit, per slice in LDS, then added to the row's;
//   gather  from the histogram every slice finds the bins that can hold a border;
//           it adds up the weights of the bins before them and lists the tokens in
//           them;
//   draw    one workgroup per row sorts the list (a few to a few hundred tokens),
//           finds the border, the slice that the draw falls in, and the token in
//           it.  Rows whose list overflows (thousands of equal logits) are
//           searched by the bits of the logit instead.
// Without top-k and top-p there is no histogram, greedy draws need the first
// launch and a choice among its results.
#include "dip_common.h"
#include "dip_internal.h"

#include <hip/hip_fp16.h>

namespace dip {
namespace {

constexpr int kThreads = 1024;      // draw
constexpr int kSliceThreads = 256;  // the other launches
constexpr int kBins = 1024;
constexpr int kListMax = 4096;
constexpr int kMaxSlices = 256;
constexpr int kRadixBins = 256;
constexpr uint32_t kKeyMinusInf = 0x007FFFFFu;  // order_key of -inf, and of NaN

// fp32 as a whole number that orders like it, -0 as 0 and NaN as -inf.
DIP_DEV uint32_t order_key(float x) {
  x += 0.f;
  if (x != x) return kKeyMinusInf;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
DIP_DEV float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

template <int kType>
DIP_DEV float load_logit(const void* row, int64_t i) {
  if (kType == DIP_F32) return static_cast<const float*>(row)[i];
  if (kType == DIP_F16) return __half2float(static_cast<const __half*>(row)[i]);
  return bf16_to_f32(static_cast<const uint16_t*>(row)[i]);
}

// A row's workspace.
struct RowState {
  uint64_t best[kMaxSlices];         // per slice: order_key << 32 | ~index of its largest
  uint32_t least[kMaxSlices];        // smallest order_key above -inf
  unsigned long long sure[kMaxSlices];  // weights before the bins of the list
  unsigned long long hw[kBins];      // histogram: weights, tokens
  uint32_t hn[kBins];
  uint32_t listed;
  uint32_t pad;
  uint64_t list[kListMax];           // order_key << 32 | ~index
};

struct SampleArgs {
  const void* logits;
  int64_t vocab, row_bytes;
  const float* u;
  double temperature, top_p, min_p;
  int64_t top_k;
  int shift;
  int slices;
  int64_t slice_vecs;  // 16-byte pieces of a row that a slice takes
  RowState* rows;
  int64_t* token;
  float* prob;
};

DIP_DEV const char* row_of(const SampleArgs& a, int r) {
  return static_cast<const char*>(a.logits) + (int64_t)r * a.row_bytes;
}

// f(index, order_key) of every token in the 16-byte pieces [v0, v1) of a row, by
// `threads` threads.  Pieces lie where memory has them; one that reaches over an
// end of the row is loaded token by token.
template <int kType, typename F>
DIP_DEV void each_token(const char* row, int64_t vocab, int64_t v0, int64_t v1, int tid,
                        int threads, F f) {
  constexpr int kSize = kType == DIP_F32 ? 4 : 2, kVec = 16 / kSize;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize;
  for (int64_t v = v0 + tid; v < v1; v += threads) {
    const int64_t e0 = v * kVec - off;
    if (e0 >= 0 && e0 + kVec <= vocab) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + e0 * kSize);
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t b = kSize == 4 ? x[i] : (x[i / 2] >> (16 * (i & 1))) & 0xFFFFu;
        const float l = kType == DIP_F32   ? __uint_as_float(b)
                        : kType == DIP_F16 ? __half2float(__ushort_as_half((unsigned short)b))
                                           : bf16_to_f32(b);
        f(e0 + i, order_key(l));
      }
    } else {
      for (int i = 0; i < kVec; ++i)
        if (e0 + i >= 0 && e0 + i < vocab)
          f(e0 + i, order_key(load_logit<kType>(row, e0 + i)));
    }
  }
}

template <int kType>
DIP_DEV int64_t row_vecs(const char* row, int64_t vocab) {
  constexpr int kSize = kType == DIP_F32 ? 4 : 2;
  return ((reinterpret_cast<uintptr_t>(row) & 15) + vocab * kSize + 15) / 16;
}

// What a row's largest logit makes of the others.
struct Weigher {
  uint32_t top;
  double most, per_log2;  // logits per factor of 2
  float bins_per_logit;
  double scale, min_p;

  DIP_DEV Weigher(const SampleArgs& a, uint32_t top_key, uint32_t least_key) : top(top_key) {
    most = key_value(top);
    per_log2 = 1.4426950408889634074 / a.temperature;
    scale = (double)(1ull << a.shift);
    min_p = a.min_p;
    // bins reach down to the smallest logit, or to the weight that counts as 0
    const double range = min(most - (double)key_value(least_key), (a.shift + 1) / per_log2);
    bins_per_logit = range > 0 ? (float)(kBins / range) : 0.f;
  }
  DIP_DEV double weight(uint32_t k) const {
    if (k == top) return 1.0;
    if (k <= kKeyMinusInf) return 0.0;
    return exp2(((double)key_value(k) - most) * per_log2);
  }
  DIP_DEV unsigned long long whole(double w) const { return (unsigned long long)(w * scale + 0.5); }
  DIP_DEV unsigned long long whole_of(uint32_t k) const { return whole(weight(k)); }
  // The weight if min-p keeps it, else 0.
  DIP_DEV unsigned long long kept_whole(uint32_t k) const {
    const double w = weight(k);
    return w >= min_p ? whole(w) : 0ull;
  }
  // Never lower for a smaller logit.
  DIP_DEV int bin(uint32_t k) const {
    if (k == top) return 0;
    return (int)fminf(((float)most - key_value(k)) * bins_per_logit, (float)(kBins - 1));
  }
};

struct Cut {  // the last kept token of the order
  uint32_t key;
  int64_t index;
};

template <int kN, typename T, typename F>
DIP_DEV T block_reduce(T v, F f, T* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = f(v, (T)__shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int i = 1; i < kN / 64; ++i) v = f(v, lds[i]);
  return v;
}

// The sum of the threads before this one; `total`: of all.
template <int kN, typename T>
DIP_DEV T block_exclusive(T v, T* lds, T& total) {
  T run = v;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const T o = __shfl_up(run, m, 64);
    if ((int)(threadIdx.x & 63) >= m) run += o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = run;
  __syncthreads();
  T before = 0;
  total = 0;
  for (int i = 0; i < kN / 64; ++i) {
    if (i == (int)(threadIdx.x >> 6)) before = total;
    total += lds[i];
  }
  return before + run - v;
}

// The row's largest and smallest logits from the slices' (one workgroup-wide
// call; every thread gets them).
template <int kN>
DIP_DEV void row_ends(const SampleArgs& a, const RowState& st, uint64_t* lds, uint64_t& best,
                      uint32_t& least) {
  uint64_t b = 0;
  uint32_t l = 0xFFFFFFFFu;
  for (int s = threadIdx.x; s < a.slices; s += kN) {
    b = max(b, st.best[s]);
    l = min(l, st.least[s]);
  }
  best = block_reduce<kN>(b, [](uint64_t x, uint64_t y) { return max(x, y); }, lds);
  least = block_reduce<kN>(l, [](uint32_t x, uint32_t y) { return min(x, y); },
                           reinterpret_cast<uint32_t*>(lds));
}

// Where the histogram says that the border lies.
struct Plan {
  int lo, hi;              // the bins to list; lo = kBins: none
  uint64_t above_n, above_w;  // tokens and weights of the bins before lo
  uint64_t tokens, total;  // of all bins
};

// One workgroup-wide call.  lds: 4 kN / 64 + 4 words of 64 bits.
template <int kN>
DIP_DEV Plan make_plan(const SampleArgs& a, const RowState& st, const Weigher& wt, uint64_t* lds) {
  constexpr int kPer = (kBins + kN - 1) / kN;
  uint64_t* sh = lds + 2 * (kN / 64);
  const int b0 = threadIdx.x * kPer;
  uint64_t n[kPer], w[kPer], sn = 0, sw = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    n[i] = b0 + i < kBins ? st.hn[b0 + i] : 0;
    w[i] = b0 + i < kBins ? st.hw[b0 + i] : 0;
    sn += n[i];
    sw += w[i];
  }
  Plan p;
  const uint64_t bn = block_exclusive<kN>(sn, lds, p.tokens);
  const uint64_t bw = block_exclusive<kN>(sw, lds, p.total);
  // the first bin at which `test(tokens, weights up to and with it)` holds: its
  // number, and tokens and weights before it
  auto first = [&](auto test) {
    __syncthreads();
    if (threadIdx.x == 0) sh[0] = kBins;
    __syncthreads();
    uint64_t cn = bn, cw = bw;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool before = test(cn, cw);
      if (b0 + i < kBins && !before && test(cn + n[i], cw + w[i])) {
        sh[0] = (uint64_t)(b0 + i);
        sh[1] = cn;
        sh[2] = cw;
      }
      cn += n[i];
      cw += w[i];
    }
    __syncthreads();
  };
  const bool by_k = a.top_k > 0 && (uint64_t)a.top_k < p.tokens;
  p.lo = p.hi = kBins;
  p.above_n = p.above_w = 0;
  uint64_t base = p.total;  // what top-p takes its share of, at least
  if (by_k) {
    first([&](uint64_t cn, uint64_t) { return cn >= (uint64_t)a.top_k; });
    p.lo = p.hi = (int)sh[0];
    p.above_n = sh[1];
    p.above_w = sh[2];
    base = sh[2];
  }
  if (a.top_p < 1) {
    const double mass = a.top_p * (double)base;
    first([&](uint64_t, uint64_t cw) { return (double)cw >= mass && cw > 0; });
    if ((int)sh[0] < p.lo) {
      p.lo = (int)sh[0];
      p.above_n = sh[1];
      p.above_w = sh[2];
    }
    if (!by_k) p.hi = p.lo;
  }
  // min-p alone cuts before the first bin to list: nothing to look for
  if (p.lo < kBins && a.min_p > 0) {
    const double least = wt.most + log2(a.min_p) / wt.per_log2;
    const double bin = (wt.most - least) * wt.bins_per_logit;
    if (p.lo > bin + 2) p.lo = p.hi = kBins;
  }
  __syncthreads();
  return p;
}

template <int kType>
__global__ __launch_bounds__(kSliceThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kSliceThreads / 64];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  RowState& st = a.rows[r];
  uint64_t best = 0;
  uint32_t least = 0xFFFFFFFFu;
  each_token<kType>(row, a.vocab, s * a.slice_vecs,
                    min((s + 1) * a.slice_vecs, row_vecs<kType>(row, a.vocab)), threadIdx.x,
                    kSliceThreads, [&](int64_t i, uint32_t k) {
                      best = max(best, (uint64_t)k << 32 | (uint32_t)~(uint32_t)i);
                      if (k > kKeyMinusInf) least = min(least, k);
                    });
  best = block_reduce<kSliceThreads>(best, [](uint64_t x, uint64_t y) { return max(x, y); }, lds);
  least = block_reduce<kSliceThreads>(least, [](uint32_t x, uint32_t y) { return min(x, y); },
                                      reinterpret_cast<uint32_t*>(lds));
  if (threadIdx.x == 0) {
    st.best[s] = best;
    st.least[s] = least;
    if (s == 0) st.listed = 0;
  }
  for (int b = s * kSliceThreads + threadIdx.x; b < kBins; b += a.slices * kSliceThreads) {
    st.hn[b] = 0;
    st.hw[b] = 0;
  }
}

template <int kType>
__global__ __launch_bounds__(kSliceThreads) void sample_hist_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kSliceThreads / 64];
  __shared__ uint32_t hn[kBins];
  __shared__ unsigned long long hw[kBins];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  RowState& st = a.rows[r];
  for (int b = threadIdx.x; b < kBins; b += kSliceThreads) hn[b] = 0, hw[b] = 0;
  uint64_t best;
  uint32_t least;
  row_ends<kSliceThreads>(a, st, lds, best, least);
  const uint32_t top = (uint32_t)(best >> 32);
  if (top <= kKeyMinusInf) return;
  const Weigher wt(a, top, least);
  __syncthreads();
  each_token<kType>(row, a.vocab, s * a.slice_vecs,
                    min((s + 1) * a.slice_vecs, row_vecs<kType>(row, a.vocab)), threadIdx.x,
                    kSliceThreads, [&](int64_t, uint32_t k) {
                      const unsigned long long w = wt.whole_of(k);
                      if (w == 0) return;
                      const int b = wt.bin(k);
                      atomicAdd(&hn[b], 1u);
                      atomicAdd(&hw[b], w);
                    });
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSliceThreads)
    if (hn[b]) {
      atomicAdd(&st.hn[b], hn[b]);
      atomicAdd(&st.hw[b], hw[b]);
    }
}

// kHist: the histogram has been made.
template <int kType, bool kHist>
__global__ __launch_bounds__(kSliceThreads) void sample_gather_kernel(SampleArgs a) {
  __shared__ uint64_t lds[4 * (kSliceThreads / 64) + 4];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  RowState& st = a.rows[r];
  uint64_t best;
  uint32_t least;
  row_ends<kSliceThreads>(a, st, lds, best, least);
  const uint32_t top = (uint32_t)(best >> 32);
  if (top <= kKeyMinusInf) return;
  const Weigher wt(a, top, least);
  int lo = kBins, hi = kBins;
  if (kHist) {
    const Plan p = make_plan<kSliceThreads>(a, st, wt, lds);
    lo = p.lo;
    hi = p.hi;
  }
  uint64_t sure = 0;
  each_token<kType>(row, a.vocab, s * a.slice_vecs,
                    min((s + 1) * a.slice_vecs, row_vecs<kType>(row, a.vocab)), threadIdx.x,
                    kSliceThreads, [&](int64_t i, uint32_t k) {
                      if (k <= kKeyMinusInf) return;
                      const int b = kHist ? wt.bin(k) : 0;
                      if (b < lo) {
                        sure += wt.kept_whole(k);
                      } else if (b <= hi && wt.whole_of(k) > 0) {
                        const uint32_t at = atomicAdd(&st.listed, 1u);
                        if (at < kListMax) st.list[at] = (uint64_t)k << 32 | (uint32_t)~(uint32_t)i;
                      }
                    });
  sure = block_reduce<kSliceThreads>(sure, [](uint64_t x, uint64_t y) { return x + y; }, lds);
  if (threadIdx.x == 0) st.sure[s] = sure;
}

// The border of the first `count` tokens (mass < 0), or of the fewest whose
// weights reach `mass`, among those that `kept` keeps: the key from its highest
// byte down, then the index among the tokens of that key.  A workgroup-wide call,
// for rows that the list cannot hold.
template <int kType, typename K>
DIP_DEV Cut search_bits(const SampleArgs& a, const char* row, const Weigher& wt, K kept,
                        uint64_t count, double mass, uint32_t* hn, unsigned long long* hw,
                        uint64_t* lds) {
  uint64_t* sh = lds + 2 * (kThreads / 64);
  const int tid = threadIdx.x;
  const bool by_mass = mass >= 0;
  const int64_t vecs = row_vecs<kType>(row, a.vocab);
  uint32_t prefix = 0;
  uint64_t above_n = 0, above_w = 0, ties = 0;
  for (int level = 24; level >= 0; level -= 8) {
    for (int b = tid; b < kRadixBins; b += kThreads) hn[b] = 0, hw[b] = 0;
    __syncthreads();
    each_token<kType>(row, a.vocab, 0, vecs, tid, kThreads, [&](int64_t i, uint32_t k) {
      if (!kept(k, i) || (level < 24 && (k >> (level + 8)) != (prefix >> (level + 8)))) return;
      const unsigned long long w = wt.whole_of(k);
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
    const double n = ceil((mass - (double)above_w) / (double)wt.whole_of(prefix));
    need = n < 1.0 ? 1 : (n < (double)ties ? (uint64_t)n : ties);
  }
  // the index of the need-th token of that key
  const int64_t per = (a.vocab + kThreads - 1) / kThreads;
  const int64_t lo = min(tid * per, a.vocab), end = min(lo + per, a.vocab);
  uint64_t mine = 0, all;
  for (int64_t i = lo; i < end; ++i) mine += order_key(load_logit<kType>(row, i)) == prefix;
  const uint64_t before = block_exclusive<kThreads>(mine, lds, all);
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

// Descending, n a power of two.
DIP_DEV void sort_list(uint64_t* v, int n) {
  for (int size = 2; size <= n; size *= 2)
    for (int step = size / 2; step > 0; step /= 2) {
      for (int t = threadIdx.x; t < n / 2; t += kThreads) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const bool down = (i & size) == 0;
        const uint64_t x = v[i], y = v[j];
        if (down ? x < y : x > y) {
          v[i] = y;
          v[j] = x;
        }
      }
      __syncthreads();
    }
}

template <int kType, bool kHist>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a) {
  __shared__ uint64_t lds[4 * (kThreads / 64) + 4];
  __shared__ uint64_t list[kListMax];
  __shared__ unsigned long long sums[kMaxSlices];
  __shared__ uint32_t hn[kRadixBins];
  __shared__ unsigned long long hw[kRadixBins];
  const int r = blockIdx.x, tid = threadIdx.x;
  const char* row = row_of(a, r);
  RowState& st = a.rows[r];
  uint64_t* sh = lds + 2 * (kThreads / 64);
  uint64_t best;
  uint32_t least;
  row_ends<kThreads>(a, st, lds, best, least);
  const uint32_t top = (uint32_t)(best >> 32);
  if (top <= kKeyMinusInf || a.temperature == 0) {  // nothing to choose from, or greedy
    if (tid == 0) {
      const bool some = top > kKeyMinusInf;
      a.token[r] = some ? (int64_t)(uint32_t)~(uint32_t)best : 0;
      if (a.prob) a.prob[r] = some ? 1.f : 0.f;
    }
    return;
  }
  const Weigher wt(a, top, least);
  constexpr int kSize = kType == DIP_F32 ? 4 : 2, kVec = 16 / kSize;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize;
  auto slice_of = [&](int64_t i) { return (int)((i + off) / kVec / a.slice_vecs); };
  for (int s = tid; s < a.slices; s += kThreads) sums[s] = st.sure[s];
  Cut cut{0u, a.vocab};
  auto kept = [&](uint32_t k, int64_t i) { return k > cut.key || (k == cut.key && i <= cut.index); };
  if (kHist) {
    const Plan p = make_plan<kThreads>(a, st, wt, lds);
    const bool by_k = a.top_k > 0 && (uint64_t)a.top_k < p.tokens;
    const uint32_t n = p.lo < kBins ? st.listed : 0u;
    if (n > kListMax) {
      if (by_k)
        cut = search_bits<kType>(a, row, wt, kept, (uint64_t)a.top_k, -1.0, hn, hw, lds);
      if (a.top_p < 1) {
        uint64_t w = 0;
        each_token<kType>(row, a.vocab, 0, row_vecs<kType>(row, a.vocab), tid, kThreads,
                          [&](int64_t i, uint32_t k) {
                            if (kept(k, i)) w += wt.whole_of(k);
                          });
        w = block_reduce<kThreads>(w, [](uint64_t x, uint64_t y) { return x + y; }, lds);
        cut = search_bits<kType>(a, row, wt, kept, 0, a.top_p * (double)w, hn, hw, lds);
      }
      for (int s = tid; s < a.slices; s += kThreads) sums[s] = 0;
      __syncthreads();
      each_token<kType>(row, a.vocab, 0, row_vecs<kType>(row, a.vocab), tid, kThreads,
                        [&](int64_t i, uint32_t k) {
                          if (!kept(k, i)) return;
                          const unsigned long long w = wt.kept_whole(k);
                          if (w) atomicAdd(&sums[slice_of(i)], w);
                        });
    } else if (n > 0) {
      int size = 64;
      while (size < (int)n) size *= 2;
      for (int i = tid; i < size; i += kThreads) list[i] = i < (int)n ? st.list[i] : 0;
      __syncthreads();
      sort_list(list, size);
      // kPer neighbours per thread, and the weights before them
      constexpr int kPer = kListMax / kThreads;
      unsigned long long w[kPer];
      uint64_t mine = 0, all;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = tid * kPer + e;
        w[e] = i < (int)n ? wt.whole_of((uint32_t)(list[i] >> 32)) : 0;
        mine += w[e];
      }
      const uint64_t before = block_exclusive<kThreads>(mine, lds, all);
      const int nk = by_k ? (int)min((uint64_t)n, (uint64_t)a.top_k - p.above_n) : (int)n;
      int last = nk - 1;  // of the list, kept
      if (a.top_p < 1) {
        // the sum that top-p takes its share of
        if (tid == 0) sh[1] = (uint64_t)nk;
        if (by_k) {
          uint64_t run = before;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            run += w[e];
            if (tid * kPer + e == nk - 1) sh[0] = p.above_w + run;
          }
        } else if (tid == 0) {
          sh[0] = p.total;
        }
        __syncthreads();
        const double mass = a.top_p * (double)sh[0];
        uint64_t run = p.above_w + before;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const bool was = (double)run >= mass;
          run += w[e];
          if (tid * kPer + e < nk && !was && (double)run >= mass) sh[1] = (uint64_t)(tid * kPer + e);
        }
        __syncthreads();
        last = min(last, (int)sh[1]);
      }
      cut.key = (uint32_t)(list[last] >> 32);
      cut.index = (int64_t)(uint32_t)~(uint32_t)list[last];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = tid * kPer + e;
        if (i > last) continue;
        const unsigned long long x = wt.kept_whole((uint32_t)(list[i] >> 32));
        if (x) atomicAdd(&sums[slice_of((int64_t)(uint32_t)~(uint32_t)list[i])], x);
      }
    }
  }
  __syncthreads();
  // the slice, then the token in it: running sums by index
  uint64_t total;
  const uint64_t mine = tid < a.slices ? sums[tid] : 0;
  const uint64_t before = block_exclusive<kThreads>(mine, lds, total);
  // u beyond 1 or NaN: the last kept token
  double t = (double)a.u[r] * (double)total;
  uint64_t goal = t >= 0 ? (t < (double)total ? (uint64_t)t : total - 1) : (t < 0 ? 0 : total - 1);
  goal = min(goal, total - 1);
  if (goal >= before && goal - before < mine) {
    sh[0] = (uint64_t)tid;
    sh[1] = before;
  }
  __syncthreads();
  const int s = (int)sh[0];
  goal -= sh[1];  // within the slice
  const int64_t lo = max((int64_t)0, s * a.slice_vecs * kVec - off);
  const int64_t end = min((s + 1) * a.slice_vecs * kVec - off, a.vocab);
  const int64_t per = (end - lo + kThreads - 1) / kThreads;
  const int64_t i0 = min(lo + tid * per, end), i1 = min(i0 + per, end);
  uint64_t here = 0, in_slice;
  for (int64_t i = i0; i < i1; ++i) {
    const uint32_t k = order_key(load_logit<kType>(row, i));
    if (k > kKeyMinusInf && kept(k, i)) here += wt.kept_whole(k);
  }
  uint64_t run = block_exclusive<kThreads>(here, lds, in_slice);
  if (goal >= run && goal - run < here) {
    for (int64_t i = i0; i < i1; ++i) {
      const uint32_t k = order_key(load_logit<kType>(row, i));
      if (k <= kKeyMinusInf || !kept(k, i)) continue;
      run += wt.kept_whole(k);
      if (run > goal) {
        a.token[r] = i;
        if (a.prob) a.prob[r] = (float)(wt.weight(k) * wt.scale / (double)total);
        break;
      }
    }
  }
}

// Slices of a row: about a thousand workgroups in all, of 512 pieces at least.
inline int slices_for(int64_t rows, int64_t vecs) {
  const int64_t want = max((int64_t)1, 1024 / rows), most = (vecs + 511) / 512;
  return (int)max((int64_t)1, min(min(want, most), (int64_t)kMaxSlices));
}

template <int kType>
int launch_sample(const SampleArgs& a, int rows, hipStream_t s) {
  const dim3 grid((unsigned)rows * a.slices), slice(kSliceThreads);
  hipLaunchKernelGGL((sample_max_kernel<kType>), grid, slice, 0, s, a);
  const bool hist = a.temperature > 0 && ((a.top_k > 0 && a.top_k < a.vocab) || a.top_p < 1);
  if (hist) {
    hipLaunchKernelGGL((sample_hist_kernel<kType>), grid, slice, 0, s, a);
    hipLaunchKernelGGL((sample_gather_kernel<kType, true>), grid, slice, 0, s, a);
    hipLaunchKernelGGL((sample_draw_kernel<kType, true>), dim3(rows), dim3(kThreads), 0, s, a);
  } else {
    if (a.temperature > 0)
      hipLaunchKernelGGL((sample_gather_kernel<kType, false>), grid, slice, 0, s, a);
    hipLaunchKernelGGL((sample_draw_kernel<kType, false>), dim3(rows), dim3(kThreads), 0, s, a);
  }
  return hip_status(hipGetLastError());
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" size_t dip_sample_workspace_size(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  return (size_t)rows * sizeof(RowState);
}

extern "C" int dip_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                          int64_t row_stride, const float* u, double temperature, int64_t top_k,
                          double top_p, double min_p, int64_t* token, float* prob,
                          void* workspace, size_t ws_bytes, void* stream) {
  if (dtype != DIP_BF16 && dtype != DIP_F16 && dtype != DIP_F32) return DIP_ERR_UNSUPPORTED;
  if (rows < 0 || rows > (1 << 22) || vocab <= 0 || vocab > (1 << 30) || row_stride < 0)
    return DIP_ERR_SHAPE;
  if (!(temperature >= 0) || temperature > 1e300 || top_k < 0 || !(top_p > 0 && top_p <= 1) ||
      !(min_p >= 0 && min_p <= 1))
    return DIP_ERR_ARG;
  if (rows == 0) return DIP_OK;
  if (!logits || !u || !token) return DIP_ERR_NULL;
  if (!workspace || ws_bytes < dip_sample_workspace_size(rows, vocab)) return DIP_ERR_WORKSPACE;
  const int size = dtype == DIP_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size || !aligned16(workspace)) return DIP_ERR_ALIGN;
  int shift = 62;
  for (int64_t n = 1; n < vocab; n *= 2) --shift;
  const int64_t vecs = (vocab * size + 15) / 16 + 1;
  const int slices = slices_for(rows, vecs);
  SampleArgs a{logits, vocab, row_stride * size, u, temperature, top_p, min_p, top_k, shift, slices,
               (vecs + slices - 1) / slices, static_cast<RowState*>(workspace), token, prob};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DIP_F32) return launch_sample<DIP_F32>(a, (int)rows, s);
  if (dtype == DIP_F16) return launch_sample<DIP_F16>(a, (int)rows, s);
  return launch_sample<DIP_BF16>(a, (int)rows, s);
}
