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
// A weight is a whole number of 64 bits, w * 2^shift rounded (shift such that a
// row's sum stays below 2^63, 51 at most; w is off by 4e-10, see Weigher): sums are
// exact, in any order and by any atomics, so the token does not depend on how a row
// is split.  In 32 bits a sum over 150000 tokens is off by more than an unlikely
// token's weight.  Weights below 2^-shift / 2 (2^-45 at 150000 tokens) are 0 and
// never drawn.
//
// Each row is cut into slices, one workgroup each, in up to four launches:
//   max     the largest logit of each slice (with its index), and the smallest;
//   hist    the weights of the tokens, and their number, added up in kBins bins of
//           even width in the logit: in LDS, kept per slice, and added to the row's;
//   gather  from the row's histogram every slice finds the bins that can hold a
//           border; it adds up its own bins before them and lists its tokens in them;
//   draw    one workgroup per row orders the list (a few to a few hundred tokens),
//           finds the border, the slice that the draw falls in, and the token in
//           it.  Rows whose list overflows (thousands of equal logits) are
//           searched by the bits of the logit instead.
// Without top-k and top-p there is no histogram; greedy draws need the first launch
// and a choice among its results.  Short rows go through all of it in one launch.
//
// 64 rows of 151936 fp32 logits (39 MB), top-p: 9 us for max, at the memory's rate;
// 19 for hist, which makes and bins each weight; 13 for gather, most of which is
// finding the borders; 9 for draw.  One row of bf16: 3, 6.5, 7 and 7.5 us, all waits
// on memory and barriers.
#include "dip_sample.h"

namespace dip {
namespace {

// kIndex: of equal ones the first, for greedy draws.
template <int kType, bool kIndex>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kLdsWords];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  RowState& st = row_state(a, r);
  float most = -INFINITY, low = INFINITY;
  int64_t at = 0;  // a thread's tokens come in ascending order
  each_token<kType>(row, a.vocab, s * a.slice_vecs,
                    min((s + 1) * a.slice_vecs, row_vecs<kType>(row, a.vocab)),
                    [&](int64_t i, float x) {
                      if (kIndex) at = x > most ? i : at;
                      most = fmaxf(most, x);
                      if (!kIndex) low = fminf(low, x == -INFINITY ? INFINITY : x);
                    });
  uint64_t best = (uint64_t)order_key(most) << 32 | (uint32_t)~(uint32_t)at;
  best = block_reduce(best, [](uint64_t x, uint64_t y) { return max(x, y); }, lds);
  const uint32_t least = block_reduce(order_key(low), [](uint32_t x, uint32_t y) { return min(x, y); },
                                      reinterpret_cast<uint32_t*>(lds));
  if (threadIdx.x == 0) {
    st.best[s] = best;
    st.least[s] = least;
    if (s == 0) st.listed = 0;
  }
  if (kIndex) return;
  for (int b = s * kThreads + threadIdx.x; b < kBins; b += a.slices * kThreads) {
    st.hn[b] = 0;
    st.hw[b] = 0;
  }
}

// kCount: top-k needs the number of tokens in the bins too.
template <int kType, bool kCount>
__global__ __launch_bounds__(kThreads) void sample_hist_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kLdsWords];
  __shared__ double roots[64];
  __shared__ uint32_t hn[kCount ? kBins : 1];
  __shared__ unsigned long long hw[kBins];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  RowState& st = row_state(a, r);
  const int64_t v0 = s * a.slice_vecs;
  const int64_t v1 = min(v0 + a.slice_vecs, row_vecs<kType>(row, a.vocab));
  const Piece<kType> head(row, a.vocab, v0 + threadIdx.x);
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    if (kCount) hn[b] = 0;
    hw[b] = 0;
  }
  uint64_t best;
  uint32_t least;
  row_ends(a, st, lds, best, least);
  const uint32_t top = (uint32_t)(best >> 32);
  if (top <= kKeyMinusInf) return;
  const Weigher wt(a, top, least, roots);
  __syncthreads();
  const auto add = [&](int64_t, float x) {
    const unsigned long long w = wt.whole_of(x);
    if (w == 0) return;
    const int b = wt.bin(x);
    if (kCount) atomicAdd(&hn[b], 1u);
    atomicAdd(&hw[b], w);
  };
  if (wt.inf)
    each_token<kType>(head, row, a.vocab, v0, v1, [&](int64_t i, float x) { add(i, wt.value(x)); });
  else
    each_token<kType>(head, row, a.vocab, v0, v1, add);
  __syncthreads();
  unsigned long long* own = slice_hist(a, r, s);
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    own[b] = hw[b];
    if (!hw[b]) continue;
    if (kCount) atomicAdd(&st.hn[b], hn[b]);
    atomicAdd(&st.hw[b], hw[b]);
  }
}

// kHist: the histogram has been made.
template <int kType, bool kHist>
__global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kLdsWords];
  __shared__ double roots[64];
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  RowState& st = row_state(a, r);
  const int64_t v0 = s * a.slice_vecs;
  const int64_t v1 = min(v0 + a.slice_vecs, row_vecs<kType>(row, a.vocab));
  // a short slice's tokens are fetched at once; a long one's only if some of them lie
  // in the bins to list, which its own histogram tells
  const bool early = !kHist || a.slice_vecs <= kThreads;
  Piece<kType> head(row, a.vocab, early ? v0 + threadIdx.x : INT32_MAX);
  uint64_t best;
  uint32_t least;
  row_ends(a, st, lds, best, least);
  const uint32_t top = (uint32_t)(best >> 32);
  Plan p{top, least, kBins, kBins, 0, 0, 0, 0, 0};
  if (top <= kKeyMinusInf) {
    if (s == 0 && threadIdx.x == 0) st.plan = p;
    return;
  }
  const Weigher wt(a, top, least, roots);
  __syncthreads();
  uint64_t sure = 0;
  if (kHist) {
    p = make_plan(a, st.hn, st.hw, wt, p, lds);
    const unsigned long long* own = slice_hist(a, r, s);
    int some = 0;
    for (int b = threadIdx.x; b <= min(p.hi, kBins - 1); b += kThreads) {
      if (b < p.lo)
        sure += own[b];
      else
        some |= own[b] != 0;
    }
    if (p.lo < kBins && __syncthreads_or(some)) {
      if (!early) head = Piece<kType>(row, a.vocab, v0 + threadIdx.x);
      each_token<kType>(head, row, a.vocab, v0, v1, [&](int64_t i, float x) {
        const float y = wt.value(x);
        const int b = wt.bin(y);
        if (b < p.lo || b > p.hi || wt.whole_of(y) == 0) return;
        const uint32_t at = atomicAdd(&st.listed, 1u);
        if (at < kListMax) st.list[at] = (uint64_t)order_key(x) << 32 | (uint32_t)~(uint32_t)i;
      });
    }
  } else {
    const auto add = [&](int64_t, float x) { sure += wt.kept_whole(x); };
    if (wt.inf)
      each_token<kType>(head, row, a.vocab, v0, v1, [&](int64_t i, float x) { add(i, wt.value(x)); });
    else
      each_token<kType>(head, row, a.vocab, v0, v1, add);
  }
  sure = block_reduce(sure, [](uint64_t x, uint64_t y) { return x + y; }, lds);
  if (threadIdx.x == 0) {
    st.sure[s] = sure;
    if (s == 0) st.plan = p;
  }
}

template <int kType>
void launch_slices_of(const SampleArgs& a, int rows, hipStream_t s) {
  const dim3 slices((unsigned)rows * a.slices), block(kThreads);
  hipLaunchKernelGGL((sample_max_kernel<kType, false>), slices, block, 0, s, a);
  if (!counts(a)) {
    hipLaunchKernelGGL((sample_gather_kernel<kType, false>), slices, block, 0, s, a);
    return;
  }
  if (a.top_k > 0 && a.top_k < a.vocab)
    hipLaunchKernelGGL((sample_hist_kernel<kType, true>), slices, block, 0, s, a);
  else
    hipLaunchKernelGGL((sample_hist_kernel<kType, false>), slices, block, 0, s, a);
  hipLaunchKernelGGL((sample_gather_kernel<kType, true>), slices, block, 0, s, a);
}

__global__ __launch_bounds__(kThreads) void sample_greedy_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kLdsWords];
  uint64_t best;
  uint32_t least;
  row_ends(a, row_state(a, blockIdx.x), lds, best, least);
  if (threadIdx.x != 0) return;
  const bool some = (uint32_t)(best >> 32) > kKeyMinusInf;
  a.token[blockIdx.x] = some ? (int64_t)(uint32_t)~(uint32_t)best : 0;
  if (a.prob) a.prob[blockIdx.x] = some ? 1.f : 0.f;
}

template <int kType, bool kHist>
__global__ __launch_bounds__(kDrawThreads) void sample_draw_kernel(SampleArgs a) {
  __shared__ uint64_t lds[lds_words<kDrawThreads>];
  __shared__ double roots[64];
  __shared__ uint64_t list[kHist ? kListMax : 1], spare[kHist ? kRankMax : 1];
  __shared__ unsigned long long sums[kMaxSlices];
  __shared__ uint32_t hn[kHist ? kRadixBins : 1];
  __shared__ unsigned long long hw[kHist ? kRadixBins : 1];
  const int r = blockIdx.x, tid = threadIdx.x;
  const char* row = row_of(a, r);
  const RowState& st = row_state(a, r);
  uint64_t* sh = lds + 2 * (kDrawThreads / 64);
  const Plan p = st.plan;
  if (p.top <= kKeyMinusInf) {  // nothing to choose from
    if (tid == 0) {
      a.token[r] = 0;
      if (a.prob) a.prob[r] = 0.f;
    }
    return;
  }
  const int n = kHist && p.lo < kBins ? (int)min(st.listed, (uint32_t)kListMax + 1) : 0;
  if (tid < a.slices) sums[tid] = st.sure[tid];
  if (kHist && n <= kListMax)
    for (int i = tid; i < n; i += kDrawThreads) list[i] = st.list[i];
  const double u = a.u[r];
  const Weigher wt(a, p.top, p.least, roots);
  __syncthreads();
  const Cut cut = cut_of_slices<kType, kHist>(a, p, row, wt, n, list, spare, sums, hn, hw, lds);
  constexpr int kSize = kType == DIP_F32 ? 4 : 2, kVec = 16 / kSize;
  const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15) / kSize;
  // the slice, then the token in it: running sums by index
  uint64_t total;
  const uint64_t mine = tid < a.slices ? sums[tid] : 0;
  const uint64_t before = block_exclusive<kDrawThreads>(mine, lds, total);
  uint64_t goal = goal_of(u, total);
  if (goal >= before && goal - before < mine) {
    sh[0] = (uint64_t)tid;
    sh[1] = before;
  }
  __syncthreads();
  const int64_t v0 = (int64_t)sh[0] * a.slice_vecs;
  const int64_t v1 = min(v0 + a.slice_vecs, row_vecs<kType>(row, a.vocab));
  goal -= sh[1];  // within the slice
  // a run of neighbouring pieces per thread; then the run that the draw falls in,
  // a token per thread
  const int64_t per = (v1 - v0 + kDrawThreads - 1) / kDrawThreads;
  const int64_t w0 = min(v0 + tid * per, v1), w1 = min(w0 + per, v1);
  uint64_t here = 0, in_slice;
  for (int64_t v = w0; v < w1; ++v)
    Piece<kType>(row, a.vocab, v).tokens(row, a.vocab, [&](int64_t i, float x) {
      const uint32_t k = order_key(x);
      if (cut.keeps(k, i)) here += wt.key_kept(k);
    });
  const uint64_t run = block_exclusive<kDrawThreads>(here, lds, in_slice);
  if (goal >= run && goal - run < here) {
    sh[0] = (uint64_t)w0;
    sh[1] = goal - run;
  }
  __syncthreads();
  const int64_t first = (int64_t)sh[0] * kVec - off;
  const int64_t end = min(first + per * kVec, a.vocab);
  goal = sh[1];
  for (int64_t i0 = max(first, (int64_t)0); i0 < end; i0 += kDrawThreads) {
    const int64_t i = i0 + tid;
    const uint32_t k = i < end ? order_key(load_logit<kType>(row, i)) : 0u;
    const uint64_t w = i < end && cut.keeps(k, i) ? wt.key_kept(k) : 0ull;
    uint64_t all;
    const uint64_t sum = block_exclusive<kDrawThreads>(w, lds, all);
    if (goal >= sum && goal - sum < w) {
      a.token[r] = i;
      if (a.prob) a.prob[r] = (float)(wt.key_scaled(k) / (double)total);
    }
    if (goal < all) break;
    goal -= all;
  }
}

// The whole draw of a row in one launch, a workgroup per row, its pieces held in
// registers from the first pass to the last.
template <int kType, int kN, bool kHist>
__global__ __launch_bounds__(kN) void sample_row_kernel(SampleArgs a) {
  __shared__ uint64_t lds[lds_words<kN>];
  __shared__ double roots[64];
  __shared__ uint64_t list[kHist ? kListMax : 1], spare[kHist ? kRankMax : 1];
  __shared__ uint32_t hn[kHist ? kBins : 1], listed;
  __shared__ unsigned long long hw[kHist ? kBins : 1];
  const int r = blockIdx.x, tid = threadIdx.x;
  const char* row = row_of(a, r);
  uint64_t* sh = lds + 2 * (kN / 64);
  const int64_t vecs = row_vecs<kType>(row, a.vocab);
  const int per = (int)((vecs + kN - 1) / kN);
  Piece<kType> p[kRowPieces];
#pragma unroll
  for (int j = 0; j < kRowPieces; ++j) p[j] = Piece<kType>(row, a.vocab, (int64_t)tid * per + j);
  const double u = a.u[r];
  auto mine = [&](auto f) {
#pragma unroll
    for (int j = 0; j < kRowPieces; ++j)
      if (j < per && (int64_t)tid * per + j < vecs) p[j].tokens(row, a.vocab, f);
  };
  if (kHist) {
    for (int b = tid; b < kBins; b += kN) hn[b] = 0, hw[b] = 0;
    if (tid == 0) listed = 0;
  }

  float most = -INFINITY, low = INFINITY;
  int64_t at = 0;
  mine([&](int64_t i, float x) {
    at = x > most ? i : at;
    most = fmaxf(most, x);
    low = fminf(low, x == -INFINITY ? INFINITY : x);
  });
  uint64_t best = (uint64_t)order_key(most) << 32 | (uint32_t)~(uint32_t)at;
  best = block_reduce<kN>(best, [](uint64_t x, uint64_t y) { return max(x, y); }, lds);
  const uint32_t top = (uint32_t)(best >> 32);
  if (top <= kKeyMinusInf || a.per_64th == 0) {  // nothing to choose from, or greedy
    if (tid == 0) {
      const bool some = top > kKeyMinusInf;
      a.token[r] = some ? (int64_t)(uint32_t)~(uint32_t)best : 0;
      if (a.prob) a.prob[r] = some ? 1.f : 0.f;
    }
    return;
  }
  const uint32_t least =
      block_reduce<kN>(order_key(low), [](uint32_t x, uint32_t y) { return min(x, y); },
                       reinterpret_cast<uint32_t*>(lds));
  const Weigher wt(a, top, least, roots);
  __syncthreads();

  const Plan plan{top, least, kBins, kBins, 0, 0, 0, 0, 0};
  const Cut cut = kHist ? cut_of_row<kType, kN>(a, plan, row, wt, mine, list, spare, &listed, hn,
                                                hw, lds)
                        : Cut{0u, a.vocab};

  // running sums by index: threads, pieces and tokens come in it
  auto weight = [&](int64_t i, float x) {
    if (kHist) {
      const uint32_t k = order_key(x);
      if (!cut.keeps(k, i)) return (uint64_t)0;
    }
    return (uint64_t)wt.kept_whole(wt.value(x));
  };
  uint64_t here = 0, total, in_run;
  mine([&](int64_t i, float x) { here += weight(i, x); });
  uint64_t run = block_exclusive<kN>(here, lds, total);
  const uint64_t goal = goal_of(u, total);
  if (goal >= run && goal - run < here) {
    sh[0] = (uint64_t)tid;
    sh[1] = goal - run;
  }
  __syncthreads();
  // the run that the draw falls in, a token per thread
  constexpr int kVec = Piece<kType>::kVec;
  const int64_t first = (int64_t)sh[0] * per * kVec -
                        (int)(reinterpret_cast<uintptr_t>(row) & 15) / Piece<kType>::kSize;
  const int64_t i = first + tid;
  const bool on = tid < per * kVec && i >= 0 && i < a.vocab;
  const uint64_t left = sh[1];
  const float x = on ? load_logit<kType>(row, i) : -INFINITY;
  const uint64_t w = on ? weight(i, x) : 0;
  const uint64_t before = block_exclusive<kN>(w, lds, in_run);
  if (left >= before && left - before < w) {
    a.token[r] = i;
    if (a.prob) a.prob[r] = (float)(wt.scaled(wt.value(x)) / (double)total);
  }
}

template <int kType, int kN>
int launch_row(const SampleArgs& a, int rows, hipStream_t s) {
  if (counts(a))
    hipLaunchKernelGGL((sample_row_kernel<kType, kN, true>), dim3(rows), dim3(kN), 0, s, a);
  else
    hipLaunchKernelGGL((sample_row_kernel<kType, kN, false>), dim3(rows), dim3(kN), 0, s, a);
  return hip_status(hipGetLastError());
}

template <int kType>
int launch_sample(const SampleArgs& a, int rows, int64_t vecs, hipStream_t s) {
  const int threads = row_threads(a, rows, vecs);
  if (threads == kThreads) return launch_row<kType, kThreads>(a, rows, s);
  if (threads) return launch_row<kType, 1024>(a, rows, s);
  const dim3 each(rows), draw(kDrawThreads);
  if (a.per_64th == 0) {
    launch_slices_max(kType, a, rows, s);
    hipLaunchKernelGGL(sample_greedy_kernel, each, dim3(kThreads), 0, s, a);
    return hip_status(hipGetLastError());
  }
  launch_slices(kType, a, rows, s);
  if (counts(a))
    hipLaunchKernelGGL((sample_draw_kernel<kType, true>), each, draw, 0, s, a);
  else
    hipLaunchKernelGGL((sample_draw_kernel<kType, false>), each, draw, 0, s, a);
  return hip_status(hipGetLastError());
}

}  // namespace

void launch_slices(int dtype, const SampleArgs& a, int rows, hipStream_t s) {
  if (dtype == DIP_F32) return launch_slices_of<DIP_F32>(a, rows, s);
  if (dtype == DIP_F16) return launch_slices_of<DIP_F16>(a, rows, s);
  launch_slices_of<DIP_BF16>(a, rows, s);
}

void launch_slices_max(int dtype, const SampleArgs& a, int rows, hipStream_t s) {
  const dim3 slices((unsigned)rows * a.slices), block(kThreads);
  if (dtype == DIP_F32)
    hipLaunchKernelGGL((sample_max_kernel<DIP_F32, true>), slices, block, 0, s, a);
  else if (dtype == DIP_F16)
    hipLaunchKernelGGL((sample_max_kernel<DIP_F16, true>), slices, block, 0, s, a);
  else
    hipLaunchKernelGGL((sample_max_kernel<DIP_BF16, true>), slices, block, 0, s, a);
}

}  // namespace dip

using namespace dip;

// For fp32 logits, which take the most slices.
extern "C" size_t dip_sample_workspace_size(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || max_vecs(vocab, 4) <= kOneLaunch) return 0;
  return (size_t)rows * (sizeof(RowState) +
                         (size_t)slices_for(rows, max_vecs(vocab, 4)) * kBins * sizeof(uint64_t));
}

extern "C" int dip_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                          int64_t row_stride, const float* u, double temperature, int64_t top_k,
                          double top_p, double min_p, int64_t* token, float* prob,
                          void* workspace, size_t ws_bytes, void* stream) {
  if (int st = check_sampling(dtype, vocab, temperature, top_k, top_p, min_p)) return st;
  if (rows < 0 || !launch_fits(rows, 1024) || row_stride < 0) return DIP_ERR_SHAPE;
  if (rows == 0) return DIP_OK;
  if (!logits || !u || !token) return DIP_ERR_NULL;
  const size_t need = dip_sample_workspace_size(rows, vocab);
  if (need && (!workspace || ws_bytes < need)) return DIP_ERR_WORKSPACE;
  const int size = dtype == DIP_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size || (need && !aligned16(workspace)))
    return DIP_ERR_ALIGN;
  const int64_t vecs = max_vecs(vocab, size);
  SampleArgs a = sample_args(rows, vocab, size, temperature, top_k, top_p, min_p);
  a.logits = logits;
  a.row_bytes = row_stride * size;
  a.u = u;
  a.rows = static_cast<char*>(workspace);
  a.token = token;
  a.prob = prob;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DIP_F32) return launch_sample<DIP_F32>(a, (int)rows, vecs, s);
  if (dtype == DIP_F16) return launch_sample<DIP_F16>(a, (int)rows, vecs, s);
  return launch_sample<DIP_BF16>(a, (int)rows, vecs, s);
}
