// dip_verify.hip — verification of drafted tokens: which of a sequence's drafts the
// target's distribution takes over, and the token that follows them.
//
// With p_t the target's probabilities behind t drafted tokens (those that dip_sample
// draws with, filters included), q_t the ones that the drafted token x_t was drawn with
// (of the drafting model's logits by the same filters; without them 1 at x_t and 0
// elsewhere) and numbers u_0 .. u_n in [0, 1):
//   x_t is accepted while u_t q_t(x_t) < p_t(x_t);
//   at the first t that is not, the token is drawn from max(p_t - q_t, 0), by index and
//   with u_n; behind n accepted ones from p_n.
// The tokens are then distributed as if each had been drawn from p.
//
// A row's weights are dip_sample's whole numbers, exact in sum, so the share of a token
// is a quotient of two of them.  What is left of p where q is taken away is held in whole
// numbers of 2^-51.
//
// Launches: the border and the sum of the weights that the filters keep, for every row
// at once (in one launch where rows fit a workgroup's registers, else in slices, as
// dip_sample's); then per sequence the rows of the drafts decide which row the token is
// drawn from, whose remainder is added up in slices; then the token.  Greedy (temperature
// 0, top-k 1): the rows' largest logits, and a choice among them.
#include "dip_sample.h"

namespace dip {
namespace {

// What the filters keep of a row.
struct Border {
  uint32_t top, least;  // order_keys of the largest logit and the smallest above -inf
  Cut cut;
  uint64_t total;  // of the kept weights; 0: nothing to choose from
  uint64_t drafted;  // weight of the row's drafted token
};

struct VerifyArgs {
  SampleArgs s;  // rows: the target's, a sequence's tokens + 1 together, then the draft's
  const int64_t* drafted;  // [seqs, tokens]
  int seqs, tokens, draft;  // draft: with its logits
  Border* borders;          // [rows]
  uint64_t* sums;  // [seqs, slices, 2]: of what is left of a slice, and of its own weights
  int slices;
  int64_t slice_vecs;
  int64_t* out;  // [seqs, tokens + 1]
  int64_t* accepted;
};

// The drafted token of a row, -1 if there is none.
DIP_DEV int64_t token_of(const VerifyArgs& a, int r) {
  const int target = a.seqs * (a.tokens + 1);
  int64_t x = -1;
  if (r >= target)
    x = a.drafted[r - target];
  else if (r % (a.tokens + 1) < a.tokens)
    x = a.drafted[(int64_t)(r / (a.tokens + 1)) * a.tokens + r % (a.tokens + 1)];
  return x >= 0 && x < a.s.vocab ? x : -1;
}

template <int kType>
DIP_DEV uint64_t weight_of(const VerifyArgs& a, int r, const char* row, const Weigher& wt,
                           const Cut& cut) {
  const int64_t x = token_of(a, r);
  if (x < 0) return 0;
  const uint32_t k = order_key(load_logit<kType>(row, x));
  return cut.keeps(k, x) ? wt.key_kept(k) : 0ull;
}

template <int kType, bool kHist>
__global__ __launch_bounds__(kDrawThreads) void verify_slices_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[lds_words<kDrawThreads>];
  __shared__ double roots[64];
  __shared__ uint64_t list[kHist ? kListMax : 1], spare[kHist ? kRankMax : 1];
  __shared__ unsigned long long sums[kMaxSlices];
  __shared__ uint32_t hn[kHist ? kRadixBins : 1];
  __shared__ unsigned long long hw[kHist ? kRadixBins : 1];
  const SampleArgs& a = v.s;
  const int r = blockIdx.x, tid = threadIdx.x;
  const char* row = row_of(a, r);
  const RowState& st = row_state(a, r);
  const Plan p = st.plan;
  if (p.top <= kKeyMinusInf) {
    if (tid == 0) v.borders[r] = Border{p.top, p.least, Cut{0u, 0}, 0, 0};
    return;
  }
  const int n = kHist && p.lo < kBins ? (int)min(st.listed, (uint32_t)kListMax + 1) : 0;
  if (tid < a.slices) sums[tid] = st.sure[tid];
  if (kHist && n <= kListMax)
    for (int i = tid; i < n; i += kDrawThreads) list[i] = st.list[i];
  const Weigher wt(a, p.top, p.least, roots);
  __syncthreads();
  const Cut cut = cut_of_slices<kType, kHist>(a, p, row, wt, n, list, spare, sums, hn, hw, lds);
  const uint64_t total = block_reduce<kDrawThreads>(
      tid < a.slices ? (uint64_t)sums[tid] : 0, [](uint64_t x, uint64_t y) { return x + y; }, lds);
  if (tid == 0)
    v.borders[r] = Border{p.top, p.least, cut, total, weight_of<kType>(v, r, row, wt, cut)};
}

template <int kType, int kN, bool kHist>
__global__ __launch_bounds__(kN) void verify_row_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[lds_words<kN>];
  __shared__ double roots[64];
  __shared__ uint64_t list[kHist ? kListMax : 1], spare[kHist ? kRankMax : 1];
  __shared__ uint32_t hn[kHist ? kBins : 1], listed;
  __shared__ unsigned long long hw[kHist ? kBins : 1];
  const SampleArgs& a = v.s;
  const int r = blockIdx.x, tid = threadIdx.x;
  const char* row = row_of(a, r);
  const int64_t vecs = row_vecs<kType>(row, a.vocab);
  const int per = (int)((vecs + kN - 1) / kN);
  Piece<kType> p[kRowPieces];
#pragma unroll
  for (int j = 0; j < kRowPieces; ++j) p[j] = Piece<kType>(row, a.vocab, (int64_t)tid * per + j);
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
  mine([&](int64_t, float x) {
    most = fmaxf(most, x);
    low = fminf(low, x == -INFINITY ? INFINITY : x);
  });
  const uint32_t top = block_reduce<kN>(order_key(most), [](uint32_t x, uint32_t y) { return max(x, y); },
                                        reinterpret_cast<uint32_t*>(lds));
  const uint32_t least = block_reduce<kN>(order_key(low), [](uint32_t x, uint32_t y) { return min(x, y); },
                                          reinterpret_cast<uint32_t*>(lds));
  if (top <= kKeyMinusInf) {
    if (tid == 0) v.borders[r] = Border{top, least, Cut{0u, 0}, 0, 0};
    return;
  }
  if (a.per_64th == 0) {  // greedy: the first of the largest
    uint32_t at = 0xFFFFFFFFu;
    mine([&](int64_t i, float x) {
      if (order_key(x) == top) at = min(at, (uint32_t)i);
    });
    at = block_reduce<kN>(at, [](uint32_t x, uint32_t y) { return min(x, y); },
                          reinterpret_cast<uint32_t*>(lds));
    if (tid == 0) v.borders[r] = Border{top, least, Cut{top, (int64_t)at}, 1, 0};
    return;
  }
  const Weigher wt(a, top, least, roots);
  __syncthreads();
  const Plan plan{top, least, kBins, kBins, 0, 0, 0, 0, 0};
  const Cut cut = kHist ? cut_of_row<kType, kN>(a, plan, row, wt, mine, list, spare, &listed, hn,
                                                hw, lds)
                        : Cut{0u, a.vocab};
  uint64_t here = 0;
  mine([&](int64_t i, float x) {
    if (!kHist || cut.keeps(order_key(x), i)) here += wt.kept_whole(wt.value(x));
  });
  const uint64_t total =
      block_reduce<kN>(here, [](uint64_t x, uint64_t y) { return x + y; }, lds);
  if (tid == 0) v.borders[r] = Border{top, least, cut, total, weight_of<kType>(v, r, row, wt, cut)};
}

// How many of a sequence's drafts are accepted: the first that `refused(t)` holds for.
template <int kN, typename F>
DIP_DEV int accepted_of(const VerifyArgs& a, F refused, uint32_t* lds) {
  uint32_t first = (uint32_t)a.tokens;
  for (int t = threadIdx.x; t < a.tokens; t += kN)
    if (refused(t)) {
      first = (uint32_t)t;
      break;
    }
  return (int)block_reduce<kN>(first, [](uint32_t x, uint32_t y) { return min(x, y); }, lds);
}

// The row that a sequence's token is drawn from, and what of it.
template <int kType>
struct Rest {
  int accepted;
  const char* row;
  const char* draft;  // the draft's row; null: its token alone is taken away
  int64_t x;          // the draft's token; -1: nothing is taken away
  Border p, q;
  double p_by, q_by;  // shares from weights, in whole numbers
};

template <int kType, int kN>
DIP_DEV Rest<kType> rest_of(const VerifyArgs& v, int seq, uint32_t* lds) {
  const int target = v.seqs * (v.tokens + 1), first = seq * (v.tokens + 1);
  const Border* d = v.borders + target + (int64_t)seq * v.tokens;
  const float* u = v.s.u + first;
  Rest<kType> r;
  r.accepted = accepted_of<kN>(
      v,
      [&](int t) {
        const Border& b = v.borders[first + t];
        if (token_of(v, first + t) < 0 || b.total == 0) return true;
        const double share = (double)b.drafted / (double)b.total;
        const double drawn = !v.draft      ? 1.0
                             : d[t].total ? (double)d[t].drafted / (double)d[t].total
                                          : 0.0;
        return !((double)u[t] * drawn < share);
      },
      lds);
  r.row = row_of(v.s, first + r.accepted);
  r.p = v.borders[first + r.accepted];
  r.x = token_of(v, first + r.accepted);  // (-1 behind the last)
  r.draft = nullptr;
  r.p_by = r.q_by = 0.0;
  if (r.x >= 0 && v.draft && r.p.total) {
    r.q = d[r.accepted];
    r.draft = row_of(v.s, target + seq * v.tokens + r.accepted);
    r.p_by = 0x1p51 / (double)r.p.total;
    r.q_by = r.q.total ? 0x1p51 / (double)r.q.total : 0.0;
  }
  return r;
}

// What the token is drawn by: a token's own weight, and what is left of it where the
// draft's share is taken away.
template <int kType>
struct Weights {
  const Rest<kType>& r;
  Weigher p, q;

  // A barrier must follow before their use.
  DIP_DEV Weights(const SampleArgs& a, const Rest<kType>& rest, double* roots)
      : r(rest),
        p(a, rest.p.top, rest.p.least, roots),
        q(a, rest.draft ? rest.q.top : rest.p.top, rest.draft ? rest.q.least : rest.p.least,
          roots) {}
  DIP_DEV uint64_t own(int64_t i, float x) const {
    const uint32_t k = order_key(x);
    return r.p.cut.keeps(k, i) ? p.key_kept(k) : 0ull;
  }
  DIP_DEV uint64_t left(int64_t i, uint64_t w) const {
    if (!r.draft) return i == r.x ? 0 : w;
    if (w == 0) return 0;
    const uint32_t k = order_key(load_logit<kType>(r.draft, i));
    const uint64_t o = r.q.cut.keeps(k, i) ? q.key_kept(k) : 0ull;
    const double d = (double)w * r.p_by - (double)o * r.q_by;
    return d > 0.0 ? Weigher::whole(d) : 0ull;
  }
};

template <int kType>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[kLdsWords];
  __shared__ double roots[64];
  const int seq = blockIdx.x / v.slices, s = blockIdx.x % v.slices;
  const Rest<kType> rest = rest_of<kType, kThreads>(v, seq, reinterpret_cast<uint32_t*>(lds));
  uint64_t left = 0, own = 0;
  if (rest.p.total) {
    const Weights<kType> w(v.s, rest, roots);
    __syncthreads();
    each_token<kType>(rest.row, v.s.vocab, s * v.slice_vecs,
                      min((s + 1) * v.slice_vecs, row_vecs<kType>(rest.row, v.s.vocab)),
                      [&](int64_t i, float x) {
                        const uint64_t o = w.own(i, x);
                        own += o;
                        left += w.left(i, o);
                      });
  }
  const auto add = [](uint64_t x, uint64_t y) { return x + y; };
  left = block_reduce(left, add, lds);
  own = block_reduce(own, add, lds);
  if (threadIdx.x == 0) {
    v.sums[2 * (int64_t)blockIdx.x] = left;
    v.sums[2 * (int64_t)blockIdx.x + 1] = own;
  }
}

// The tokens but the one that is drawn.
template <int kN>
DIP_DEV void put_drafts(const VerifyArgs& v, int seq, int accepted) {
  for (int t = threadIdx.x; t <= v.tokens; t += kN)
    if (t != accepted)
      v.out[(int64_t)seq * (v.tokens + 1) + t] =
          t < accepted ? v.drafted[(int64_t)seq * v.tokens + t] : -1;
  if (threadIdx.x == 0) v.accepted[seq] = accepted;
}

template <int kType>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[lds_words<kDrawThreads>];
  __shared__ double roots[64];
  const int seq = blockIdx.x, tid = threadIdx.x;
  const int64_t vocab = v.s.vocab;
  uint64_t* sh = lds + 2 * (kDrawThreads / 64);
  const Rest<kType> rest = rest_of<kType, kDrawThreads>(v, seq, reinterpret_cast<uint32_t*>(lds));
  put_drafts<kDrawThreads>(v, seq, rest.accepted);
  int64_t* token = v.out + (int64_t)seq * (v.tokens + 1) + rest.accepted;
  if (rest.p.total == 0) {  // nothing to choose from
    if (tid == 0) *token = 0;
    return;
  }
  const Weights<kType> w(v.s, rest, roots);
  if (tid < 2) sh[tid] = 0;
  const uint64_t* sums = v.sums + 2 * (int64_t)seq * v.slices;
  const uint64_t slice_left = tid < v.slices ? sums[2 * tid] : 0;
  const uint64_t slice_own = tid < v.slices ? sums[2 * tid + 1] : 0;
  uint64_t total;
  uint64_t mine = slice_left, before = block_exclusive<kDrawThreads>(mine, lds, total);
  // (nothing left: numbers u outside [0, 1), or p and q the same)
  const bool own = total == 0;
  if (own) {
    mine = slice_own;
    before = block_exclusive<kDrawThreads>(mine, lds, total);
  }
  uint64_t goal = goal_of(v.s.u[(int64_t)seq * (v.tokens + 1) + v.tokens], total);
  if (goal >= before && goal - before < mine) {
    sh[0] = (uint64_t)tid;
    sh[1] = before;
  }
  __syncthreads();
  auto weight = [&](int64_t i, float x) {
    const uint64_t o = w.own(i, x);
    return own ? o : w.left(i, o);
  };
  // a run of neighbouring pieces of the slice per thread; then the run that the draw
  // falls in, a token per thread
  constexpr int kSize = kType == DIP_F32 ? 4 : 2, kVec = 16 / kSize;
  const int off = (int)(reinterpret_cast<uintptr_t>(rest.row) & 15) / kSize;
  const int64_t v0 = (int64_t)sh[0] * v.slice_vecs;
  const int64_t v1 = min(v0 + v.slice_vecs, row_vecs<kType>(rest.row, vocab));
  goal -= sh[1];
  const int64_t per = (v1 - v0 + kDrawThreads - 1) / kDrawThreads;
  const int64_t w0 = min(v0 + tid * per, v1), w1 = min(w0 + per, v1);
  uint64_t here = 0, all;
  for (int64_t j = w0; j < w1; ++j)
    Piece<kType>(rest.row, vocab, j).tokens(rest.row, vocab, [&](int64_t i, float x) {
      here += weight(i, x);
    });
  const uint64_t run = block_exclusive<kDrawThreads>(here, lds, all);
  if (goal >= run && goal - run < here) {
    sh[0] = (uint64_t)w0;
    sh[1] = goal - run;
  }
  __syncthreads();
  const int64_t first = (int64_t)sh[0] * kVec - off, end = min(first + per * kVec, vocab);
  goal = sh[1];
  for (int64_t i0 = max(first, (int64_t)0); i0 < end; i0 += kDrawThreads) {
    const int64_t i = i0 + tid;
    const uint64_t o = i < end ? weight(i, load_logit<kType>(rest.row, i)) : 0ull;
    const uint64_t sum = block_exclusive<kDrawThreads>(o, lds, all);
    if (goal >= sum && goal - sum < o) *token = i;
    if (goal < all) break;
    goal -= all;
  }
}

// kSlices: the rows' largest logits are still in slices.
template <bool kSlices>
__global__ __launch_bounds__(kThreads) void verify_greedy_kernel(VerifyArgs v) {
  __shared__ uint32_t lds[kThreads / 64];
  const int seq = blockIdx.x, first = seq * (v.tokens + 1);
  if (kSlices) {
    for (int t = threadIdx.x >> 6; t <= v.tokens; t += kThreads / 64) {
      const RowState& st = row_state(v.s, first + t);
      uint64_t best = 0;
      for (int s = threadIdx.x & 63; s < v.s.slices; s += 64) best = max(best, st.best[s]);
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) best = max(best, (uint64_t)__shfl_xor(best, m, 64));
      const bool some = (uint32_t)(best >> 32) > kKeyMinusInf;
      if ((threadIdx.x & 63) == 0)
        v.borders[first + t] =
            Border{(uint32_t)(best >> 32), 0u, Cut{0u, some ? (int64_t)(uint32_t)~(uint32_t)best : 0},
                   some, 0};
    }
    __syncthreads();
  }
  const int accepted = accepted_of<kThreads>(
      v,
      [&](int t) {
        const Border& b = v.borders[first + t];
        return b.total == 0 || b.cut.index != token_of(v, first + t);
      },
      lds);
  put_drafts<kThreads>(v, seq, accepted);
  if (threadIdx.x == 0) v.out[first + accepted] = v.borders[first + accepted].cut.index;
}

template <int kType, int kN>
void launch_rows(const VerifyArgs& v, int rows, hipStream_t s) {
  if (counts(v.s))
    hipLaunchKernelGGL((verify_row_kernel<kType, kN, true>), dim3(rows), dim3(kN), 0, s, v);
  else
    hipLaunchKernelGGL((verify_row_kernel<kType, kN, false>), dim3(rows), dim3(kN), 0, s, v);
}

template <int kType>
int launch_verify(const VerifyArgs& v, int rows, int64_t vecs, hipStream_t s) {
  const bool greedy = v.s.per_64th == 0;
  const int threads = row_threads(v.s, rows, vecs);
  if (threads == kThreads) {
    launch_rows<kType, kThreads>(v, rows, s);
  } else if (threads) {
    launch_rows<kType, 1024>(v, rows, s);
  } else if (greedy) {
    hipLaunchKernelGGL((sample_max_kernel<kType, true>), dim3((unsigned)rows * v.s.slices),
                       dim3(kThreads), 0, s, v.s);
  } else {
    launch_slices<kType>(v.s, rows, s);
    if (counts(v.s))
      hipLaunchKernelGGL((verify_slices_kernel<kType, true>), dim3(rows), dim3(kDrawThreads), 0,
                         s, v);
    else
      hipLaunchKernelGGL((verify_slices_kernel<kType, false>), dim3(rows), dim3(kDrawThreads), 0,
                         s, v);
  }
  if (greedy) {
    if (threads)
      hipLaunchKernelGGL(verify_greedy_kernel<false>, dim3(v.seqs), dim3(kThreads), 0, s, v);
    else
      hipLaunchKernelGGL(verify_greedy_kernel<true>, dim3(v.seqs), dim3(kThreads), 0, s, v);
    return hip_status(hipGetLastError());
  }
  hipLaunchKernelGGL((verify_rest_kernel<kType>), dim3((unsigned)v.seqs * v.slices),
                     dim3(kThreads), 0, s, v);
  hipLaunchKernelGGL((verify_draw_kernel<kType>), dim3(v.seqs), dim3(kDrawThreads), 0, s, v);
  return hip_status(hipGetLastError());
}

inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }
inline int64_t rows_of(int64_t seqs, int64_t tokens, bool draft) {
  return seqs * (tokens + 1 + (draft ? tokens : 0));
}
// Sequences, drafts and logits that one call takes.
inline bool sizes_ok(int64_t seqs, int64_t tokens, int64_t vocab) {
  return seqs >= 0 && seqs <= (1 << 22) && tokens >= 0 && tokens <= (1 << 20) && vocab > 0 &&
         vocab <= (1 << 30) && launch_fits(seqs * (2 * tokens + 1), 1024);
}

}  // namespace
}  // namespace dip

using namespace dip;

// For fp32 logits, which take the most slices.
extern "C" size_t dip_verify_workspace_size(int64_t seqs, int64_t tokens, int64_t vocab,
                                            int draft_logits) {
  if (!sizes_ok(seqs, tokens, vocab) || seqs == 0) return 0;
  const int64_t rows = rows_of(seqs, tokens, draft_logits != 0), vecs = max_vecs(vocab, 4);
  size_t n = up16(rows * sizeof(Border)) + (size_t)seqs * slices_for(seqs, vecs) * 16;
  if (vecs > kOneLaunch)
    n += (size_t)rows *
         (sizeof(RowState) + (size_t)slices_for(rows, vecs) * kBins * sizeof(uint64_t));
  return n;
}

extern "C" int dip_verify(const void* logits, int dtype, int64_t seqs, int64_t tokens,
                          int64_t vocab, int64_t row_stride, const int64_t* drafted,
                          const void* draft_logits, int64_t draft_row_stride, const float* u,
                          double temperature, int64_t top_k, double top_p, double min_p,
                          int64_t* token, int64_t* accepted, void* workspace, size_t ws_bytes,
                          void* stream) {
  if (int st = check_sampling(dtype, vocab, temperature, top_k, top_p, min_p)) return st;
  if (!sizes_ok(seqs, tokens, vocab) || row_stride < 0 || (draft_logits && draft_row_stride < 0))
    return DIP_ERR_SHAPE;
  if (seqs == 0) return DIP_OK;
  if (!logits || !u || !token || !accepted || (tokens > 0 && !drafted)) return DIP_ERR_NULL;
  const int size = dtype == DIP_F32 ? 4 : 2;
  SampleArgs s = sample_args(seqs * (tokens + 1), vocab, size, temperature, top_k, top_p, min_p);
  const bool draft = draft_logits && tokens > 0 && s.per_64th > 0;  // (greedy asks for none)
  const int64_t rows = rows_of(seqs, tokens, draft), vecs = max_vecs(vocab, size);
  const size_t need = dip_verify_workspace_size(seqs, tokens, vocab, draft);
  if (!workspace || ws_bytes < need) return DIP_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(logits) % size || !aligned16(workspace) ||
      (draft && reinterpret_cast<uintptr_t>(draft_logits) % size))
    return DIP_ERR_ALIGN;
  s = sample_args(rows, vocab, size, temperature, top_k, top_p, min_p);
  s.rows1 = (int)(seqs * (tokens + 1));
  s.logits = logits;
  s.row_bytes = row_stride * size;
  s.more = draft_logits;
  s.more_bytes = draft_row_stride * size;
  s.u = u;
  VerifyArgs v{};
  v.drafted = drafted;
  v.seqs = (int)seqs;
  v.tokens = (int)tokens;
  v.draft = draft;
  v.slices = slices_for(seqs, vecs);
  v.slice_vecs = (vecs + v.slices - 1) / v.slices;
  char* w = static_cast<char*>(workspace);
  v.borders = reinterpret_cast<Border*>(w);
  w += up16(rows * sizeof(Border));
  v.sums = reinterpret_cast<uint64_t*>(w);
  s.rows = w + (size_t)seqs * v.slices * 16;
  v.s = s;
  v.out = token;
  v.accepted = accepted;
  if (!launch_fits(rows * s.slices, kThreads) || !launch_fits(seqs * v.slices, kThreads))
    return DIP_ERR_SHAPE;
  hipStream_t q = (hipStream_t)stream;
  if (dtype == DIP_F32) return launch_verify<DIP_F32>(v, (int)rows, vecs, q);
  if (dtype == DIP_F16) return launch_verify<DIP_F16>(v, (int)rows, vecs, q);
  return launch_verify<DIP_BF16>(v, (int)rows, vecs, q);
}
