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
// A row's weights are dip_sample's whole numbers, so a token's share is a quotient: its
// weight over the row's sum.  With filters the sum is exact, in any order.  Without any it
// is put together of the slices' sums, each of weights by the slice's own largest logit,
// in 64-bit floating point: off by 2^-30 of itself as a weight and a slice's factor are
// (4e-10 each), and by what the weights' rounding to whole numbers does, which is finer
// against a smaller largest logit (half a unit of 2^-43 for each of 2^19 tokens, the most
// that go this way: 2^-25).  By that much the sum may be another one where the call's
// number of rows cuts them otherwise, and a draft whose u q lies that near to p taken or
// refused.  (Exact here too would take the largest logit of the whole row first, a launch
// and a reading of the rows more.)  What is left of p where q is taken away is held in
// whole numbers of 2^-51.
//
// Launches: the border and the sum of the weights that the filters keep, for every row
// at once (in one launch where rows fit a workgroup's registers, else in slices, as
// dip_sample's); then per sequence the rows of the drafts decide which row the token is
// drawn from, whose remainder is added up in slices; then the token.  Greedy (temperature
// 0, top-k 1): the rows' largest logits, and a choice among them.  With top-k up to 64
// each slice of a row gives its k largest tokens, of them the row's k largest are found and
// weighed, and everything else is a matter of lists of k: three launches, each logit read
// once.  Without filters a slice's weights are added up by its own largest logit and the
// slices' sums taken to the row's by the two launches that need them: three, too.
//
// 5 rows of 151936 bf16 logits, top-k 20 and top-p: 6, 8 and 4.5 us, all waits in a row
// (by the histogram's launches 39 in all).  16 sequences of 5 drafts over 151936 fp32 with
// the draft's logits, top-p and min-p (107 MB): 18 for max, the memory; 31 for hist, the
// weights' instructions; 21 for gather, which reads the rows again for their borders'
// tokens; 5, 10 and 8 for the rest.  50 of 3 over 32003 bf16, no filter: 16 for the sums, 15
// and 10 (in one workgroup a row 27, 12 and 12, as 350 of them go unevenly onto 256 CUs).
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

constexpr int kSumPieces = 4;  // of a thread
constexpr int kTopMost = 64;
struct TopRow {  // the k largest tokens of a row: what the filters keep of their weights
  uint64_t weight[kTopMost];
  uint32_t index[kTopMost];
};

struct Part {  // of a slice, by its own largest logit
  uint32_t top;
  uint64_t sum;
};

struct Decided {  // of a sequence, by the launch that adds up what is left
  Border p, q;
  int64_t accepted;
};

struct VerifyArgs {
  SampleArgs s;  // rows: the target's, a sequence's tokens + 1 together, then the draft's
  const int64_t* drafted;  // [seqs, tokens]
  int seqs, tokens, draft;  // draft: with its logits
  Border* borders;          // [rows]
  uint64_t* sums;  // [seqs, slices, 2]: of what is left of a slice, and of its own weights
  Decided* decided;  // [seqs]
  int slices;
  int64_t slice_vecs;
  int64_t* out;  // [seqs, tokens + 1]
  int64_t* accepted;
  Part* parts;     // no filters: [rows, s.slices]
  uint64_t* best;  // top-k up to kTopMost: [rows, slices, k] order_key << 32 | ~index
  TopRow* tops;    // [rows]
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

// p: the row's border behind the accepted drafts, q its draft's, if there is `some`.
template <int kType>
DIP_DEV Rest<kType> rest_at(const VerifyArgs& v, int seq, int accepted, const Border& p, bool some,
                            const Border& q) {
  const int r = seq * (v.tokens + 1) + accepted;
  Rest<kType> rest;
  rest.accepted = accepted;
  rest.row = row_of(v.s, r);
  rest.p = p;
  rest.x = token_of(v, r);  // (-1 behind the last)
  rest.draft = nullptr;
  rest.p_by = rest.q_by = 0.0;
  rest.q = q;
  if (rest.x >= 0 && some && p.total) {
    rest.draft = row_of(v.s, v.seqs * (v.tokens + 1) + seq * v.tokens + accepted);
    rest.p_by = 0x1p51 / (double)p.total;
    rest.q_by = q.total ? 0x1p51 / (double)q.total : 0.0;
  }
  return rest;
}

// Whether a draft is refused, of what its rows say.
DIP_DEV bool refuses(const Border& p, bool some, const Border& q, float u) {
  if (p.total == 0) return true;
  const double share = (double)p.drafted / (double)p.total;
  const double drawn = !some ? 1.0 : q.total ? (double)q.drafted / (double)q.total : 0.0;
  return !((double)u * drawn < share);
}

template <int kType, int kN>
DIP_DEV Rest<kType> rest_of(const VerifyArgs& v, int seq, uint32_t* lds) {
  const int first = seq * (v.tokens + 1);
  // (without the draft's logits: not read)
  const Border* d = v.borders + (v.draft ? v.seqs * (v.tokens + 1) + (int64_t)seq * v.tokens : 0);
  const int accepted = accepted_of<kN>(
      v,
      [&](int t) {
        return token_of(v, first + t) < 0 ||
               refuses(v.borders[first + t], v.draft, d[v.draft ? t : 0], v.s.u[first + t]);
      },
      lds);
  const bool some = v.draft && accepted < v.tokens;
  return rest_at<kType>(v, seq, accepted, v.borders[first + accepted], some,
                        d[some ? accepted : 0]);
}

// A row's border from its slices' sums, by a wave; `roots` are there.
template <int kType>
DIP_DEV Border border_of(const VerifyArgs& v, int r, const double* roots) {
  const int l = threadIdx.x & 63;
  const Part part = l < v.s.slices ? v.parts[(int64_t)r * v.s.slices + l] : Part{0u, 0};
  const int64_t x = token_of(v, r);
  const uint32_t key = x < 0 ? 0u : order_key(load_logit<kType>(row_of(v.s, r), x));
  uint32_t top = part.top;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor(top, m, 64));
  if (top <= kKeyMinusInf) return Border{top, top, Cut{0u, v.s.vocab}, 0, 0};
  const Weigher wt(v.s, roots, top, top);
  // what a weight by the slice's largest is by the row's
  double sum = part.top > kKeyMinusInf
                   ? (double)part.sum * (wt.key_scaled(part.top) / (double)(1ull << v.s.shift))
                   : 0.0;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m, 64);
  return Border{top, top, Cut{0u, v.s.vocab}, (uint64_t)(sum + 0.5),
                x < 0 ? 0 : wt.key_whole(key)};
}

// rest_of where rows have slices' sums: a wave per draft, and for the row behind the last.
// The first kKept drafts' borders are kept for the one that matters.
template <int kType, int kN>
DIP_DEV Rest<kType> rest_of_parts(const VerifyArgs& v, int seq, const double* roots,
                                  uint32_t* lds) {
  constexpr int kKept = 8;
  __shared__ Border kept[kKept][2];
  const int first = seq * (v.tokens + 1), draft = v.seqs * (v.tokens + 1) + seq * v.tokens;
  uint32_t accepted = (uint32_t)v.tokens;
  auto borders = [&](int t, Border& p, Border& q) {
    p = border_of<kType>(v, first + t, roots);
    q = p;
    if (v.draft && t < v.tokens) q = border_of<kType>(v, draft + t, roots);
  };
  for (int t = threadIdx.x >> 6; t <= v.tokens; t += kN / 64) {
    Border p, q;
    borders(t, p, q);
    if (t < kKept && (threadIdx.x & 63) == 0) kept[t][0] = p, kept[t][1] = q;
    if (t == v.tokens || (token_of(v, first + t) >= 0 && !refuses(p, v.draft, q, v.s.u[first + t])))
      continue;
    accepted = (uint32_t)t;
    break;
  }
  accepted = block_reduce<kN>(accepted, [](uint32_t x, uint32_t y) { return min(x, y); }, lds);
  Border p, q;
  if (accepted < kKept)
    p = kept[accepted][0], q = kept[accepted][1];
  else
    borders((int)accepted, p, q);
  return rest_at<kType>(v, seq, (int)accepted, p, v.draft && (int)accepted < v.tokens, q);
}

// What the token is drawn by: a token's own weight, and what is left of it where the
// draft's share is taken away.
template <int kType>
struct Weights {
  const Rest<kType>& r;
  Weigher p, q;

  DIP_DEV Weights(const SampleArgs& a, const Rest<kType>& rest, const double* roots)
      : r(rest),
        p(a, roots, rest.p.top, rest.p.least),
        q(a, roots, rest.draft ? rest.q.top : rest.p.top,
          rest.draft ? rest.q.least : rest.p.least) {}
  DIP_DEV uint64_t own(int64_t i, float x) const {
    const uint32_t k = order_key(x);
    return r.p.cut.keeps(k, i) ? p.key_kept(k) : 0ull;
  }
  DIP_DEV uint64_t left(int64_t i, uint64_t w) const {
    if (!r.draft) return i == r.x ? 0 : w;
    if (w == 0) return 0;
    return left(i, w, load_logit<kType>(r.draft, i));
  }
  DIP_DEV uint64_t left(int64_t i, uint64_t w, float y) const {
    const uint32_t k = order_key(y);
    const uint64_t o = r.q.cut.keeps(k, i) ? q.key_kept(k) : 0ull;
    const double d = (double)w * r.p_by - (double)o * r.q_by;
    return d > 0.0 ? Weigher::whole(d) : 0ull;
  }
};

template <int kType, bool kParts>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[kLdsWords];
  __shared__ double roots[64];
  const int seq = blockIdx.x / v.slices, s = blockIdx.x % v.slices;
  Weigher::put_roots(v.s, roots);
  __syncthreads();
  uint32_t* words = reinterpret_cast<uint32_t*>(lds);
  const Rest<kType> rest = kParts ? rest_of_parts<kType, kThreads>(v, seq, roots, words)
                                  : rest_of<kType, kThreads>(v, seq, words);
  uint64_t left = 0, own = 0;
  if (rest.p.total) {
    const Weights<kType> w(v.s, rest, roots);
    const int64_t vocab = v.s.vocab, v0 = s * v.slice_vecs;
    const int64_t v1 = min(v0 + v.slice_vecs, row_vecs<kType>(rest.row, vocab));
    const auto add = [&](int64_t i, float x) {
      const uint64_t o = w.own(i, x);
      own += o;
      left += w.left(i, o);
    };
    // Filters keep few tokens, whose draft's logits are fetched one by one; without any,
    // pieces of both rows are, where they lie alike.
    if (kParts && rest.draft &&
        ((reinterpret_cast<uintptr_t>(rest.draft) ^ reinterpret_cast<uintptr_t>(rest.row)) & 15) ==
            0) {
      for (int64_t at = v0 + threadIdx.x; at < v1; at += kThreads) {
        const Piece<kType> p(rest.row, vocab, at), q(rest.draft, vocab, at);
        Piece<kType>::pairs(p, q, rest.row, rest.draft, vocab, [&](int64_t i, float x, float y) {
          const uint64_t o = w.own(i, x);
          own += o;
          left += w.left(i, o, y);
        });
      }
    } else {
      each_token<kType>(rest.row, vocab, v0, v1, add);
    }
  }
  const auto add = [](uint64_t x, uint64_t y) { return x + y; };
  left = block_reduce(left, add, lds);
  own = block_reduce(own, add, lds);
  if (threadIdx.x == 0) {
    // (with filters the draw finds it out again: kept from here, this launch took 22 us
    // for 9, 16 rows of 151936 fp32, and the draw 7.7 for 8.4)
    if (kParts && s == 0) v.decided[seq] = Decided{rest.p, rest.q, rest.accepted};
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

template <int kType, bool kParts>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[lds_words<kDrawThreads>];
  __shared__ double roots[64];
  const int seq = blockIdx.x, tid = threadIdx.x;
  const int64_t vocab = v.s.vocab;
  uint64_t* sh = lds + 2 * (kDrawThreads / 64);
  const uint64_t* sums = v.sums + 2 * (int64_t)seq * v.slices;
  const uint64_t slice_left = tid < v.slices ? sums[2 * tid] : 0;
  const uint64_t slice_own = tid < v.slices ? sums[2 * tid + 1] : 0;
  Weigher::put_roots(v.s, roots);
  __syncthreads();
  const Decided& d = v.decided[kParts ? seq : 0];
  const Rest<kType> rest =
      kParts ? rest_at<kType>(v, seq, (int)d.accepted, d.p, v.draft && d.accepted < v.tokens, d.q)
             : rest_of<kType, kDrawThreads>(v, seq, reinterpret_cast<uint32_t*>(lds));
  put_drafts<kDrawThreads>(v, seq, rest.accepted);
  int64_t* token = v.out + (int64_t)seq * (v.tokens + 1) + rest.accepted;
  if (rest.p.total == 0) {  // nothing to choose from
    if (tid == 0) *token = 0;
    return;
  }
  const Weights<kType> w(v.s, rest, roots);
  if (tid < 2) sh[tid] = 0;
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

// A slice's weights added up by its own largest logit, its pieces held in registers.
template <int kType>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(VerifyArgs v) {
  __shared__ uint64_t lds[kLdsWords];
  __shared__ double roots[64];
  const SampleArgs& a = v.s;
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
  const char* row = row_of(a, r);
  const int64_t v0 = s * a.slice_vecs;
  const int64_t v1 = min(v0 + a.slice_vecs, row_vecs<kType>(row, a.vocab));
  Piece<kType> p[kSumPieces];
#pragma unroll
  for (int j = 0; j < kSumPieces; ++j) {
    const int64_t at = v0 + threadIdx.x + j * kThreads;
    p[j] = Piece<kType>(row, a.vocab, at < v1 ? at : INT32_MAX);
  }
  auto mine = [&](auto f) {
#pragma unroll
    for (int j = 0; j < kSumPieces; ++j)
      if (v0 + threadIdx.x + j * kThreads < v1)
        p[j].tokens(row, a.vocab, [&](int64_t, float x) { f(x); });
  };
  Weigher::put_roots(a, roots);
  float most = -INFINITY;
  mine([&](float x) { most = fmaxf(most, x); });
  const uint32_t top =
      block_reduce(order_key(most), [](uint32_t x, uint32_t y) { return max(x, y); },
                   reinterpret_cast<uint32_t*>(lds));
  uint64_t sum = 0;
  if (top > kKeyMinusInf) {
    const Weigher wt(a, roots, top, top);
    mine([&](float x) { sum += wt.whole_of(wt.value(x)); });
  }
  sum = block_reduce(sum, [](uint64_t x, uint64_t y) { return x + y; }, lds);
  if (threadIdx.x == 0) v.parts[blockIdx.x] = Part{top, sum};
}

// Whether a thread may have one of a workgroup's k largest words (order_key << 32 | ~index):
// only the k threads whose own largest are the k largest of these do.  `most`: the thread's,
// 0 if it has none; threads have their words in the order of their indices, so of threads
// with equal keys the first ones count.  least: the k-th largest of the keys, which the
// words that count are not below.  kBits: the keys' upper bits that differ at all.
template <int kBits>
DIP_DEV bool among_largest(uint64_t most, int k, uint32_t* lds, uint32_t& least) {
  constexpr int kShift = 32 - kBits;
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t mine = (uint32_t)(most >> 32) >> kShift;
  lds[threadIdx.x] = mine;
  __syncthreads();
  uint32_t v[kThreads / 64];
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v[i] = lds[64 * i + l];
  uint32_t kth = 0;  // the largest number that k of them reach, a bit at a time
#pragma unroll
  for (int bit = kBits - 1; bit >= 0; --bit) {
    const uint32_t next = kth | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) n += __popcll(__ballot(v[i] >= next));
    kth = n >= k ? next : kth;
  }
  least = kth << kShift;
  int more = 0, before = 0;  // threads above it; equal ones before this
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    more += __popcll(__ballot(v[i] > kth));
    const uint64_t same = __ballot(v[i] == kth);
    before += i < wave ? __popcll(same) : i == wave ? __popcll(same & ((1ull << l) - 1)) : 0;
  }
  return most > 0 && (mine > kth || (mine == kth && before < k - more));
}

// The k largest of `list` (n words, that differ) in descending order to out, 0 behind the
// last.
DIP_DEV void put_largest(const uint64_t* list, int n, int k, uint64_t* out) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t x = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > x;
    if (rank < k) out[rank] = x;
  }
  for (int i = n + (int)threadIdx.x; i < k; i += kThreads) out[i] = 0;
}

// A slice's k largest tokens, a run of neighbouring pieces per thread.
template <int kType, int kPieces>
__global__ __launch_bounds__(kThreads) void verify_top_kernel(VerifyArgs v) {
  constexpr int kVec = Piece<kType>::kVec;
  constexpr int kBits = kType == DIP_BF16 ? 16 : kType == DIP_F16 ? 20 : 32;
  __shared__ uint64_t list[kTopMost * kPieces * kVec];
  __shared__ uint32_t lds[kThreads];
  __shared__ int listed;
  const SampleArgs& a = v.s;
  const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices, k = (int)a.top_k;
  const char* row = row_of(a, r);
  const int64_t v0 = s * a.slice_vecs;
  const int64_t v1 = min(v0 + a.slice_vecs, row_vecs<kType>(row, a.vocab));
  const int64_t at = v0 + (int)threadIdx.x * kPieces;
  Piece<kType> p[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    p[j] = Piece<kType>(row, a.vocab, at + j < v1 ? at + j : INT32_MAX);
  auto mine = [&](auto f) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      if (at + j < v1)
        p[j].tokens(row, a.vocab, [&](int64_t i, float x) {
          const uint32_t key = order_key(x);
          if (key > kKeyMinusInf) f((uint64_t)key << 32 | (uint32_t)~(uint32_t)i);
        });
  };
  if (threadIdx.x == 0) listed = 0;
  uint64_t most = 0;
  mine([&](uint64_t x) { most = max(most, x); });
  uint32_t least;
  if (among_largest<kBits>(most, k, lds, least))
    mine([&](uint64_t x) {
      if ((uint32_t)(x >> 32) >= least) list[atomicAdd(&listed, 1)] = x;
    });
  __syncthreads();
  put_largest(list, listed, k, v.best + (int64_t)blockIdx.x * k);
}

// A row's k largest of its slices', their weights, and what the filters keep of them.
__global__ __launch_bounds__(kThreads) void verify_top_rows_kernel(VerifyArgs v) {
  __shared__ uint64_t list[kTopMost * kMaxSlices * kTopMost / kThreads];
  __shared__ uint32_t lds[kThreads];
  __shared__ uint64_t top[kTopMost];
  __shared__ double roots[64];
  __shared__ int listed;
  const SampleArgs& a = v.s;
  const int r = blockIdx.x, k = (int)a.top_k, n = a.slices * k, tid = threadIdx.x;
  const uint64_t* best = v.best + (int64_t)r * n;
  const int64_t x = token_of(v, r);
  if (a.slices == 1) {
    if (tid < k) top[tid] = best[tid];
  } else {
    if (tid == 0) listed = 0;
    // a run of neighbours per thread: slices come in the order of their indices, and
    // equal keys of a slice too
    const int per = (n + kThreads - 1) / kThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
    uint64_t most = 0;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) most = max(most, best[i]);
    uint32_t least;
    if (among_largest<32>(most, k, lds, least))
#pragma unroll 8
      for (int i = i0; i < i1; ++i) {
        const uint64_t x = best[i];
        if (x > 0 && (uint32_t)(x >> 32) >= least) list[atomicAdd(&listed, 1)] = x;
      }
    __syncthreads();
    put_largest(list, listed, k, top);
  }
  __syncthreads();
  const uint32_t first = (uint32_t)(top[0] >> 32);
  if (first <= kKeyMinusInf) {
    if (tid == 0) v.borders[r] = Border{first, 0u, Cut{0u, 0}, 0, 0};
    return;
  }
  const Weigher wt(a, first, first, roots);
  __syncthreads();
  if (tid >= 64) return;
  const uint64_t mine = tid < k ? top[tid] : 0;
  const uint32_t key = (uint32_t)(mine >> 32), index = (uint32_t)~(uint32_t)mine;
  const double w = mine ? wt.key_scaled(key) : 0.0;
  const uint64_t whole = Weigher::whole(w);
  uint64_t run = whole;  // of the tokens up to this one
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = __shfl_up(run, m, 64);
    if (tid >= m) run += o;
  }
  const double mass = a.top_p * (double)(uint64_t)__shfl(run, 63, 64);
  const bool kept = mine && (a.top_p >= 1 || (double)(run - whole) < mass) && w >= wt.least;
  const uint64_t weight = kept ? whole : 0;
  uint64_t total = weight, drafted = (int64_t)index == x ? weight : 0;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    total += __shfl_xor(total, m, 64);
    drafted += __shfl_xor(drafted, m, 64);
  }
  v.tops[r].weight[tid] = weight;
  v.tops[r].index[tid] = index;
  if (tid == 0) v.borders[r] = Border{first, 0u, Cut{0u, 0}, total, drafted};
}

// The token of such rows: a wave per sequence, a token per lane.
template <int kType>
__global__ __launch_bounds__(64) void verify_top_draw_kernel(VerifyArgs v) {
  __shared__ uint32_t lds[1];
  const int seq = blockIdx.x, l = threadIdx.x, first = seq * (v.tokens + 1);
  const Rest<kType> rest = rest_of<kType, 64>(v, seq, lds);
  put_drafts<64>(v, seq, rest.accepted);
  int64_t* token = v.out + first + rest.accepted;
  if (rest.p.total == 0) {  // nothing to choose from
    if (l == 0) *token = 0;
    return;
  }
  const TopRow& p = v.tops[first + rest.accepted];
  const uint64_t own = p.weight[l];
  const uint32_t index = p.index[l];
  uint64_t left = own;
  if (rest.draft && rest.q.total) {
    const TopRow& q = v.tops[v.seqs * (v.tokens + 1) + seq * v.tokens + rest.accepted];
    const uint64_t qw = q.weight[l];
    const uint32_t qi = q.index[l];
    uint64_t taken = 0;
    for (int j = 0; j < 64; ++j) {
      const uint64_t w = __shfl(qw, j, 64);
      if (__shfl(qi, j, 64) == index) taken += w;  // (words without a token weigh 0)
    }
    const double d = (double)own * rest.p_by - (double)taken * rest.q_by;
    left = own && d > 0.0 ? Weigher::whole(d) : 0;
  } else if (!rest.draft && (int64_t)index == rest.x) {
    left = 0;
  }
  uint64_t total = left;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) total += __shfl_xor(total, m, 64);
  if (total == 0) {  // (numbers u outside [0, 1), or p and q the same)
    left = own;
    total = rest.p.total;
  }
  uint64_t before = 0;  // by index
  for (int j = 0; j < 64; ++j) {
    const uint64_t w = __shfl(left, j, 64);
    if (__shfl(index, j, 64) < index) before += w;
  }
  const uint64_t goal = goal_of(v.s.u[first + v.tokens], total);
  if (goal >= before && goal - before < left) *token = index;
}

// Slices of `pieces` 16-byte pieces per thread.  One keeps a single sequence's launch
// short, four many rows' launches few.
constexpr int kTopPieces = 4;
inline int64_t top_slice(int64_t rows, int64_t vecs) {
  return rows * ((vecs + kThreads - 1) / kThreads) <= 2048 && vecs <= kMaxSlices * kThreads
             ? kThreads
             : kTopPieces * kThreads;
}
// Whether the k largest tokens of a row are found first.
inline bool by_top(int64_t top_k, int64_t vocab, int64_t vecs) {
  return top_k > 1 && top_k <= kTopMost && top_k < vocab && vecs <= kMaxSlices * kTopPieces * kThreads;
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
  if (v.best) {
    const dim3 slices((unsigned)rows * v.s.slices);
    if (v.s.slice_vecs <= kThreads)
      hipLaunchKernelGGL((verify_top_kernel<kType, 1>), slices, dim3(kThreads), 0, s, v);
    else
      hipLaunchKernelGGL((verify_top_kernel<kType, kTopPieces>), slices, dim3(kThreads), 0, s, v);
    hipLaunchKernelGGL(verify_top_rows_kernel, dim3(rows), dim3(kThreads), 0, s, v);
    hipLaunchKernelGGL((verify_top_draw_kernel<kType>), dim3(v.seqs), dim3(64), 0, s, v);
    return hip_status(hipGetLastError());
  }
  if (v.parts) {
    hipLaunchKernelGGL((verify_sum_kernel<kType>), dim3((unsigned)rows * v.s.slices),
                       dim3(kThreads), 0, s, v);
    hipLaunchKernelGGL((verify_rest_kernel<kType, true>), dim3((unsigned)v.seqs * v.slices),
                       dim3(kThreads), 0, s, v);
    hipLaunchKernelGGL((verify_draw_kernel<kType, true>), dim3(v.seqs), dim3(kDrawThreads), 0, s,
                       v);
    return hip_status(hipGetLastError());
  }
  const bool greedy = v.s.per_64th == 0;
  const int threads = row_threads(v.s, rows, vecs);
  if (threads == kThreads) {
    launch_rows<kType, kThreads>(v, rows, s);
  } else if (threads) {
    launch_rows<kType, 1024>(v, rows, s);
  } else if (greedy) {
    launch_slices_max(kType, v.s, rows, s);
  } else {
    launch_slices(kType, v.s, rows, s);
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
  hipLaunchKernelGGL((verify_rest_kernel<kType, false>), dim3((unsigned)v.seqs * v.slices),
                     dim3(kThreads), 0, s, v);
  hipLaunchKernelGGL((verify_draw_kernel<kType, false>), dim3(v.seqs), dim3(kDrawThreads), 0, s, v);
  return hip_status(hipGetLastError());
}

inline size_t top_bytes(int64_t rows, int64_t vecs, int64_t k) {
  const int64_t per = top_slice(rows, vecs);
  return (size_t)rows * (sizeof(TopRow) + (vecs + per - 1) / per * k * sizeof(uint64_t));
}
// Slices of rows without filters, 64 at most and of kSumPieces per thread at most; 0: too
// long.  About two thousand workgroups in all.
inline int sum_slices(int64_t rows, int64_t vecs) {
  const int64_t least = (vecs + kSumPieces * kThreads - 1) / (kSumPieces * kThreads);
  const int64_t most = min((vecs + kThreads - 1) / kThreads, (int64_t)64);
  return least > 64 ? 0 : (int)max(least, min(most, 2048 / rows));
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

// For `rows` rows of any type (fp32 rows take the most slices) and any filters.
inline size_t workspace_of(int64_t seqs, int64_t rows, int64_t vocab) {
  const int64_t vecs = max_vecs(vocab, 4);
  size_t n = (size_t)seqs * slices_for(seqs, vecs) * 16;
  if (vecs > kOneLaunch)
    n += (size_t)rows *
         (sizeof(RowState) + (size_t)slices_for(rows, vecs) * kBins * sizeof(uint64_t));
  for (int size = 2; size <= 4; size += 2) {  // (shorter rows may be cut finer)
    const int64_t w = max_vecs(vocab, size);
    if (by_top(kTopMost, kTopMost + 1, w)) n = max(n, top_bytes(rows, w, kTopMost));
    n = max(n, (size_t)seqs * slices_for(seqs, w) * 16 +
                   (size_t)rows * sum_slices(rows, w) * sizeof(Part));
  }
  return up16(rows * sizeof(Border)) + up16(seqs * sizeof(Decided)) + n;
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" size_t dip_verify_workspace_size(int64_t seqs, int64_t tokens, int64_t vocab,
                                            int draft_logits) {
  if (!sizes_ok(seqs, tokens, vocab) || seqs == 0) return 0;
  // fewer rows may be cut finer, and greedy calls do without the draft's
  size_t n = workspace_of(seqs, rows_of(seqs, tokens, false), vocab);
  if (draft_logits) n = max(n, workspace_of(seqs, rows_of(seqs, tokens, true), vocab));
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
  v.decided = reinterpret_cast<Decided*>(w);
  w += up16(seqs * sizeof(Decided));
  if (s.per_64th > 0 && by_top(top_k, vocab, vecs)) {
    v.tops = reinterpret_cast<TopRow*>(w);
    v.best = reinterpret_cast<uint64_t*>(w + rows * sizeof(TopRow));
    s.slice_vecs = top_slice(rows, vecs);
    s.slices = (int)((vecs + s.slice_vecs - 1) / s.slice_vecs);
  }
  v.sums = reinterpret_cast<uint64_t*>(w);
  w += (size_t)seqs * v.slices * 16;
  s.rows = w;
  if (s.per_64th > 0 && !counts(s) && min_p == 0 && sum_slices(rows, vecs)) {
    v.parts = reinterpret_cast<Part*>(w);
    s.slices = sum_slices(rows, vecs);
    s.slice_vecs = (vecs + s.slices - 1) / s.slices;
  }
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
