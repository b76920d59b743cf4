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
// (logit, index), so ties are cut by index and nothing is sorted.
//
// Weights and their sums are held in 64 bits: with 150000 tokens a sum in 32
// bits is off by more than an unlikely token's weight.
#include "dip_common.h"
#include "dip_internal.h"

#include <hip/hip_fp16.h>

namespace dip {
namespace {

constexpr int kThreads = 1024;
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

struct SampleArgs {
  const void* logits;
  int64_t vocab, row_bytes;
  const float* u;
  double temperature, top_p, min_p;
  int64_t top_k;
  int shift;  // weights as whole numbers: w * 2^shift, whose sums stay below 2^63
  int64_t* token;
  float* prob;
};

struct Cut {  // the last kept token of the order
  uint32_t key;
  int64_t index;
};

template <typename T, typename F>
DIP_DEV T block_reduce(T v, F f, T* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = f(v, (T)__shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int i = 1; i < kThreads / 64; ++i) v = f(v, lds[i]);
  return v;
}

// The sum of the threads before this one; `total`: of all.
template <typename T>
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
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i == (int)(threadIdx.x >> 6)) before = total;
    total += lds[i];
  }
  return before + run - v;
}

template <int kType>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ uint64_t lds[kThreads / 64];
  __shared__ uint32_t hn[kRadixBins];
  __shared__ unsigned long long hw[kRadixBins];
  __shared__ uint64_t sh[4];
  const char* row = static_cast<const char*>(a.logits) + (int64_t)blockIdx.x * a.row_bytes;
  const int tid = threadIdx.x;
  uint32_t top = 0;
  for (int64_t i = tid; i < a.vocab; i += kThreads) top = max(top, order_key(load_logit<kType>(row, i)));
  top = block_reduce(top, [](uint32_t x, uint32_t y) { return max(x, y); },
                     reinterpret_cast<uint32_t*>(lds));
  if (top <= kKeyMinusInf) {  // nothing to choose from
    if (tid == 0) {
      a.token[blockIdx.x] = 0;
      if (a.prob) a.prob[blockIdx.x] = 0.f;
    }
    return;
  }
  const double most = key_value(top);
  auto weight = [&](uint32_t k) {
    if (k == top) return 1.0;
    if (a.temperature == 0 || k <= kKeyMinusInf) return 0.0;
    return exp(((double)key_value(k) - most) / a.temperature);
  };
  Cut cut{0u, a.vocab};
  auto kept = [&](uint32_t k, int64_t i) { return k > cut.key || (k == cut.key && i <= cut.index); };

  // The border of the first `count` tokens (by_mass false) or of the fewest kept
  // tokens whose weights reach `mass`: the key from its highest byte down, then
  // the index among the tokens of that key.
  auto find = [&](bool by_mass, uint64_t count, double mass) {
    uint32_t prefix = 0;
    uint64_t above_n = 0, above_w = 0, tie_w = 0;
    for (int level = 24; level >= 0; level -= 8) {
      for (int b = tid; b < kRadixBins; b += kThreads) hn[b] = 0, hw[b] = 0;
      __syncthreads();
      for (int64_t i = tid; i < a.vocab; i += kThreads) {
        const uint32_t k = order_key(load_logit<kType>(row, i));
        if (!kept(k, i) || (level < 24 && (k >> (level + 8)) != (prefix >> (level + 8)))) continue;
        atomicAdd(&hn[(k >> level) & 255], 1u);
        if (by_mass)
          atomicAdd(&hw[(k >> level) & 255],
                    (unsigned long long)(ldexp(weight(k), a.shift) + 0.5));
      }
      __syncthreads();
      if (tid == 0) {
        uint64_t n = above_n, w = above_w;
        int b = kRadixBins - 1, last = -1;
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
      tie_w = sh[3];
      __syncthreads();
    }
    const uint64_t ties = tie_w;
    uint64_t need = count - above_n;
    if (by_mass) {
      const double w = (double)(uint64_t)(ldexp(weight(prefix), a.shift) + 0.5);
      const double n = w > 0 ? ceil((mass - (double)above_w) / w) : 1.0;
      need = n < 1.0 ? 1 : (n < (double)ties ? (uint64_t)n : ties);
    }
    // the index of the need-th token of that key
    const int64_t chunk = (a.vocab + kThreads - 1) / kThreads;
    const int64_t lo = min(tid * chunk, a.vocab), hi = min(lo + chunk, a.vocab);
    uint64_t mine = 0, all;
    for (int64_t i = lo; i < hi; ++i) mine += order_key(load_logit<kType>(row, i)) == prefix;
    const uint64_t before = block_exclusive(mine, lds, all);
    if (before < need && need <= before + mine) {
      uint64_t left = need - before;
      for (int64_t i = lo; i < hi; ++i)
        if (order_key(load_logit<kType>(row, i)) == prefix && --left == 0) {
          sh[0] = (uint64_t)i;
          break;
        }
    }
    __syncthreads();
    const Cut c{prefix, (int64_t)sh[0]};
    __syncthreads();
    return c;
  };

  if (a.temperature == 0) {
    cut = find(false, 1, 0.0);
  } else {
    if (a.top_k > 0 && a.top_k < a.vocab) cut = find(false, (uint64_t)a.top_k, 0.0);
    if (a.top_p < 1) {
      uint64_t w = 0;
      for (int64_t i = tid; i < a.vocab; i += kThreads) {
        const uint32_t k = order_key(load_logit<kType>(row, i));
        if (kept(k, i)) w += (uint64_t)(ldexp(weight(k), a.shift) + 0.5);
      }
      w = block_reduce(w, [](uint64_t x, uint64_t y) { return x + y; }, lds);
      cut = find(true, 0, a.top_p * (double)w);
    }
  }

  // running sums by index
  const int64_t chunk = (a.vocab + kThreads - 1) / kThreads;
  const int64_t lo = min(tid * chunk, a.vocab), hi = min(lo + chunk, a.vocab);
  auto final_weight = [&](int64_t i) {
    const uint32_t k = order_key(load_logit<kType>(row, i));
    if (!kept(k, i)) return 0.0;
    const double w = weight(k);
    return w >= a.min_p ? w : 0.0;
  };
  double mine = 0, total;
  for (int64_t i = lo; i < hi; ++i) mine += final_weight(i);
  const double before = block_exclusive(mine, reinterpret_cast<double*>(lds), total);
  const double t = (double)a.u[blockIdx.x] * total;
  int64_t found = INT64_MAX, last = -1;
  if (mine > 0) {
    double run = before;
    for (int64_t i = lo; i < hi; ++i) {
      const double w = final_weight(i);
      if (w == 0) continue;
      run += w;
      last = i;
      if (run > t) {
        found = i;
        break;
      }
    }
  }
  found = block_reduce(found, [](int64_t x, int64_t y) { return min(x, y); },
                       reinterpret_cast<int64_t*>(lds));
  last = block_reduce(last, [](int64_t x, int64_t y) { return max(x, y); },
                      reinterpret_cast<int64_t*>(lds));
  if (tid == 0) {
    const int64_t i = found != INT64_MAX ? found : last;  // u at or beyond 1: the last kept
    a.token[blockIdx.x] = i;
    if (a.prob) a.prob[blockIdx.x] = (float)(final_weight(i) / total);
  }
}

}  // namespace
}  // namespace dip

using namespace dip;

extern "C" size_t dip_sample_workspace_size(int64_t rows, int64_t vocab) {
  (void)rows;
  (void)vocab;
  return 0;
}

extern "C" int dip_sample(const void* logits, int dtype, int64_t rows, int64_t vocab,
                          int64_t row_stride, const float* u, double temperature, int64_t top_k,
                          double top_p, double min_p, int64_t* token, float* prob,
                          void* workspace, size_t ws_bytes, void* stream) {
  if (dtype != DIP_BF16 && dtype != DIP_F16 && dtype != DIP_F32) return DIP_ERR_UNSUPPORTED;
  if (rows < 0 || rows > INT32_MAX || vocab <= 0 || vocab > INT32_MAX || row_stride < 0)
    return DIP_ERR_SHAPE;
  if (!(temperature >= 0) || temperature > 1e300 || top_k < 0 || !(top_p > 0 && top_p <= 1) ||
      !(min_p >= 0 && min_p <= 1))
    return DIP_ERR_ARG;
  if (rows == 0) return DIP_OK;
  if (!logits || !u || !token) return DIP_ERR_NULL;
  const size_t need = dip_sample_workspace_size(rows, vocab);
  if (need && (!workspace || ws_bytes < need)) return DIP_ERR_WORKSPACE;
  const int size = dtype == DIP_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return DIP_ERR_ALIGN;
  int shift = 62;
  for (int64_t n = 1; n < vocab; n *= 2) --shift;
  SampleArgs a{logits, vocab, row_stride * size, u, temperature, top_p, min_p, top_k, shift, token,
               prob};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DIP_F32)
    hipLaunchKernelGGL((sample_kernel<DIP_F32>), dim3((unsigned)rows), dim3(kThreads), 0, s, a);
  else if (dtype == DIP_F16)
    hipLaunchKernelGGL((sample_kernel<DIP_F16>), dim3((unsigned)rows), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((sample_kernel<DIP_BF16>), dim3((unsigned)rows), dim3(kThreads), 0, s, a);
  return hip_status(hipGetLastError());
}
