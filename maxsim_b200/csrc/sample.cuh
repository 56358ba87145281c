// Drawing candidates from score rows, next to the ranking of pack.cuh.
//
// For a row of scores s: candidates are the entries that are neither NaN nor
// -inf.  With a_i = (s_i - max s) / T (0 where s_i = max s, also when that is
// +inf) a candidate weighs w_i = exp(a_i); under a_i = -700 it counts as none.  In the order
// "score descending, index ascending" every filter keeps a prefix:
//   top-k   the first k
//   top-p   of those, the ones before which less than p of their mass lies
//   min-p   w_i >= min_p (times the best weight, which is 1)
// n candidates are drawn without replacement: the n largest of
// a_i - log(-log u_i) among the kept, largest first, equal ones by lowest
// index.  -log(u_i) / w_i is the arrival time of an exponential clock of rate
// w_i, so the arrivals in order are n successive draws, each in proportion to the
// weights still there (the exponential race; for n = 1 the Gumbel-max form of
// sampling).
//
// Which candidates come out hangs on comparisons, so a, w and the race are 64-bit
// and masses are whole numbers (w * 2^shift), whose sums do not depend
// on the order they are taken in.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace maxsim {
namespace sample {

constexpr int kThreads = 256;
constexpr double kLeast = -700.0;  // exponents below it weigh nothing

// A parameter of the call: one value, or one per row.
template <typename T, typename S>
struct Param {
  S value;
  const T* rows;
  __device__ __forceinline__ S at(int64_t row) const { return rows ? (S)rows[row] : value; }
};

struct Args {
  const float* scores;
  const float* uniforms;
  int64_t score_stride, uniform_stride;
  int64_t rows;
  int cols, n;
  Param<float, double> temperature, top_p, min_p;
  Param<int32_t, int64_t> top_k;
  int shift;  // masses are w * 2^shift: the sum of cols of them stays under 2^63
  int64_t* indices;
  float* probabilities;
};

// Order-preserving image of a float; -0 and +0 are equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* shared, Op op) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < kThreads / 32; ++w) v = op(v, shared[w]);
  return v;
}

// One CTA per row; every step is a pass over the row in memory and a reduction,
// thresholds are found by bisection over the 32-bit image of the scores.
__global__ void __launch_bounds__(kThreads) sample_rows_kernel(Args A) {
  __shared__ unsigned long long red[kThreads / 32];
  __shared__ double red_d[kThreads / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, C = A.cols;
  const float* s = A.scores + row * A.score_stride;
  const float* u = A.uniforms + row * A.uniform_stride;
  const double T = A.temperature.at(row);
  const auto add = [](unsigned long long a, unsigned long long b) { return a + b; };
  const auto most = [](unsigned long long a, unsigned long long b) { return a > b ? a : b; };

  // the best candidate (key 0: there is none)
  unsigned long long k0 = 0;
  for (int i = tid; i < C; i += kThreads) {
    const float v = s[i];
    if (v > -INFINITY) k0 = most(k0, key_of(v));
  }
  const uint32_t best_key = (uint32_t)block_reduce(k0, red, most);
  const uint32_t b = (best_key & 0x80000000u) ? (best_key & 0x7fffffffu) : ~best_key;
  const float best = __uint_as_float(b);
  const bool some = best_key != 0 && T > 0.0;

  const auto exponent = [&](float v) { return v == best ? 0.0 : ((double)v - (double)best) / T; };
  const auto candidate = [&](float v) { return v > -INFINITY && exponent(v) >= kLeast; };
  const double scale = ldexp(1.0, A.shift);
  const auto mass = [&](float v) { return (unsigned long long)__double2ull_rn(exp(exponent(v)) * scale); };
  const auto count_from = [&](uint32_t key) {  // candidates with at least this key
    unsigned long long n = 0;
    for (int i = tid; i < C; i += kThreads) n += candidate(s[i]) && key_of(s[i]) >= key;
    return block_reduce(n, red, add);
  };

  // The kept prefix as (cut, ties): all with a larger key, and the first `ties` with key `cut`.
  uint32_t cut = 0;
  unsigned long long ties = ~0ull;
  unsigned long long all = some ? count_from(0) : 0;
  int64_t k = A.top_k.at(row);
  if (some && k > 0 && (unsigned long long)k < all) {
    uint32_t lo = 0, hi = best_key;  // count_from(lo) >= k; the largest such key is wanted
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (count_from(mid) >= (unsigned long long)k) lo = mid; else hi = mid - 1;
    }
    cut = lo;
    ties = (unsigned long long)k - (cut == 0xffffffffu ? 0 : count_from(cut + 1));
  }
  const auto key_value = [](uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
  };
  const auto mass_above = [&](uint32_t key) {
    unsigned long long m = 0;
    for (int i = tid; i < C; i += kThreads)
      if (candidate(s[i]) && key_of(s[i]) > key) m += mass(s[i]);
    return block_reduce(m, red, add);
  };
  const double p = A.top_p.at(row);
  if (some && p > 0.0 && p < 1.0) {
    unsigned long long M = mass_above(cut);
    if (cut) M += ties * mass(key_value(cut));
    const double limit = p * (double)M;
    uint32_t lo = cut, hi = best_key;  // the smallest key with mass_above(key) < limit
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if ((double)mass_above(mid) < limit) hi = mid; else lo = mid + 1;
    }
    if (lo > 0) {
      const unsigned long long above = mass_above(lo), each = mass(key_value(lo));
      unsigned long long equal = count_from(lo) - (lo == 0xffffffffu ? 0 : count_from(lo + 1));
      if (lo == cut && ties < equal) equal = ties;
      // how many r >= 0 have above + r * each < limit
      unsigned long long r = equal;
      if (each > 0) {
        const double q = (limit - (double)above) / (double)each;
        r = q >= (double)equal ? equal : (unsigned long long)q;
        while (r < equal && (double)(above + r * each) < limit) ++r;
        while (r > 1 && (double)(above + (r - 1) * each) >= limit) --r;
      }
      cut = lo;
      ties = r < 1 ? 1 : r;
    }
  }
  // ties are taken in index order: those before `bound`
  int bound = C;
  if (some && cut > 0) {
    int lo = 0, hi = C;  // the smallest bound with `ties` equal keys before it, or C
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      unsigned long long n = 0;
      for (int i = tid; i < mid; i += kThreads) n += candidate(s[i]) && key_of(s[i]) == cut;
      if (block_reduce(n, red, add) >= ties) hi = mid; else lo = mid + 1;
    }
    bound = lo;
  }
  const double least_share = A.min_p.at(row);
  const bool by_share = least_share > 0.0 && least_share <= 1.0;
  const auto kept = [&](int i) {
    const float v = s[i];
    if (!some || !candidate(v)) return false;
    const uint32_t key = key_of(v);
    if (key < cut || (key == cut && i >= bound)) return false;
    return !by_share || exp(exponent(v)) >= least_share;
  };
  unsigned long long sum = 0;
  for (int i = tid; i < C; i += kThreads)
    if (kept(i)) sum += mass(s[i]);
  const double total = (double)block_reduce(sum, red, add);

  // n rounds: the largest race value behind the one drawn last
  double last = INFINITY;
  int last_i = -1;
  bool open = some;
  for (int d = 0; d < A.n; ++d) {
    double g = -INFINITY;
    int at = C;
    if (open)
      for (int i = tid; i < C; i += kThreads) {
        if (!kept(i)) continue;
        double r = exponent(s[i]) - log(-log((double)u[i]));
        if (!(r >= -1e300)) {
          if (r != r) continue;  // a uniform that is none
          r = -1e300;            // a uniform of 0 comes last
        }
        if (r > last || (r == last && i <= last_i)) continue;
        if (r > g) { g = r; at = i; }
      }
    const double top = block_reduce(g, red_d, [](double a, double b2) { return a > b2 ? a : b2; });
    const unsigned long long mine = g == top && top > -INFINITY ? (unsigned long long)at : ~0ull;
    const unsigned long long first =
        block_reduce(mine, red, [](unsigned long long a, unsigned long long b2) { return a < b2 ? a : b2; });
    if (first == ~0ull) open = false;
    else { last = top; last_i = (int)first; }
    if (tid == 0) {
      A.indices[row * A.n + d] = open ? (int64_t)last_i : -1;
      A.probabilities[row * A.n + d] = open ? (float)(exp(exponent(s[last_i])) * scale / total) : 0.f;
    }
  }
}

}  // namespace sample
}  // namespace maxsim
