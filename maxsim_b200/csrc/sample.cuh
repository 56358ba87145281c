// Drawing candidates from score rows, next to the ranking of pack.cuh.
//
// For a row of scores s: candidates are the entries that are neither NaN nor
// -inf.  With a_i = (s_i - max s) / T (0 where s_i = max s, also when that is
// +inf) a candidate weighs w_i = exp(a_i); under a_i = -700 it counts as none.  In the order
// "score descending, index ascending" every filter keeps a prefix:
//   top-k   the first k
//   top-p   of those, the ones before which less than p of their mass lies
//   min-p   a_i >= log(min_p): w_i >= min_p times the best weight, which is 1
// n candidates are drawn without replacement: the n largest of
// a_i - log(-log u_i) among the kept, largest first, equal ones by lowest
// index.  -log(u_i) / w_i is the arrival time of an exponential clock of rate
// w_i, so the arrivals in order are n successive draws, each in proportion to the
// weights still there (the exponential race; for n = 1 the Gumbel-max form of
// sampling).
//
// Which candidates come out hangs on comparisons, so a and the race are 64-bit
// and masses are whole numbers (w * 2^shift), whose sums do not depend
// on the order they are taken in.  Their sum has to fit 63 bits: shift is 51 for up to 2048
// columns and 42 for 2^20, so a mass is off by half of 2^-51 to 2^-42 of the best weight (one below
// that is none), and by the 3e-13 of its size that the exponential's series leaves.  (The total of the
// kept weights only scales the fp32 probabilities: 64-bit floating point, summed in a fixed order,
// each weight good to 6e-9, a tenth of an fp32 rounding.)
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "async.cuh"

namespace maxsim {
namespace sample {

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

// The exponent of a candidate, as defined (best: the row's largest score).
__device__ __forceinline__ double exponent(float v, float best, double T) {
  return v == best ? 0.0 : ((double)v - (double)best) / T;
}
// 2^y for -1010 < y <= 0, as 2^n times the Taylor series of 2^f = e^(f ln 2) up to f^DEGREE, n the
// whole number next to y and |f| <= 1/2.  The first term left out is below 6e-9 for degree 7 and
// 3e-13 for degree 10.  n comes out of the low bits of y + 1.5 * 2^52 and goes into the
// exponent's, with `more` added to it.
template <int DEGREE>
__device__ __forceinline__ double exp2_series(double y, int more) {
  constexpr double c[11] = {1.0,
                            0.6931471805599453,
                            0.2402265069591007,
                            0.055504108664821576,
                            0.009618129107628477,
                            0.0013333558146428441,
                            0.00015403530393381606,
                            1.5252733804059838e-05,
                            1.3215486790144305e-06,
                            1.0178086009239696e-07,
                            7.054911620801121e-09};
  const double whole = y + 6755399441055744.0, f = y - (whole - 6755399441055744.0);
  double e = c[DEGREE];
#pragma unroll
  for (int k = DEGREE - 1; k >= 0; --k) e = e * f + c[k];
  return __hiloint2double(__double2hiint(e) + ((__double2loint(whole) + more) << 20), __double2loint(e));
}
// An infinite score as a finite one: only the difference of two scores counts, and where
// the best is infinite every candidate is.
__device__ __forceinline__ double finite(float v) { return (double)fminf(v, 3.402823466e38f); }

// w * 2^shift as a whole number (shift <= 51), per_bit = 1 / (T ln 2); v not so far below the best
// that w < 2^-900.
__device__ __forceinline__ unsigned long long mass_here(float v, double best, double per_bit, int shift) {
  const double m = exp2_series<10>((finite(v) - best) * per_bit, shift) + 4503599627370496.0;  // 2^52: rounds
  return (unsigned long long)__double_as_longlong(m) & 0xfffffffffffffull;
}
// The functions of more 64-bit arithmetic are calls: inlined wherever they are used they
// made the kernel large enough that a CTA spent much of its time fetching it.
__device__ __noinline__ unsigned long long mass_of(float v, double best, double per_bit, int shift) {
  return mass_here(v, best, per_bit, shift);
}
__device__ __noinline__ double race_of(float v, float best, double T, float u) {
  const double r = exponent(v, best, T) - log(-log((double)u));
  return r < -1e300 ? -1e300 : r;  // a uniform of 0 comes last; NaN stays
}
__device__ __noinline__ float share_of(float v, float best, double T, double total) {
  return (float)(exp(exponent(v, best, T)) / total);
}
// Floats in order, as integers; -0 and +0 are one.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// The smallest finite score whose exponent is at least `least` (<= 0): exponents rise with
// scores, so one comparison of floats decides afterwards.  best + least * T is a few roundings
// away as a number, which near zero can be a great many floats: steps that double, then
// halving, some 60 tries at the very most.
__device__ __noinline__ float first_score(float best, double T, double least) {
  const auto holds = [&](uint32_t key) { return exponent(value_of(key), best, T) >= least; };
  const double guess = (double)best + least * T;
  const uint32_t lowest = key_of(-3.402823466e38f), top = key_of(best);  // holds(top)
  uint32_t x = guess >= best ? top : guess > -3.4e38 ? key_of(__double2float_ru(guess)) : lowest;
  uint32_t out = x, in = x;  // !holds(out), holds(in)
  if (holds(x)) {
    for (uint32_t step = 1;; step += step) {
      if (in == lowest) return value_of(in);
      const uint32_t next = in - lowest <= step ? lowest : in - step;
      if (!holds(next)) { out = next; break; }
      in = next;
    }
  } else {
    for (uint32_t step = 1;; step += step) {
      const uint32_t next = top - out <= step ? top : out + step;
      if (next == top || holds(next)) { in = next; break; }
      out = next;
    }
  }
  while (in - out > 1) {
    const uint32_t mid = out + (in - out) / 2;
    if (holds(mid)) in = mid; else out = mid;
  }
  return value_of(in);
}

struct Add {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Least {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a < b ? a : b; }
};
struct Most {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};

struct Or {
  __device__ __forceinline__ int operator()(int a, int b) const { return a | b; }
};

// The CTAs of a cluster and each other's shared memory.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// What every thread of the cluster wrote to any of its CTAs before is seen by all of them afterwards.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The address of a CTA's own shared variable in the CTA of that rank.
__device__ __forceinline__ uint32_t at_rank(const void* mine, uint32_t rank) {
  uint32_t there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  return there;
}
__device__ __forceinline__ void store_at(uint32_t there, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(v) : "memory");
}
__device__ __forceinline__ void store_at(uint32_t there, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there), "l"(v) : "memory");
}
__device__ __forceinline__ uint2 load_pair_at(uint32_t there) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(there) : "memory");
  return v;
}

// A CTA per row.  The row's scores are kept in shared memory (kCached, up to
// kMostCached columns) or read again from memory for each pass; with the race
// they are overwritten by its values.
//
// A threshold ("the k-th largest", "the last one before the mass reaches p") is found
// with histograms over a linear map of the scores, kBins bins from the largest to
// the smallest, of counts or of masses as two 32-bit words (shared-memory atomics of 32 bits are
// native, and integer sums do not depend on their order).  The bin that holds the threshold is looked at
// again: its members are ranked against each other when there are at most
// kListed, else the map zooms into it.  Every zoom separates its largest from its smallest
// member, so it ends; members that are all equal are taken in index order.
//
// The race is run twice: in 32 bits over all kept candidates, as lower bounds
// with the arithmetic's error taken off, whose n-th largest leaves out everything
// that cannot be among the n best; and in 64 bits for the few that are left.
//
// Few long rows get a cluster of CTAs each (kCluster): a CTA takes a slice of the row,
// reductions go on through the other CTAs' shared memory, every CTA adds up all the
// histograms, and every CTA comes to the same cut.  The candidates left for the 64-bit race
// go to the cluster's first CTA.  All branches around a cluster's barrier hang on values that are the
// same in all its CTAs.
//
// What bounds it: instructions and latency, not memory.  A row is read once, but
// every element then takes an exponential, two logarithms and a histogram step, and a
// row goes through some twenty barriers.
constexpr int kRaced = 2048;         // candidates of a row that are raced in 64 bits (a power of two)
constexpr int kFew = 384;            // kept candidates that go to the 64-bit race without the 32-bit one
constexpr int kMostCached = 40960;   // columns of a row (or of a CTA's slice) in shared memory
constexpr int kMostCtas = 16;        // of a cluster

template <int THREADS>
struct Shared {
  static constexpr int kBins = 2 * THREADS;
  static constexpr int kListed = THREADS < 256 ? THREADS : 256;  // members that are ranked against each other
  union {
    uint32_t bins[2][kBins];              // low and high words of a histogram
    struct {
      unsigned long long mass[kListed];   // of the ranked members, best first
      float score[kListed];
      int32_t index[kListed];
    } ranked;
    unsigned long long race[kRaced];      // order-preserving images of 64-bit race values
  };
  int32_t list[kRaced];
  unsigned long long words[2][5][THREADS / 32];
  unsigned long long ranks[2][5][kMostCtas];  // what the CTAs of a cluster reduced, by rank
  float all_score[kListed];                   // members of all CTAs
  int32_t all_index[kListed];
  unsigned long long found_above;
  float found_score;
  int32_t found_bin, found_index, members;
};

template <int THREADS, bool kCluster>
struct Block {
  Shared<THREADS>& sh;
  uint32_t rank, ctas;
  int half = 0, ranks_half = 0;

  // Every thread gets the results over all threads (of all CTAs); up to five values at once.  One
  // barrier: the next call uses the other words.
  template <typename V, typename Op>
  __device__ __forceinline__ static V lanes(V v, Op op, int from) {
    for (int off = from; off > 0; off >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
  }
  template <typename V>
  __device__ __forceinline__ V* slot(int k) const { return reinterpret_cast<V*>(sh.words[half][k]); }

  template <typename V, typename Op, typename... Rest>
  __device__ __forceinline__ void put(int k, V v, Op op, Rest... rest) {
    v = lanes(v, op, 16);
    if ((threadIdx.x & 31) == 0) slot<V>(k)[threadIdx.x >> 5] = v;
    if constexpr (sizeof...(rest) > 0) put(k + 1, rest...);
  }
  template <typename V, typename Op, typename... Rest>
  __device__ __forceinline__ void get(int k, V& v, Op op, Rest&&... rest) {
    v = lanes(slot<V>(k)[threadIdx.x & (THREADS / 32 - 1)], op, THREADS / 64);
    if constexpr (sizeof...(rest) > 0) get(k + 1, rest...);
  }
  template <typename V, typename Op, typename... Rest>
  __device__ __forceinline__ void put_rank(int k, V v, Op, Rest... rest) const {
    unsigned long long bits = 0;
    memcpy(&bits, &v, sizeof v);
    if (threadIdx.x < ctas) store_at(at_rank(&sh.ranks[ranks_half][k][rank], threadIdx.x), bits);
    if constexpr (sizeof...(rest) > 0) put_rank(k + 1, rest...);
  }
  template <typename V>
  __device__ __forceinline__ V of_rank(int which, int k, uint32_t r) const {
    V v;
    memcpy(&v, &sh.ranks[which][k][r], sizeof v);
    return v;
  }
  template <typename V, typename Op, typename... Rest>
  __device__ __forceinline__ void get_ranks(int k, V& v, Op op, Rest&&... rest) const {
    v = of_rank<V>(ranks_half, k, 0);
    for (uint32_t r = 1; r < ctas; ++r) v = op(v, of_rank<V>(ranks_half, k, r));
    if constexpr (sizeof...(rest) > 0) get_ranks(k + 1, rest...);
  }
  // reduce(value, op, value, op, ...): the values are replaced by the results.
  template <typename... Pairs>
  __device__ __forceinline__ void reduce(Pairs&&... pairs) {
    static_assert(sizeof...(pairs) <= 10, "five values");
    put(0, pairs...);
    __syncthreads();
    get(0, pairs...);
    half ^= 1;
    if constexpr (kCluster) {
      put_rank(0, pairs...);
      cluster_sync();
      get_ranks(0, pairs...);
      ranks_half ^= 1;
    }
  }
  // Of the last reduce's value k, an int: the sum over the CTAs before this one.
  __device__ __forceinline__ int before_rank(int k) const {
    int sum = 0;
    for (uint32_t r = 0; r < rank; ++r) sum += of_rank<int>(ranks_half ^ 1, k, r);
    return sum;
  }
  // All threads are through with a histogram; then bins b and b + 1 of it (b even), of all CTAs.
  __device__ __forceinline__ void meet() const {
    if constexpr (kCluster) cluster_sync(); else __syncthreads();
  }
  __device__ __forceinline__ void bins(int b, bool masses, unsigned long long& w0, unsigned long long& w1) const {
    if constexpr (kCluster) {
      w0 = w1 = 0;
#pragma unroll 4
      for (uint32_t r = 0; r < ctas; ++r) {
        const uint2 lo = load_pair_at(at_rank(&sh.bins[0][b], r));
        w0 += lo.x;
        w1 += lo.y;
        if (masses) {
          const uint2 up = load_pair_at(at_rank(&sh.bins[1][b], r));
          w0 += (unsigned long long)up.x << 32;
          w1 += (unsigned long long)up.y << 32;
        }
      }
    } else {
      w0 = sh.bins[0][b];
      w1 = sh.bins[0][b + 1];
      if (masses) {
        w0 += (unsigned long long)sh.bins[1][b] << 32;
        w1 += (unsigned long long)sh.bins[1][b + 1] << 32;
      }
    }
  }
  // Sum of the threads before this one.
  __device__ __forceinline__ unsigned long long before(unsigned long long v, unsigned long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long upto = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += up;
    }
    unsigned long long* words = sh.words[half][0];
    half ^= 1;
    if (lane == 31) words[warp] = upto;
    __syncthreads();
    unsigned long long w = words[lane & (THREADS / 32 - 1)], all = w;
    if (lane >= warp) w = 0;  // warps before this one (THREADS / 32 <= 32 words)
    if (lane >= THREADS / 32) all = 0;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      w += __shfl_xor_sync(0xffffffffu, w, off);
      all += __shfl_xor_sync(0xffffffffu, all, off);
    }
    *total = all;
    return w + upto - v;
  }
};

// Four consecutive elements of a row, `none` behind its end.
struct Quad {
  float v[4];
};
__device__ __forceinline__ Quad load_quad(const float* row, int q, int C, float none) {
  Quad out;
  if (4 * q + 3 < C && ((uintptr_t)row & 15) == 0) {
    const float4 f = reinterpret_cast<const float4*>(row)[q];
    out.v[0] = f.x; out.v[1] = f.y; out.v[2] = f.z; out.v[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) out.v[e] = 4 * q + e < C ? row[4 * q + e] : none;
  }
  return out;
}
__device__ __forceinline__ float most_of(const Quad& x) {  // NaN is none
  return fmaxf(fmaxf(x.v[0], x.v[1]), fmaxf(x.v[2], x.v[3]));
}

template <int THREADS, bool kCached, bool kCluster>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
sample_rows_kernel(const __grid_constant__ Args A) {
  using S = Shared<THREADS>;
  constexpr int kBins = S::kBins, kListed = S::kListed;
  extern __shared__ __align__(16) float cache[];
  __shared__ S sh;
  const uint32_t rank = kCluster ? cluster_rank() : 0, ctas = kCluster ? cluster_ctas() : 1;
  Block<THREADS, kCluster> block{sh, rank, ctas};
  const int64_t row = kCluster ? blockIdx.x / ctas : blockIdx.x;
  const int tid = threadIdx.x, C = A.cols, n = A.n;
  const float* const scores = A.scores + row * A.score_stride;
  const float* const uniforms = A.uniforms + row * A.uniform_stride;
  int64_t* const indices = A.indices + row * n;
  float* const probabilities = A.probabilities + row * n;
  const double T = A.temperature.at(row);

  // the slice of the row that this CTA looks at
  const int quads = (C + 3) / 4, share = kCluster ? (quads + (int)ctas - 1) / (int)ctas : quads;
  const int q_from = kCluster ? min((int)rank * share, quads) : 0, q_to = kCluster ? min(q_from + share, quads) : quads;
  const int i_from = kCluster ? min(4 * q_from, C) : 0, i_to = kCluster ? min(4 * q_to, C) : C;
  const auto score = [&](int i) { return kCached ? cache[i - i_from] : scores[i]; };
  const auto score_quad = [&](int q) {
    if (!kCached) return load_quad(scores, q, C, -INFINITY);
    Quad out;
    *reinterpret_cast<float4*>(&out) = reinterpret_cast<const float4*>(cache)[q - q_from];
    return out;
  };

  // The row comes into shared memory with everything in flight at once; its uniforms, needed
  // several passes later, are asked into L2 meanwhile.
  if (kCached) {
    if (((uintptr_t)scores & 15) == 0) {
      for (int i = i_from + 4 * tid; i + 3 < i_to; i += 4 * THREADS) copy_async<16>(cache + (i - i_from), scores + i);
      for (int i = max(i_from, i_to & ~3) + tid; i < i_to; i += THREADS) copy_async<4>(cache + (i - i_from), scores + i);
    } else {
      for (int i = i_from + tid; i < i_to; i += THREADS) copy_async<4>(cache + (i - i_from), scores + i);
    }
    copies_commit();
    if (q_from < q_to && i_to + tid < 4 * q_to) cache[i_to - i_from + tid] = -INFINITY;
  }
  for (int i = i_from + 32 * tid; i < i_to; i += 32 * THREADS) asm volatile("prefetch.global.L2 [%0];" ::"l"(uniforms + i));
  if (kCached) {
    copies_wait<0>();
    __syncthreads();
  }
  if (kCluster) cluster_sync();  // all CTAs have begun: their shared memory may be written
  // the largest and the smallest score, and how many there are
  float best = -INFINITY, least = INFINITY;
  int some = 0;
  for (int q = q_from + tid; q < q_to; q += THREADS) {
    const Quad x = score_quad(q);
    best = fmaxf(best, most_of(x));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool there = x.v[e] > -INFINITY;
      least = fminf(least, there ? x.v[e] : INFINITY);
      some += there;
    }
  }
  block.reduce(best, Most(), least, Least(), some, Add());
  if (some == 0 || !(T > 0.0)) {
    for (int d = tid; rank == 0 && d < n; d += THREADS) {
      indices[d] = -1;
      probabilities[d] = 0.f;
    }
    return;
  }
  const double inv_T = fmin(1.0 / T, 1e300), per_bit = inv_T * 1.4426950408889634;
  // candidates are the scores from `first` on (false for NaN and -inf)
  const float first = (double)least - (double)best > -699.0 * T
                          ? least
                          : first_score(best, T, kLeast);

  // The filters keep a prefix: scores above `cut`, and those equal to it up to index `cut_index`.
  float cut = -INFINITY;
  int32_t cut_index = -1;
  const auto inside = [&](float v, int i) { return v > cut || (v == cut && i <= cut_index); };
  const double best_d = finite(best);

  const int64_t k = A.top_k.at(row);
  const double p = A.top_p.at(row);
  const bool by_count = k > 0 && k < some, by_mass = p > 0.0 && p < 1.0;
  if (by_count && least < first) {  // entries that weigh nothing are no candidates
    least = INFINITY;
    some = 0;
    for (int i = i_from + tid; i < i_to; i += THREADS) {
      const float v = score(i);
      if (v >= first) {
        least = fminf(least, v);
        ++some;
      }
    }
    block.reduce(least, Least(), some, Add());
  }
  // Twice the same search: what the members add up to (one each, or their masses) has to
  // reach `limit`, and the new last member is the last one before which it has not.
#pragma unroll 1
  for (int masses = 0; masses < 2; ++masses) {
    if (masses ? !by_mass : !(by_count && k < some)) continue;
    double limit = (double)k;
    float high = best, low = fmaxf(fmaxf(least, first), cut);
    if (masses) {  // below -(shift + 2) ln 2 a mass rounds to none
      const float none = __double2float_rd(best_d - 0.6931471805599453 * (A.shift + 2) * T);
      low = fminf(fmaxf(low, none), best);
    }
    const auto weight = [&](float v) { return masses ? mass_of(v, best_d, per_bit, A.shift) : 1ull; };
    const auto enough = [&](unsigned long long sum) { return !((double)sum < limit); };
    unsigned long long above = 0;
    bool fresh = true;
    for (;;) {
      const auto member = [&](float v, int i) {  // low is at least the cut
        return v >= low && v <= high && (v != cut || i <= cut_index);
      };
      // the map falls with the score; in halves where a difference would overflow
      const float half = high - low < 3e38f ? 1.f : 0.5f;
      const float per = (kBins - 1) / (half * high - half * low);
      const auto bin_of = [&](float v) {
        return low == high ? 0 : min((int)((half * high - half * v) * per), kBins - 1);
      };
      __syncthreads();  // whatever the words of the union held has been read
      for (int i = tid; i < kBins; i += THREADS) sh.bins[0][i] = sh.bins[1][i] = 0;
      if (tid == 0) {
        sh.members = 0;
        sh.found_bin = kBins - 1;  // replaced below
        sh.found_above = above;
      }
      __syncthreads();
      if (masses) {
        for (int q = q_from + tid; q < q_to; q += THREADS) {
          const Quad x = score_quad(q);
          if (!(most_of(x) >= low)) continue;
          unsigned long long w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = mass_here(fmaxf(x.v[e], low), best_d, per_bit, A.shift);
            if (!member(x.v[e], 4 * q + e)) w[e] = 0;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (w[e] == 0) continue;
            const int bin = bin_of(x.v[e]);
            const uint32_t lo = (uint32_t)w[e], old = atomicAdd(&sh.bins[0][bin], lo);
            const uint32_t up = (uint32_t)(w[e] >> 32) + (old + lo < old ? 1u : 0u);
            if (up) atomicAdd(&sh.bins[1][bin], up);
          }
        }
      } else {
        for (int q = q_from + tid; q < q_to; q += THREADS) {
          const Quad x = score_quad(q);
          if (!(most_of(x) >= low)) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (member(x.v[e], 4 * q + e)) atomicAdd(&sh.bins[0][bin_of(x.v[e])], 1u);
        }
      }
      block.meet();
      const int b0 = 2 * tid;
      unsigned long long w0, w1, total;
      block.bins(b0, masses, w0, w1);
      const unsigned long long pre = above + block.before(w0 + w1, &total);
      if (masses && fresh) limit = p * (double)total;
      fresh = false;
      if (!enough(pre) && enough(pre + w0 + w1)) {  // one thread
        const bool second = !enough(pre + w0);
        sh.found_bin = b0 + second;
        sh.found_above = second ? pre + w0 : pre;
      }
      __syncthreads();
      const int bin = sh.found_bin;
      above = sh.found_above;
      float most = -INFINITY, fewest = INFINITY;
      int members = 0;
      // nothing of the bin lies below this: its lower end, a hundredth of its width and the rounding beyond
      const float lowest = low == high || !(per < 3e38f)
                               ? low
                               : fmaxf(low, (half * high - (bin + 1.01f) / per) / half -
                                                4e-7f * fmaxf(fabsf(high), fabsf(low)));
      for (int q = q_from + tid; q < q_to; q += THREADS) {
        const Quad x = score_quad(q);
        if (!(most_of(x) >= lowest)) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = x.v[e];
          const int i = 4 * q + e;
          if (!(v >= lowest) || !member(v, i) || bin_of(v) != bin) continue;
          most = fmaxf(most, v);
          fewest = fminf(fewest, v);
          if (kCluster) ++members;
          const int at = atomicAdd(&sh.members, 1);
          if (at < kListed) sh.list[at] = i;
        }
      }
      if (kCluster) {
        block.reduce(most, Most(), fewest, Least(), members, Add());
      } else {
        block.reduce(most, Most(), fewest, Least());
        members = sh.members;
      }
      if (members <= kListed) {
        if (kCluster) {  // every CTA gets everybody's members
          const int at = block.before_rank(2) + tid;
          if (tid < sh.members) {
            const int i = sh.list[tid];
            for (uint32_t r = 0; r < ctas; ++r) {
              store_at(at_rank(&sh.all_score[at], r), __float_as_uint(score(i)));
              store_at(at_rank(&sh.all_index[at], r), (uint32_t)i);
            }
          }
          cluster_sync();
          if (tid < members) sh.list[tid] = sh.all_index[tid];
        }
        static_assert(THREADS >= kListed, "a thread per ranked member");
        float mine = 0.f;
        int index = 0, rank = 0;
        if (tid < members) {
          index = sh.list[tid];
          mine = kCluster ? sh.all_score[tid] : score(index);
          sh.ranked.score[tid] = mine;
        }
        __syncthreads();
        if (tid < members) {
          int equal = 0;
#pragma unroll 8
          for (int j = 0; j < members; ++j) {
            const float v = sh.ranked.score[j];
            rank += v > mine;
            equal += v == mine;
          }
          if (equal > 1)
            for (int j = 0; j < members; ++j) rank += sh.ranked.score[j] == mine && sh.list[j] < index;
        }
        __syncthreads();
        if (tid < members) {
          sh.ranked.score[rank] = mine;
          sh.ranked.index[rank] = index;
          sh.ranked.mass[rank] = weight(mine);
        }
        __syncthreads();
        if (tid < 32) {  // the last member before which the sum is not enough
          unsigned long long sum = above;
          int last = 0;
#pragma unroll 1
          for (int base = 0; base < members; base += 32) {
            const unsigned long long w = base + tid < members ? sh.ranked.mass[base + tid] : 0;
            unsigned long long upto = w;
            for (int off = 1; off < 32; off <<= 1) {
              const unsigned long long up = __shfl_up_sync(0xffffffffu, upto, off);
              if (tid >= off) upto += up;
            }
            const bool in = base + tid < members && !enough(sum + upto - w);
            const unsigned votes = __ballot_sync(0xffffffffu, in);
            if (votes) last = base + 31 - __clz(votes);
            sum += __shfl_sync(0xffffffffu, upto, 31);
          }
          if (tid == 0) {
            sh.found_score = sh.ranked.score[last];
            sh.found_index = sh.ranked.index[last];
          }
        }
        __syncthreads();
        cut = sh.found_score;
        cut_index = sh.found_index;
        break;
      }
      if (most == fewest) {
        // More equal members than are listed: how many stay, and the index of the last of them.
        const unsigned long long each = weight(most);
        int lo = 1, hi = members;  // the largest r with !enough(above + (r - 1) * each)
        while (lo < hi) {
          const int mid = lo + (hi - lo + 1) / 2;
          if (!enough(above + (unsigned long long)(mid - 1) * each)) lo = mid; else hi = mid - 1;
        }
        int from = 0, to = C - 1;  // the smallest index up to which there are lo of them
        while (from < to) {
          const int mid = from + (to - from) / 2;
          int equal = 0;
          for (int i = i_from + tid; i <= mid && i < i_to; i += THREADS) {
            const float v = score(i);
            equal += v == most && inside(v, i);
          }
          block.reduce(equal, Add());
          if (equal >= lo) to = mid; else from = mid + 1;
        }
        cut = most;
        cut_index = from;
        break;
      }
      high = most;
      low = fewest;
    }
  }
  const double least_share = A.min_p.at(row);
  const bool by_share = least_share > 0.0 && least_share <= 1.0;
  const float floor_score = by_share ? fmaxf(first, first_score(best, T, log(least_share))) : first;
  const auto kept = [&](float v, int i) { return v >= floor_score && inside(v, i); };

  // The race in 32 bits: lower bounds.  -log u is a polynomial in 1 - u where u is near 1 (to
  // 3e-6 of its size) and the hardware's logarithm elsewhere (2^-22 of at least 0.06); the
  // outer logarithm is off by 2^-22 and what its argument is off by, a by a few 2^-24 of its size.  With
  // -4.6 < -log(-log u) < 16.7 that is less than a quarter of the 1e-6 (|sum| + 40) taken off.
  // a is (v - best) * part times 1 / (T * part), part a power of two that keeps both inside the 32-bit range
  // where scores are further apart than it, and where T is subnormal (there, if best * part overflows, none but the
  // best themselves are kept, with a = 0).  A subnormal second factor is off by at most 2^-150, a by 2.4e-7.
  const float lowest_kept = fmaxf(floor_score, cut);
  float part = 1.f;
  double per_part = inv_T;
  if (inv_T > 1e38) {
    part = 0x1p126f;
    per_part *= 0x1p-126;
  } else if (best < INFINITY && !(best - lowest_kept < 3.4e38f)) {
    part = 0.5f;
    per_part *= 2.0;
  }
  const float best_part = best * part, inv_Tf = (float)per_part;
  const auto lower = [&](float v, float u) {
    const float t = 1.f - u;
    const float l = t < 0.0625f ? t * (1.f + t * (0.5f + t * (0.33333333f + t * 0.25f))) : -__logf(u);
    const float g = (v == best ? 0.f : fmaf(v, part, -best_part) * inv_Tf) - __logf(l);
    return g - 1e-6f * (fabsf(g) + 40.f);
  };
  constexpr float kLeastUniform = 1.17549435e-38f;  // subnormal ones are raced in 64 bits
  const bool filtered = by_count || by_mass || by_share;
  double total = 0.0;
  float g_most = -INFINITY, g_least = INFINITY;
  int open = 0, odd = 0;  // candidates in the race; 1: a uniform of 0, 2: of 1 or subnormal
  __syncthreads();
  if (tid == 0) sh.members = 0;
  __syncthreads();
  for (int q = q_from + tid; q < q_to; q += THREADS) {
    const Quad x = score_quad(q);
    Quad g;
#pragma unroll
    for (int e = 0; e < 4; ++e) g.v[e] = -INFINITY;
    if (most_of(x) >= lowest_kept) {
      const Quad u = load_quad(uniforms, q, C, -1.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!kept(x.v[e], 4 * q + e)) continue;
        total += exp2_series<7>((finite(x.v[e]) - best_d) * per_bit, 0);
        if (u.v[e] >= kLeastUniform && u.v[e] < 1.f) {
          g.v[e] = lower(x.v[e], u.v[e]);
          g_most = fmaxf(g_most, g.v[e]);
          g_least = fminf(g_least, g.v[e]);
          ++open;
          if (filtered) {
            const int at = atomicAdd(&sh.members, 1);
            if (at < kFew) sh.list[at] = 4 * q + e;
          }
        } else if (u.v[e] >= 0.f && u.v[e] <= 1.f) {
          odd |= u.v[e] > 0.f ? 2 : 1;
        }
      }
    }
    if (kCached) reinterpret_cast<float4*>(cache)[q - q_from] = *reinterpret_cast<const float4*>(&g);
  }
  block.reduce(total, Add(), g_most, Most(), g_least, Least(), open, Add(), odd, Or());
  // -inf marks what is not in the race, the padding behind the row among it: whatever the
  // bounds are, none of that is listed below
  g_least = fmaxf(g_least, -3.4e38f);

  bool listed = !(odd & 2) && (open >= n || !(odd & 1));
  if (listed && open > 0) {
    int members = open, place = kCluster ? block.before_rank(3) : 0;  // of all; the first of this CTA's among them
    if (!filtered || open > kFew) {
      const float per = g_most > g_least ? (kBins - 1) / (g_most - g_least) : 0.f;
      const auto bounds = [&](int q) {
        Quad g = score_quad(q);
        if (kCached || !(most_of(g) >= lowest_kept)) {
          if (!kCached)
            for (int e = 0; e < 4; ++e) g.v[e] = -INFINITY;
          return g;
        }
        const Quad u = load_quad(uniforms, q, C, -1.f);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          g.v[e] = kept(g.v[e], 4 * q + e) && u.v[e] >= kLeastUniform && u.v[e] < 1.f ? lower(g.v[e], u.v[e]) : -INFINITY;
        return g;
      };
      float edge = g_least;  // at least n lower bounds reach it
      __syncthreads();
      if (tid == 0) sh.members = 0;
      if (open > n) {
        for (int i = tid; i < kBins; i += THREADS) sh.bins[0][i] = 0;
        if (tid == 0) sh.found_bin = kBins - 1;
        __syncthreads();
        for (int q = q_from + tid; q < q_to; q += THREADS) {
          const Quad g = bounds(q);
          if (!(most_of(g) >= g_least)) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (g.v[e] >= g_least) atomicAdd(&sh.bins[0][min((int)((g_most - g.v[e]) * per), kBins - 1)], 1u);
        }
        block.meet();
        unsigned long long c0, c1, all;
        block.bins(2 * tid, false, c0, c1);
        const unsigned long long pre = block.before(c0 + c1, &all), want = n;
        if (pre < want && pre + c0 + c1 >= want) sh.found_bin = 2 * tid + (pre + c0 < want);
        __syncthreads();
        // the lower end of the bin, a hundredth of its width and a rounding of the sum beyond it
        if (sh.found_bin < kBins - 1 && per > 0.f)
          edge = fmaxf(edge, g_most - (sh.found_bin + 1.01f) / per - 4e-7f * (fabsf(g_most) + fabsf(g_least)));
      }
      edge -= 2.1e-6f * (fabsf(edge) + 41.f);  // what an upper bound may lie above its lower one
      __syncthreads();
      members = 0;
      for (int q = q_from + tid; q < q_to; q += THREADS) {
        const Quad g = bounds(q);
        if (!(most_of(g) >= edge)) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!(g.v[e] >= edge)) continue;
          if (kCluster) ++members;
          const int at = atomicAdd(&sh.members, 1);
          if (at < kRaced) sh.list[at] = 4 * q + e;
        }
      }
      if (kCluster) {
        block.reduce(members, Add());
        place = block.before_rank(0);
      } else {
        __syncthreads();
        members = sh.members;
      }
    }
    listed = members <= kRaced;
    if (listed) {
#pragma unroll 1
      for (int j = tid; j < (kCluster ? sh.members : members); j += THREADS) {
        const int i = sh.list[j];
        const double r = race_of(scores[i], best, T, uniforms[i]) + 0.0;  // -0 as 0
        const unsigned long long bits = (unsigned long long)__double_as_longlong(r);
        const unsigned long long image = bits >> 63 ? ~bits : bits | (1ull << 63);
        if (kCluster) {  // the first CTA's own stay where they are, the others' come behind them
          store_at(at_rank(&sh.race[place + j], 0), image);
          store_at(at_rank(&sh.list[place + j], 0), (uint32_t)i);
        } else {
          sh.race[j] = image;
        }
      }
      block.meet();
      if (rank != 0) return;
      if (members <= kListed) {  // ranked against each other
        if (tid < members) {
          const unsigned long long mine = sh.race[tid];
          const int i = sh.list[tid];
          int rank = 0, equal = 0;
#pragma unroll 8
          for (int o = 0; o < members; ++o) {
            const unsigned long long other = sh.race[o];
            rank += other > mine;
            equal += other == mine;
          }
          if (equal > 1)
            for (int o = 0; o < members; ++o) rank += sh.race[o] == mine && sh.list[o] < i;
          if (rank < n) {
            indices[rank] = i;
            probabilities[rank] = share_of(scores[i], best, T, total);
          }
        }
      } else {  // sorted, best first
        int size = 2 * kListed;
        while (size < members) size *= 2;
        for (int j = members + tid; j < size; j += THREADS) {
          sh.race[j] = 0;
          sh.list[j] = 0x7fffffff;
        }
        __syncthreads();
#pragma unroll 1
        for (int span = 2; span <= size; span <<= 1) {
#pragma unroll 1
          for (int gap = span >> 1; gap > 0; gap >>= 1) {
#pragma unroll 1
            for (int q = tid; q < size / 2; q += THREADS) {
              const int a = ((q & ~(gap - 1)) << 1) | (q & (gap - 1)), b = a | gap;
              const unsigned long long ra = sh.race[a], rb = sh.race[b];
              const int ia = sh.list[a], ib = sh.list[b];
              const bool b_first = rb > ra || (rb == ra && ib < ia);
              if (b_first == ((a & span) == 0)) {
                sh.race[a] = rb;
                sh.race[b] = ra;
                sh.list[a] = ib;
                sh.list[b] = ia;
              }
            }
            __syncthreads();
          }
        }
        for (int d = tid; d < min(n, members); d += THREADS) {
          indices[d] = sh.list[d];
          probabilities[d] = share_of(scores[sh.list[d]], best, T, total);
        }
      }
      for (int d = members + tid; d < n; d += THREADS) {
        indices[d] = -1;
        probabilities[d] = 0.f;
      }
      return;
    }
  }
  // Uniforms of 0, 1 or below the normal range among the draws, more equal race values than are
  // listed, or nobody in the race: one pass for each draw, over the row in memory.
  double last = INFINITY;
  int last_index = -1;
  bool more = true;
#pragma unroll 1
  for (int d = 0; d < n; ++d) {
    double g = -INFINITY;
    int at = C;
    if (more) {
#pragma unroll 1
      for (int i = i_from + tid; i < i_to; i += THREADS) {
        if (!kept(scores[i], i)) continue;
        const double r = race_of(scores[i], best, T, uniforms[i]);
        if (!(r >= -1e300) || r > last || (r == last && i <= last_index)) continue;
        if (r > g) {
          g = r;
          at = i;
        }
      }
    }
    double most = g;
    block.reduce(most, Most());
    if (g != most || !(most > -INFINITY)) at = C;
    block.reduce(at, Least());
    more = at < C;
    last = most;
    last_index = at;
    if (rank == 0 && tid == 0) {
      indices[d] = more ? at : -1;
      probabilities[d] = more ? share_of(scores[at], best, T, total) : 0.f;
    }
  }
}

}  // namespace sample
}  // namespace maxsim
